// What the kernels over a paged cache have in common: the pool, a step's requests, and the host's checks
// of pools and outputs.
//
// A pool of pages holds the keys (and another the values) of requests of different lengths: page
// j, KV head g, slot s at element j * page_stride + g * head_stride + s * 128, 128 elements each,
// with page_size slots per page (a power of two from 16 on). Token t of request b is in page
// table[b][t / page_size], slot t % page_size. A step brings rows q_start[b] .. q_start[b + 1] - 1
// of request b: its newest tokens, the last of them at position lens[b] - 1.
//
// Everything that decides an address is read on the device and checked there: rows outside
// [0, T), positions outside the table and page ids outside the pool are neither read nor written
// (an absent key is masked, an absent place is not stored to).
#pragma once
#include "dkv_common.h"
#include "dkv_mfma_ops.h"
#include "dkv_paged_index.h"

namespace {

constexpr int PG_DH = 128;
static_assert(paged_slot_at(1) == PG_DH, "");

// x / d for 0 <= x < 2^31, by a product: m = ceil(2^32 / d) gives the quotient or one more.
struct Divisor {
  uint32_t d, m;
};
inline Divisor divisor(int d) { return {(uint32_t)d, d > 1 ? (uint32_t)((0x100000000ULL + d - 1) / d) : 0u}; }
__device__ __forceinline__ int quot(const Divisor& v, int x) {
  uint32_t q = __umulhi((uint32_t)x, v.m);
  q -= q * v.d > (uint32_t)x;
  return v.d == 1 ? x : (int)q;
}

__device__ __forceinline__ int pg_wave_scan(int v) {  // inclusive, as dkv_wave_scan_fast
  v += dkv_dpp_i32<0x111>(v);
  v += dkv_dpp_i32<0x112>(v);
  v += dkv_dpp_i32<0x114>(v);
  v += dkv_dpp_i32<0x118>(v);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
  return v;
}

struct PagedPool {
  long long page_stride, head_stride;  // elements
  int num_pages, page_size, page_shift;
  const int* table;  // (B, cols), row stride ld
  long long table_ld;
  int cols;
};

// One request of the step, clamped to what the buffers hold.
struct PagedRequest {
  int row0, n;  // its rows of the step
  int len;      // keys it attends (the last row's), at most what the table has room for
  int pos0;     // position of its first row (negative where the lengths do not fit the rows)
};

__device__ __forceinline__ PagedRequest paged_request(const PagedPool& pool, const int* q_start,
                                                      const int* lens, int b, int T) {
  PagedRequest r;
  const int a = q_start[b], e = q_start[b + 1], len = lens[b];
  r.row0 = max(a, 0);
  r.n = min(e, T) - r.row0;
  r.pos0 = len - (e - a) + (r.row0 - a);
  const long long room = (long long)pool.cols << pool.page_shift;
  r.len = (int)min((long long)max(len, 0), room);
  return r;
}

// The same in scalar registers, for a request that is the whole wave's.
__device__ __forceinline__ PagedRequest uniform(PagedRequest r) {
  r.row0 = __builtin_amdgcn_readfirstlane(r.row0);
  r.n = __builtin_amdgcn_readfirstlane(r.n);
  r.len = __builtin_amdgcn_readfirstlane(r.len);
  r.pos0 = __builtin_amdgcn_readfirstlane(r.pos0);
  return r;
}

// The page of token t of request b, or -1 where there is none.
__device__ __forceinline__ int paged_page(const PagedPool& pool, int b, int t) {
  const int c = t >> pool.page_shift;
  if (t < 0 || c >= pool.cols) return -1;
  const int id = pool.table[(long long)b * pool.table_ld + c];
  return id >= 0 && id < pool.num_pages ? id : -1;
}

template <int DT>
__device__ __forceinline__ void load8(const uint16_t* p, float (&f)[8]) {
  const dkv_u32x4 v = *(const dkv_u32x4*)p;
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    f[2 * k] = dkv_elt_to_f32<DT>(w[k] & 0xffffu);
    f[2 * k + 1] = dkv_elt_to_f32<DT>(w[k] >> 16);
  }
}
template <int DT>
__device__ __forceinline__ dkv_u32x4 round8(const float (&f)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if constexpr (DT == DKV_BF16)
      w[k] = dkv_f32_to_bf16_bits(f[2 * k]) | (dkv_f32_to_bf16_bits(f[2 * k + 1]) << 16);
    else
      w[k] = dkv_f32_to_f16_bits(f[2 * k]) | (dkv_f32_to_f16_bits(f[2 * k + 1]) << 16);
  }
  return dkv_u32x4{w[0], w[1], w[2], w[3]};
}

// The last request for which starts(b) holds, as it does for every one before (64 a step, one per lane);
// 0 if for none.
template <class F>
__device__ __forceinline__ int last_request(int B, int lane, F&& starts) {
  int lo = 0, n = B;
  while (n > 1) {
    const int step = (n + 63) / 64;
    const int i = lo + lane * step;
    const bool at = lane * step < n && starts(min(i, B - 1));
    const int cnt = max(1, __popcll(__ballot(at)));
    const int skip = (cnt - 1) * step;
    lo += skip;
    n = min(step, n - skip);
  }
  return lo;
}
// The request of row `row`: the last one that starts at or before it, or -1 for a row of no request.
__device__ __forceinline__ int request_of_row(const int* q_start, int B, int row, int lane) {
  if (row < q_start[0] || row >= q_start[B]) return -1;
  return last_request(B, lane, [&](int b) { return q_start[b] <= row; });
}

// A head's 128 values at src, optionally normed with weights nw and rotated by position pos: dims
// 8c .. 8c + 7 in ox, 64 + 8c .. 64 + 8c + 7 in oy. The eight lanes c of a head work together.
template <int DT>
__device__ __forceinline__ void paged_turn(const uint16_t* src, const uint16_t* nw, float eps, int pos,
                                           const double* rev, int c, float (&ox)[8], float (&oy)[8]) {
  float x[8], y[8];
  load8<DT>(src + 8 * c, x);
  load8<DT>(src + 64 + 8 * c, y);
  if (nw) {
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], fmaf(y[e], y[e], ss));
#pragma unroll
    for (int o = 1; o <= 4; o <<= 1) ss += __shfl_xor(ss, o, 64);
    const float inv = 1.0f / sqrtf(ss * (1.0f / PG_DH) + eps);
    float wx[8], wy[8];
    load8<DT>(nw + 8 * c, wx);
    load8<DT>(nw + 64 + 8 * c, wy);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = x[e] * inv * wx[e];
      y[e] = y[e] * inv * wy[e];
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const double r = (double)pos * rev[8 * c + e];
    const float f = (float)(r - floor(r));  // part of a revolution: 0 .. 1
    const float sn = __builtin_amdgcn_sinf(f), cs = __builtin_amdgcn_cosf(f);
    ox[e] = x[e] * cs - y[e] * sn;
    oy[e] = y[e] * cs + x[e] * sn;
  }
}

// ---- pages of 8 bits ----
//
// Codes are e4m3 (finite, NaN at 0x7f and 0xff), and the 16 tokens of a block (slots 16i .. 16i + 15 of a
// page's head, keys or values) share a scale 2^(byte - 127): block i's at byte i of (page, head), strides
// page_stride and head_stride of the scales. The value is code * scale, which dkv_paged_append8 keeps
// within the numbers of the model's type.
constexpr int PG_BLOCK = 16;
struct PagedScales {
  const uint8_t* k;
  const uint8_t* v;
  long long page_stride, head_stride;
};
// As the conversions to 16 bits take it (by its exponent field), and as a factor in fp32.
__device__ __forceinline__ float pg_scale(uint32_t byte) { return __uint_as_float(byte << 23); }
__device__ __forceinline__ float pg_factor(uint32_t byte) {
  return __uint_as_float(byte == 0 ? 0x00400000u : byte == 255 ? 0x7fc00000u : byte << 23);
}

// Two codes of a dword times a scale, as two 16-bit numbers (exact where they are such numbers).
template <int DT, bool HIGH>
__device__ __forceinline__ uint32_t pg_pair(uint32_t codes, float scale) {
  if constexpr (DT == DKV_BF16)
    return __builtin_bit_cast(uint32_t,
                              __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, HIGH));
  else
    return __builtin_bit_cast(uint32_t,
                              __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, scale, HIGH));
}
// Eight codes in fp32.
__device__ __forceinline__ void pg_codes8(const uint8_t* p, float scale, float (&f)[8]) {
  const dkv_u32x2 w = *(const dkv_u32x2*)p;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    f[4 * k] = __builtin_amdgcn_cvt_f32_fp8(w[k], 0) * scale;
    f[4 * k + 1] = __builtin_amdgcn_cvt_f32_fp8(w[k], 1) * scale;
    f[4 * k + 2] = __builtin_amdgcn_cvt_f32_fp8(w[k], 2) * scale;
    f[4 * k + 3] = __builtin_amdgcn_cvt_f32_fp8(w[k], 3) * scale;
  }
}

inline int check_scales(const PagedScales& s, int num_pages, int page_size, int Hkv) {
  if (!s.k || !s.v || s.page_stride < 0 || s.head_stride < 0) return DKV_E_ARG;
  if (s.head_stride < page_size / PG_BLOCK && Hkv > 1) return DKV_E_ARG;
  if (s.page_stride < page_size / PG_BLOCK && num_pages > 1) return DKV_E_ARG;
  return DKV_OK;
}

inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// T x H segments of `len` bytes, segment (i, h) at `at` + i st + h sh; a stride of a size of one is any.
struct Segments {
  long long at, st, sh, len;
  int T, H;
  long long end() const { return at + (T - 1) * st + (H - 1) * sh + len; }
};
// Whether a segment of a and one of b, of the same strides, have a byte in common (of one array with
// itself: two of its segments).
inline bool segments_meet(const Segments& a, const Segments& b, bool itself = false) {
  const long long st = a.T > 1 ? a.st : 0;
  for (int dh = 1 - a.H; dh < b.H; ++dh) {
    // the least di for which b's segment ends behind the start of a's
    const long long x = b.at - a.at + dh * b.sh;
    long long di = 1 - a.T;
    if (st > 0 && x + di * st + b.len <= 0) di += (-b.len - x - di * st) / st + 1;
    if (itself && dh == 0 && di <= 0) di = 1;
    if (di < a.T && x + di * st + b.len > 0 && x + di * st < a.len) return true;
  }
  return false;
}
// Whether an output's rows may be written while an operator reads `in`: apart from it (or, with its
// strides, between its rows), or in its place, row for row; no two of them on top of each other.
inline bool output_apart(const Segments& out, const Segments& in, bool in_place) {
  const bool nested =  // (the usual layouts: rows of heads, or heads of rows)
      (out.sh >= out.len && (out.T == 1 || out.st >= (out.H - 1) * out.sh + out.len)) ||
      (out.st >= out.len && (out.H == 1 || out.sh >= (out.T - 1) * out.st + out.len));
  if (!nested && segments_meet(out, out, true)) return false;
  if (in_place || out.end() <= in.at || in.end() <= out.at) return true;
  const bool alike = (out.T == 1 || out.st == in.st) &&
                     ((out.H == 1 && in.H == 1) || (out.H == in.H ? out.sh == in.sh : in.H == 1));
  if (alike && out.H == in.H) return !segments_meet(in, out);
  if (!alike) return false;
  for (int h = 0; h < out.H; ++h) {
    const Segments one = {out.at + h * out.sh, out.st, 0, out.len, out.T, 1};
    if (segments_meet(in, one)) return false;
  }
  return true;
}

inline int fill_pool(PagedPool& pool, long long page_stride, long long head_stride, int num_pages,
                     int page_size, const int* table, long long table_ld, int cols, int Hkv,
                     int aligned = 8) {  // elements of 16 bytes
  if (num_pages < 0 || cols < 0 || table_ld < cols) return DKV_E_ARG;
  if (page_size < 16 || (page_size & (page_size - 1))) return DKV_E_UNSUPPORTED;
  if (head_stride < (long long)page_size * PG_DH && Hkv > 1) return DKV_E_ARG;
  if (page_stride < 0 || head_stride < 0) return DKV_E_ARG;
  if (page_stride % aligned || head_stride % aligned) return DKV_E_UNSUPPORTED;
  if (page_stride < (long long)page_size * PG_DH && num_pages > 1) return DKV_E_ARG;
  if (cols > 0 && !table) return DKV_E_ARG;
  if ((long long)cols * page_size > 0x7fffffffLL - 4096) return DKV_E_UNSUPPORTED;
  pool.page_stride = page_stride;
  pool.head_stride = head_stride;
  pool.num_pages = num_pages;
  pool.page_size = page_size;
  pool.page_shift = __builtin_ctz((unsigned)page_size);
  pool.table = table;
  pool.table_ld = table_ld;
  pool.cols = cols;
  return DKV_OK;
}

}  // namespace
