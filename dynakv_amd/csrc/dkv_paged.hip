// The paged cache: the append of a step's keys and values, and the attention of its new tokens.
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
#include "dkv_common.h"
#include "dkv_mfma_ops.h"

#include <mutex>

namespace {

constexpr int PG_DH = 128;

// x / d for 0 <= x < 2^31, by a product: m = ceil(2^32 / d) gives the quotient or one more.
struct Divisor {
  uint32_t d, m;
};
Divisor divisor(int d) { return {(uint32_t)d, d > 1 ? (uint32_t)((0x100000000ULL + d - 1) / d) : 0u}; }
__device__ __forceinline__ int quot(const Divisor& v, int x) {
  uint32_t q = __umulhi((uint32_t)x, v.m);
  q -= q * v.d > (uint32_t)x;
  return v.d == 1 ? x : (int)q;
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

// ---------------------------------------------------------------------------------------
// Append: per row of the fused q/k/v projection and head, optionally the RMS norm of the head's
// 128 values with a weight (queries and keys), the rotation by the row's position (queries and
// keys), then the queries to q_out and the keys and values to their page. In fp32 with one
// rounding at the end:
//   y = x / sqrt(mean(x^2) + eps) * w,   o_j = y_j cos a_j - y_{j+64} sin a_j,
//   o_{j+64} = y_{j+64} cos a_j + y_j sin a_j,   a_j = pos * f_j.
// The angle is formed in 64 bits, in revolutions: at position 100000 a 32-bit angle is off by up to
// 2^-8 of a radian, as much as a bf16 rounding; reduced to one revolution it fits 32 bits.
// One wave per row and 8 heads: lane (head h = lane / 8, piece c = lane % 8) holds dims
// 8c .. 8c + 7 and 64 + 8c .. 64 + 8c + 7, so both halves of its eight pairs.
//
// Bound by memory where there is much to do: 8192 tokens of 32 + 2 x 8 heads with norms 44.6 us, 4.5 TB/s
// of reads and writes (a large copy has 4.8); 16 tokens 4.0 us, the chain of loads to the page id.
// Stores past the caches (non-temporal) take 3 us off the former and add 9 to the attention after it.
// ---------------------------------------------------------------------------------------
struct AppendParams {
  const uint16_t* qkv;
  long long qkv_ld;
  uint16_t* q_out;
  long long q_st, q_sh;
  uint16_t* k;
  uint16_t* v;
  PagedPool pool;
  const int* q_start;
  const int* lens;
  int B, T, Hq, Hkv;
  const uint16_t* q_norm;  // (128,), or null: no norm
  const uint16_t* k_norm;
  float eps;
  double rev[PG_DH / 2];  // revolutions per position of each pair
};

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

// The request of row `row`: the last one that starts at or before it (64 starts per step, one per
// lane), or -1 for a row of no request.
__device__ __forceinline__ int request_of_row(const int* q_start, int B, int row, int lane) {
  if (row < q_start[0] || row >= q_start[B]) return -1;
  int lo = 0, n = B;
  while (n > 1) {
    const int step = (n + 63) / 64;
    const int i = lo + lane * step;
    const bool at = lane * step < n && q_start[min(i, B - 1)] <= row;
    const int cnt = max(1, __popcll(__ballot(at)));
    const int skip = (cnt - 1) * step;
    lo += skip;
    n = min(step, n - skip);
  }
  return lo;
}

constexpr int AP_WAVES = 4;

template <int DT>
__global__ __launch_bounds__(64 * AP_WAVES) void paged_append_kernel(AppendParams p) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int heads = p.Hq + 2 * p.Hkv;
  const int groups = (heads + 7) / 8;
  const long long item = (long long)blockIdx.x * AP_WAVES + wave;
  if (item >= (long long)p.T * groups) return;
  const int row = (int)(item / groups);
  const int h = (int)(item % groups) * 8 + (lane >> 3);
  const int c = lane & 7;
  const int b = request_of_row(p.q_start, p.B, row, lane);
  if (b < 0) return;
  const int a0 = p.q_start[b], a1 = p.q_start[b + 1];
  const int pos = p.lens[b] - (a1 - a0) + (row - a0);
  if (pos < 0 || h >= heads) return;
  const uint16_t* src = p.qkv + (long long)row * p.qkv_ld + (long long)h * PG_DH + 8 * c;
  const bool is_q = h < p.Hq, is_v = h >= p.Hq + p.Hkv;
  uint16_t* dst;
  if (is_q) {
    dst = p.q_out + (long long)row * p.q_st + (long long)h * p.q_sh;
  } else {
    const int page = paged_page(p.pool, b, pos);
    const int g = is_v ? h - p.Hq - p.Hkv : h - p.Hq;
    dst = page < 0 ? nullptr
                   : (is_v ? p.v : p.k) + (long long)page * p.pool.page_stride +
                         (long long)g * p.pool.head_stride +
                         (long long)(pos & (p.pool.page_size - 1)) * PG_DH;
  }
  if (is_v) {
    if (dst) {
      *(dkv_u32x4*)(dst + 8 * c) = *(const dkv_u32x4*)src;
      *(dkv_u32x4*)(dst + 64 + 8 * c) = *(const dkv_u32x4*)(src + 64);
    }
    return;
  }
  float x[8], y[8];
  load8<DT>(src, x);
  load8<DT>(src + 64, y);
  const uint16_t* nw = is_q ? p.q_norm : p.k_norm;
  if (nw) {
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], fmaf(y[e], y[e], ss));
#pragma unroll
    for (int o = 1; o <= 4; o <<= 1) ss += __shfl_xor(ss, o, 64);
    const float inv = 1.0f / sqrtf(ss * (1.0f / PG_DH) + p.eps);
    float wx[8], wy[8];
    load8<DT>(nw + 8 * c, wx);
    load8<DT>(nw + 64 + 8 * c, wy);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = x[e] * inv * wx[e];
      y[e] = y[e] * inv * wy[e];
    }
  }
  if (!dst) return;
  float ox[8], oy[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const double r = (double)pos * p.rev[8 * c + e];
    const float f = (float)(r - floor(r));  // part of a revolution: 0 .. 1
    const float sn = __builtin_amdgcn_sinf(f), cs = __builtin_amdgcn_cosf(f);
    ox[e] = x[e] * cs - y[e] * sn;
    oy[e] = y[e] * cs + x[e] * sn;
  }
  *(dkv_u32x4*)(dst + 8 * c) = round8<DT>(ox);
  *(dkv_u32x4*)(dst + 64 + 8 * c) = round8<DT>(oy);
}

// ---------------------------------------------------------------------------------------
// Attention of the new tokens over their request's pages: the token at position t attends keys
// 0 .. t; o = sum_k exp(s_k - m) v_k / sum_k exp(s_k - m), s_k = scale q . k, one pass over the
// keys with a running maximum and sum.
// ---------------------------------------------------------------------------------------
// A running maximum of no keys: finite, so that exp2(-inf - it) is 0, and below every other score.
constexpr float PG_NO_MAX = -3.4028234663852886e38f;
// Weights are powers of two measured from a row's reference (log2 units), which is PG_BIAS below a running
// maximum and raised when a score exceeds that by more than the kernel's rescale step. fp16's step is
// 2^-24 for all numbers below 2^-14, so its weights are kept as large as it can hold: the largest of a row at
// 2^12 to 2^15, so that the others have all their bits down to 2^-26 of it (18 nats) and some to 2^-36.
// With the largest at 1 to 2^8, 4000 keys 18 nats below one whose value is 0 came out up to 11% off in
// chunks, 1.7% for single tokens; with this 2e-5 and 2e-6, in the same time. The power cancels in the
// division; maxima in records are references. bf16 has fp32's range.
template <int DT>
constexpr float PG_BIAS = DT == DKV_F16 ? 12.f : 0.f;
constexpr float PG_F16_RESCALE = 3.f;  // 2^(12 + 3) and a rounding below fp16's 65504
struct AttendParams {
  const uint16_t* q;
  long long q_st, q_sh;
  const uint16_t* k;
  const uint16_t* v;
  PagedPool pool;
  const int* q_start;
  const int* lens;
  void* out;
  long long o_st, o_sh;
  int B, T, Hq, Hkv, hpg;
  Divisor by_hpg, by_hkv;
  float scale_log2;  // softmax scale * log2(e)
  float* records;    // split records
  int* counters;     // arrival counters, zero between calls
  int split;         // whether a request's keys may be split among workgroups
  int out_wide;      // output rows begin at multiples of four values, aligned as such
};

// N loads of 16 bytes a lane, at byte offset off[i] + 1024 i of a buffer resource, into LDS at lds_base +
// 1024 i + 16 * lane (an instruction's offset counts on both sides, so that M0 is set once; one block of
// inline assembly, so that the compiler does not change M0 in between, neither moves LDS accesses across
// it nor waits for it before later LDS reads; the kernels wait for these loads themselves).
// ONCE: data that no other workgroup reads, passed by the caches (two requests of 65533 tokens, single
// new ones: 89 us, 6.0 TB/s, against 101 us without; 16 of 8192: 88 against 101).
template <bool ONCE, int N>
__device__ __forceinline__ void pg_lds_loads(__amdgpu_buffer_rsrc_t rsrc, uint32_t lds_base,
                                             const uint32_t (&off)[N]) {
  static_assert(N == 2 || N == 4, "");
  if constexpr (ONCE && N == 4)
    asm volatile(
        "s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %5, 0 offen nt lds\n\t"
        "buffer_load_dwordx4 %2, %5, 0 offen offset:1024 nt lds\n\t"
        "buffer_load_dwordx4 %3, %5, 0 offen offset:2048 nt lds\n\t"
        "buffer_load_dwordx4 %4, %5, 0 offen offset:3072 nt lds" ::"s"(lds_base),
        "v"(off[0]), "v"(off[1]), "v"(off[2]), "v"(off[3]), "s"(rsrc)
        : "memory", "m0");
  else if constexpr (N == 4)
    asm volatile(
        "s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %5, 0 offen lds\n\t"
        "buffer_load_dwordx4 %2, %5, 0 offen offset:1024 lds\n\t"
        "buffer_load_dwordx4 %3, %5, 0 offen offset:2048 lds\n\t"
        "buffer_load_dwordx4 %4, %5, 0 offen offset:3072 lds" ::"s"(lds_base),
        "v"(off[0]), "v"(off[1]), "v"(off[2]), "v"(off[3]), "s"(rsrc)
        : "memory", "m0");
  else
    asm volatile(
        "s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %3, 0 offen lds\n\t"
        "buffer_load_dwordx4 %2, %3, 0 offen offset:1024 lds" ::"s"(lds_base),
        "v"(off[0]), "v"(off[1]), "s"(rsrc)
        : "memory", "m0");
}
__device__ __forceinline__ void pg_wait_vm() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
typedef __attribute__((address_space(3))) dkv_i16x4 pg_lds_i16x4;
__device__ __forceinline__ dkv_u32x2 pg_read_tr(const uint8_t* p) {
  return __builtin_bit_cast(
      dkv_u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                     (pg_lds_i16x4*)(__attribute__((address_space(3))) uint8_t*)p));
}

// ---- few rows: single tokens, a few drafted ones ----
//
// A request whose new tokens times query heads per KV head fill at most 16 rows. Bound by the keys
// and values it reads once. A unit is (request, KV head); its keys go to the waves of one
// workgroup, or of several (parts), in tiles of 16, which lie in one page each. A wave's tile of K
// and V (4 KB each) lands in its own part of LDS by direct-to-LDS loads, 16-byte pieces XOR-swizzled
// by token, the next tile's loads in flight meanwhile; the resource of a load ends with the request's
// tokens, so slots behind them read as zero and cost nothing. S^T = K Q^T and P V on 16x16x32 MFMA
// with the rows in the operand's columns; the weights go to the products as 16-bit hi + lo
// pairs, which the 32 deep products of 16 tokens have room for. Waves are joined in LDS, parts by the
// unit's last one to arrive. 16 requests of 2K to 8K tokens (8 KV heads) 63 us, 5.6 TB/s; two of 65533
// 89 us, 6.0 TB/s; one of 96 5.0 us, the latency of lengths, page ids, one tile and the joins.
//
// How a step's units are cut, where there are fewer than D_WGS: requests have any lengths, which only
// the device knows, and the launch has a fixed number of workgroups. Every wave finds the smallest part C
// (tiles) for which sum over units of ceil(tiles / C) parts fit the launch, and takes its own from the
// running sums. From D_WGS units on (32 requests of 8 KV heads) a unit is one workgroup's, whatever its
// length: 32 requests of 8192 tokens 159 us (6.7 TB/s, partly from the memory-side cache), 33 of them 226,
// a second round of workgroups; one of 65536 beside 39 of 500 570 us, beside 20 of 500, in parts, 66.
constexpr int DSLOT = 2;                    // tile slots per wave
constexpr int DTILE = 16;
constexpr int DTILE_BYTES = DTILE * PG_DH * 2;
constexpr int DSLOT_BYTES = 2 * DTILE_BYTES;
constexpr int DROWS = 16;
constexpr int DREC = DROWS * (PG_DH + 2);   // floats of a record: m, l and acc[128] of 16 rows
constexpr int D_COUNTERS = 16384;           // leading workspace ints
constexpr int D_WGS = 256;                  // workgroups of 8 waves: one per CU
constexpr int D_SPLIT_B = 256;              // requests a wave can hold the lengths of (4 a lane)
static_assert(D_WGS <= D_SPLIT_B && D_WGS <= D_COUNTERS, "units that are cut: fewer than D_WGS");
constexpr int D_MIN_TILES = 16;             // least part
template <int DT>                           // log2 units the running maximum may be exceeded by
constexpr float D_RESCALE = DT == DKV_F16 ? PG_F16_RESCALE : 11.5f;

__device__ __forceinline__ int pg_wave_sum(int v) { return dkv_wave_sum_fast_i(v); }
__device__ __forceinline__ int pg_wave_scan(int v) {  // inclusive, as dkv_wave_scan_fast
  v += dkv_dpp_i32<0x111>(v);
  v += dkv_dpp_i32<0x112>(v);
  v += dkv_dpp_i32<0x114>(v);
  v += dkv_dpp_i32<0x118>(v);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
  return v;
}
__device__ __forceinline__ PagedRequest pg_lane(const PagedRequest& r, int l) {  // lane l's, for all
  return {__builtin_amdgcn_readlane(r.row0, l), __builtin_amdgcn_readlane(r.n, l),
          __builtin_amdgcn_readlane(r.len, l), __builtin_amdgcn_readlane(r.pos0, l)};
}

// Workgroup `wg` of `wgs`, of DW waves; `sRing`: DW * DSLOT * DSLOT_BYTES of LDS, `sLast` an int of it.
template <int DT, int ODT, int DW>
__device__ __forceinline__ void few_rows(const AttendParams& p, int wg, int wgs, uint8_t* sRing,
                                         int* sLast) {
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 15, g = lane >> 4;

  // tiles of a request's keys; 0 for one without rows or with too many
  auto tiles_of = [&](const PagedRequest& r) {
    if (r.n <= 0 || r.n * p.hpg > DROWS) return 0;
    return max(1, (r.len + DTILE - 1) / DTILE);
  };
  PagedRequest r;
  int b, kvh, part = 0, parts = 1, first = 0;
  if (p.split) {
    PagedRequest rs[D_SPLIT_B / 64];
    int t[D_SPLIT_B / 64], total = 0, units = 0;
    const int used = (p.B + 63) / 64;
#pragma unroll
    for (int j = 0; j < D_SPLIT_B / 64; ++j) {
      t[j] = 0;
      if (64 * j + lane < p.B) {
        rs[j] = paged_request(p.pool, p.q_start, p.lens, 64 * j + lane, p.T);
        t[j] = tiles_of(rs[j]);
      }
      total += t[j];
      units += t[j] > 0;
    }
    total = pg_wave_sum(total) * p.Hkv;
    units = pg_wave_sum(units) * p.Hkv;
    const int G = wgs;  // at least the units
    // Parts of size c; the same in every wave of the launch, whatever the rounding. At most 0.65
    // sqrt(tiles): a part costs its join what two tiles cost (one user of 8192 tokens: 15.6 us in 16
    // parts, 18.0 in 32; of 2048 tokens: 12.6 in 4, 11.5 in 8).
    auto parts_of = [&](int tiles, float inv) {
      const float most = 0.65f * __builtin_amdgcn_sqrtf((float)tiles) + 0.5f;
      return tiles > 0 ? max(1, (int)fminf((float)tiles * inv + 0.999f, most)) : 0;
    };
    // the least c lies between total / G (no rounding up) and total / (G - units) (each unit
    // rounded up by a whole part)
    float lo = max((float)total / (float)G, (float)D_MIN_TILES);
    float hi = G > units ? max((float)total / (float)(G - units), lo) : 1e9f;
    for (int it = 0; it < 6; ++it) {
      const float c = it == 0 ? lo : 0.5f * (lo + hi), inv = 1.0f / c;
      int sum = 0;
#pragma unroll
      for (int j = 0; j < D_SPLIT_B / 64; ++j)
        if (j < used) sum += parts_of(t[j], inv);
      if (pg_wave_sum(sum) * p.Hkv <= G) {
        hi = c;
        if (it == 0) break;
      } else {
        lo = c;
      }
    }
    float inv = 1.0f / hi;
    {  // hi may still be the untested bound
      int sum = 0;
#pragma unroll
      for (int j = 0; j < D_SPLIT_B / 64; ++j)
        if (j < used) sum += parts_of(t[j], inv);
      if (pg_wave_sum(sum) * p.Hkv > G) inv = 0.f;  // one part each
    }
    // this workgroup's place in the running sums
    int base = 0;
    b = -1;
#pragma unroll
    for (int j = 0; j < D_SPLIT_B / 64; ++j) {
      if (j >= used || b >= 0) continue;
      const int s = parts_of(t[j], inv) * p.Hkv;
      const int run = pg_wave_scan(s);
      const unsigned long long hit = __ballot(wg < base + run);
      if (hit) {
        const int l = __ffsll((long long)hit) - 1;
        b = 64 * j + l;
        first = base + __builtin_amdgcn_readlane(run - s, l);
        parts = quot(p.by_hkv, __builtin_amdgcn_readlane(s, l));
        r = pg_lane(rs[j], l);
      } else {
        base += __builtin_amdgcn_readlane(run, 63);
      }
    }
    b = __builtin_amdgcn_readfirstlane(b);
    if (b < 0) return;
    first = __builtin_amdgcn_readfirstlane(first);
    parts = __builtin_amdgcn_readfirstlane(parts);
    const int rel = wg - first;
    kvh = rel / parts;
    part = rel % parts;
    first += kvh * parts;
  } else {
    b = quot(p.by_hkv, wg);
    kvh = wg - b * p.Hkv;
    r = paged_request(p.pool, p.q_start, p.lens, b, p.T);
  }
  r = uniform(r);
  const int n_all = tiles_of(r);
  if (n_all == 0) return;
  const int rows = r.n * p.hpg;
  const int per = (n_all + parts - 1) / parts;
  const int t_begin = part * per, t_end = min(n_all, t_begin + per);
  const int n_iter = max(0, (t_end - t_begin - wave + DW - 1) / DW);
  auto tix = [&](int j) { return t_begin + wave + DW * j; };

  uint8_t* ring = sRing + wave * DSLOT * DSLOT_BYTES;
  uint32_t piece_off[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int t = 4 * i + (lane >> 4);
    piece_off[i] = (uint32_t)((lane >> 4) * 256 + 16 * ((lane & 15) ^ t));
  }
  int ids = -1;  // lane l: the page of the wave's tile l of the 64 being issued
  auto issue = [&](int j) {  // the tile's loads; returns its page (scalar)
    if (j >= n_iter) return -1;
    if ((j & 63) == 0) {
      const int t = tix(j + lane);
      ids = t < t_end ? paged_page(p.pool, b, t * DTILE) : -1;
    }
    const int page = __builtin_amdgcn_readlane(ids, j & 63), tok = tix(j) * DTILE;
    const long long at = (long long)max(page, 0) * p.pool.page_stride +
                         (long long)kvh * p.pool.head_stride +
                         (long long)(tok & (p.pool.page_size - 1)) * PG_DH;
    const uint32_t bytes = page < 0 ? 0u : (uint32_t)min(r.len - tok, DTILE) * (PG_DH * 2);
    const __amdgpu_buffer_rsrc_t rk = dkv_make_rsrc(p.k + at, bytes);
    const __amdgpu_buffer_rsrc_t rv = dkv_make_rsrc(p.v + at, bytes);
    const uint32_t slot = dkv_lds_addr(ring + (j % DSLOT) * DSLOT_BYTES);
    pg_lds_loads<true>(rk, slot, piece_off);
    pg_lds_loads<true>(rv, slot + DTILE_BYTES, piece_off);
    return page;
  };
  int page_next = issue(0);

  // query operand: column n = row n (new token n / hpg, head n % hpg; rows past the request's
  // zero), dims 32c + 8g .. +8
  dkv_u32x4 bq[4];
  const bool has = n < rows;
  const int qi = has ? quot(p.by_hpg, n) : 0;  // the row's new token
  const uint16_t* qr = p.q + (long long)(r.row0 + qi) * p.q_st +
                       (long long)(kvh * p.hpg + (has ? n - qi * p.hpg : 0)) * p.q_sh;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const dkv_u32x4 v = *(const dkv_u32x4*)(qr + 32 * c + 8 * g);
    bq[c] = has ? v : dkv_u32x4{0u, 0u, 0u, 0u};
  }
  // settled here (with tile 0), not inside the loop, where the wait would drain the next tile too
#pragma unroll
  for (int c = 0; c < 4; ++c) asm volatile("" : "+v"(bq[c]));
  const int limit = min(r.pos0 + qi, r.len - 1);  // the row's last key

  dkv_f32x4 acc[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = dkv_f32x4{0.f, 0.f, 0.f, 0.f};
  float m_run = PG_NO_MAX, l_run = 0.f;  // the row's reference (log2 units) and sum

  for (int j = 0; j < n_iter; ++j) {
    pg_wait_vm();
    const int page = page_next;
    page_next = issue(j + 1);
    const uint8_t* slot = ring + (j % DSLOT) * DSLOT_BYTES;
    const int key0 = tix(j) * DTILE;
    dkv_u32x4 xk[4];
#pragma unroll
    for (int c = 0; c < 4; ++c)
      xk[c] = *(const dkv_u32x4*)(slot + n * 256 + 16 * ((4 * c + g) ^ n));
    dkv_f32x4 sc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < 4; ++c) sc = dkv_mfma32<DT>(xk[c], bq[c], sc);
    // lane (row n, keys 4g + u): scores in log2 units
    const int last = page < 0 ? -1 : limit - key0 - 4 * g;
    float z[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) z[u] = u <= last ? sc[u] * p.scale_log2 : -INFINITY;
    float tmax = dkv_max3(dkv_max3(z[0], z[1], z[2]), z[3], z[3]);
    tmax = dkv_lane_max32(tmax);
    tmax = dkv_lane_max16(tmax);
    if (__ballot(tmax > m_run + (PG_BIAS<DT> + D_RESCALE<DT>))) {
      const float m_new = fmaxf(m_run, tmax - PG_BIAS<DT>);
      const float alpha = __builtin_amdgcn_exp2f(m_run - m_new);
      l_run *= alpha;
      m_run = m_new;
      float au[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) au[u] = __shfl(alpha, 4 * g + u, 64);
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int u = 0; u < 4; ++u) acc[i][u] *= au[u];
    }
    float pu[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      pu[u] = __builtin_amdgcn_exp2f(z[u] - m_run);
      l_run += pu[u];
    }
    // P.V: A = P (row n; its 16 tokens twice, as hi and lo parts: k = 8g + e is part e / 4 of token
    // 4g + e % 4), B = V (the token's value, column = dim 16 blk + n) read transposed: lane (n, g)
    // reads 8 bytes of token 4g + n / 4 and receives tokens 4g .. 4g + 3 of dim 16 blk + n
    dkv_u32x4 pa;
    if constexpr (DT == DKV_BF16) {
      uint32_t h01, h23, l01, l23;
      dkv_split_bf16x2(pu[0], pu[1], h01, l01);
      dkv_split_bf16x2(pu[2], pu[3], h23, l23);
      pa = dkv_u32x4{h01, h23, l01, l23};
    } else {
      float lo[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) lo[u] = pu[u] - (float)(_Float16)pu[u];
      pa = dkv_u32x4{dkv_pack_f16x2(pu[0], pu[1]), dkv_pack_f16x2(pu[2], pu[3]),
                     dkv_pack_f16x2(lo[0], lo[1]), dkv_pack_f16x2(lo[2], lo[3])};
    }
    const int vtok = 4 * g + (n >> 2);
    dkv_u32x2 xv[8];
#pragma unroll
    for (int blk = 0; blk < 8; ++blk) {
      const int piece = 2 * blk + ((n & 3) >> 1);
      xv[blk] = pg_read_tr(slot + DTILE_BYTES + vtok * 256 + 16 * (piece ^ vtok) + 8 * (n & 1));
    }
    if (key0 + DTILE - 1 <= r.pos0 || r.n == 1) {
#pragma unroll
      for (int blk = 0; blk < 8; ++blk)
        acc[blk] = dkv_mfma32<DT>(pa, dkv_u32x4{xv[blk].x, xv[blk].y, xv[blk].x, xv[blk].y},
                                  acc[blk]);
    } else {
      // Keys that some of the rows attend and others do not (they come after them): a product per
      // new token with the later keys' values cleared, of which its own rows are taken, so that an
      // infinity or NaN there, whose weight is 0, stays out of the rows before it.
      for (int i = 0; i < r.n; ++i) {
        const int cut = r.pos0 + i - key0 - 4 * g;  // the token's last key, from this lane's first
        const uint32_t m0 = (cut >= 0 ? 0xffffu : 0u) | (cut >= 1 ? 0xffff0000u : 0u);
        const uint32_t m1 = (cut >= 2 ? 0xffffu : 0u) | (cut >= 3 ? 0xffff0000u : 0u);
#pragma unroll
        for (int blk = 0; blk < 8; ++blk) {
          const uint32_t v0 = xv[blk].x & m0, v1 = xv[blk].y & m1;
          const dkv_f32x4 o = dkv_mfma32<DT>(pa, dkv_u32x4{v0, v1, v0, v1},
                                             dkv_f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int x = 4 * g + u - i * p.hpg;
            if (x >= 0 && x < p.hpg) acc[blk][u] += o[u];
          }
        }
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
  pg_wait_vm();  // nothing lands in the ring once it is reused below

  // ---- join the waves through LDS ----
  float l_tot = l_run;
  l_tot += __shfl_xor(l_tot, 16, 64);
  l_tot += __shfl_xor(l_tot, 32, 64);
  __syncthreads();
  float* sw = reinterpret_cast<float*>(sRing);  // per wave: 16 m, 16 l, 16 x 128 acc
  constexpr int WREC = 2 * DROWS + DROWS * PG_DH;
  static_assert(DW * WREC * 4 <= DW * DSLOT * DSLOT_BYTES, "the epilogue's floats fit the ring");
  float* my = sw + wave * WREC;
  if (g == 0) {
    my[n] = m_run;
    my[DROWS + n] = l_tot;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int u = 0; u < 4; ++u) my[2 * DROWS + (4 * g + u) * PG_DH + 16 * i + n] = acc[i][u];
  __syncthreads();
  auto joined = [&](int row, int d, float& M, float& L) {  // sum of dim d, with the row's M and L
    float mw[DW], A = 0.f;
    M = -INFINITY;
    L = 0.f;
#pragma unroll
    for (int w = 0; w < DW; ++w) {
      mw[w] = sw[w * WREC + row];
      M = fmaxf(M, mw[w]);
    }
#pragma unroll
    for (int w = 0; w < DW; ++w) {
      const float wt = exp2f(mw[w] - M);
      L += wt * sw[w * WREC + DROWS + row];
      A += wt * sw[w * WREC + 2 * DROWS + row * PG_DH + d];
    }
    return A;
  };
  auto store = [&](int row, int d, float A, float L) {
    const int i = quot(p.by_hpg, row);
    const long long oi = (long long)(r.row0 + i) * p.o_st +
                         (long long)((kvh - i) * p.hpg + row) * p.o_sh + d;
    dkv_store_f32<ODT>(p.out, oi, L == 0.f ? 0.f : A / L);  // (a NaN among the weights stays)
  };
  if (parts == 1) {
    for (int idx = tid; idx < rows * PG_DH; idx += 64 * DW) {
      float M, L;
      const float A = joined(idx / PG_DH, idx % PG_DH, M, L);
      store(idx / PG_DH, idx % PG_DH, A, L);
    }
    return;
  }
  // This part's record: per row m and l, then acc[128], as pairs (8-byte accesses that all XCDs see).
  auto put = [&](float* a, float x, float y) {
    __hip_atomic_store((unsigned long long*)a,
                       __float_as_uint(x) | ((unsigned long long)__float_as_uint(y) << 32),
                       __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  };
  float* rec = p.records + (long long)wg * DREC;
  for (int idx = tid; idx < rows * (PG_DH / 2); idx += 64 * DW) {
    const int row = idx / (PG_DH / 2), d = 2 * (idx % (PG_DH / 2));
    float M, L;
    const float x = joined(row, d, M, L), y = joined(row, d + 1, M, L);
    float* rr = rec + row * (PG_DH + 2);
    put(rr + 2 + d, x, y);
    if (d == 0) put(rr, M, L);
  }
  // ---- the unit's last part to arrive joins the parts ----
  pg_wait_vm();
  __syncthreads();
  if (tid == 0) {
    const int old = __hip_atomic_fetch_add(p.counters + b * p.Hkv + kvh, 1, __ATOMIC_RELAXED,
                                           __HIP_MEMORY_SCOPE_AGENT);
    *sLast = old == parts - 1;
  }
  __syncthreads();
  if (!*sLast) return;
  const float* recs = p.records + (long long)first * DREC;
  auto get = [&](const float* a) {
    return __hip_atomic_load((const unsigned long long*)a, __ATOMIC_RELAXED,
                             __HIP_MEMORY_SCOPE_AGENT);
  };
  constexpr int AHEAD = 8;  // parts whose loads are on their way together
  for (int idx = tid; idx < rows * (PG_DH / 2); idx += 64 * DW) {
    const int row = idx / (PG_DH / 2), d = 2 * (idx % (PG_DH / 2));
    float M = -INFINITY, L = 0.f, A0 = 0.f, A1 = 0.f;
    for (int s0 = 0; s0 < parts; s0 += AHEAD) {
      unsigned long long ml[AHEAD], xy[AHEAD];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        if (s0 + u >= parts) break;
        const float* rr = recs + (long long)(s0 + u) * DREC + row * (PG_DH + 2);
        ml[u] = get(rr);
        xy[u] = get(rr + 2 + d);
      }
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) {
        if (s0 + u >= parts) break;
        const float mu = __uint_as_float((uint32_t)ml[u]);
        const float Mn = fmaxf(M, mu);
        const float so = exp2f(M - Mn), sn = exp2f(mu - Mn);
        L = L * so + __uint_as_float((uint32_t)(ml[u] >> 32)) * sn;
        A0 = A0 * so + __uint_as_float((uint32_t)xy[u]) * sn;
        A1 = A1 * so + __uint_as_float((uint32_t)(xy[u] >> 32)) * sn;
        M = Mn;
      }
    }
    store(row, d, A0, L);
    store(row, d + 1, A1, L);
  }
  if (tid == 0) p.counters[b * p.Hkv + kvh] = 0;
}

template <int DT, int ODT>
__global__ __launch_bounds__(512, 2) void paged_few_kernel(AttendParams p) {
  __shared__ __attribute__((aligned(256))) uint8_t sRing[8 * DSLOT * DSLOT_BYTES];
  __shared__ int sLast;
  few_rows<DT, ODT, 8>(p, blockIdx.x, gridDim.x, sRing, &sLast);
}

// ---- many rows: prompts and their chunks ----
//
// A request's new tokens and a KV head's query heads make rows (token R / hpg, head R % hpg), so the
// heads that read the same keys share their tiles. One workgroup has BQ = 16 QB NW rows of one
// request and KV head (NW waves of QB blocks of 16 rows) and all the keys they attend, or, where
// there are few rows to fill the chip with, one of `splits` ranges of them (records joined by a
// second launch). Key tiles of 64 are staged in LDS (double-buffered, direct-to-LDS loads, 16-byte
// pieces XOR-swizzled by key so that the row reads of K do not meet in a bank; of the transposed reads of
// V those of keys 2i and 2i + 1 do, two cycles a read by SQ_LDS_BANK_CONFLICT); a tile is four blocks of 16 keys, each within one page, and a wave loads one of them
// (NW = 8: half of one) through a resource that ends with the request's keys. S^T = K Q^T on
// 16x16x32 MFMA (a lane then holds one row's scores for 16 keys); softmax in fp32, the running
// maximum raised only when a tile's exceeds it by more than 2^8 (fp16: 2^3); P V on 16x16x32 MFMA with
// the weights rounded once to the cache's type and summed as rounded: a weight is off by at most half a
// step (fp16: or 2^-37 of the row's largest, above), and a row, which its sum divides, by at most two half
// steps of sum p |v|; as the errors are of either sign, with the output's own rounding they come to 1.25
// to 1.4 times that alone (normal scores, measured against 64 bits; a second product with what the
// rounding left would take half as many products again, which are the prompts' bound).
//
// Bound by the SIMDs' issue slots: per wave and tile (QB = 2) 68 products of 16 cycles beside ~190
// vector instructions, 32 of them exponentials of 16 cycles; two waves a SIMD fill one's products with
// the other's vector work in part. Four prompts of 2048 tokens (32 and 8 heads): 158 us, 0.87 PFLOP/s
// (a workgroup's start and end are as long as three of its 17 tiles), one of 8192: 500 us, 1.10 PFLOP/s,
// where a large library product reaches 1.23. (Sums by additions and equal priorities: 2% more.) Key
// tiles of 32 and three waves a SIMD: the same at 8192, 10% slower on chunks. Deeper rings of tiles, the
// scores of the next tile among this one's softmax, K operands read before the next tile's loads: nothing.
constexpr int CK = 64;                      // keys per tile
constexpr int CTILE_BYTES = CK * PG_DH * 2;
template <int DT>                           // log2 units the running maximum may be exceeded by
constexpr float C_RESCALE = DT == DKV_F16 ? PG_F16_RESCALE : 8.f;

struct ChunkParams {
  AttendParams a;
  float* records;
  // rows of a workgroup and their log2; row tiles that have key ranges, and how many (further tiles
  // have one, and no record); rows up to which the other kernel works
  int bq, bq_shift, items, splits, few_rows;
  Divisor by_splits;
};

// The work item of a workgroup: row tile `rt` of request b. Items are counted request by request,
// a request's later rows (with more keys) first.
struct ChunkItem {
  int b, rt;  // b < 0: none
  PagedRequest r;
};
__device__ __forceinline__ ChunkItem chunk_item(const ChunkParams& p, int item, int lane) {
  const AttendParams& a = p.a;
  int base = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    int t = 0;
    PagedRequest r = {0, 0, 0, 0};
    if (b0 + lane < a.B) {
      r = paged_request(a.pool, a.q_start, a.lens, b0 + lane, a.T);
      const int rows = r.n * a.hpg;
      t = r.n > 0 && rows > p.few_rows ? (rows + p.bq - 1) >> p.bq_shift : 0;
    }
    const int run = pg_wave_scan(t);
    const unsigned long long hit = __ballot(item < base + run);
    if (hit) {
      const int l = __ffsll((long long)hit) - 1;
      ChunkItem it;
      it.b = b0 + l;
      it.rt = base + __builtin_amdgcn_readlane(run, l) - 1 - item;
      it.r = pg_lane(r, l);
      return it;
    }
    base += __builtin_amdgcn_readlane(run, 63);
  }
  return ChunkItem{-1, 0, {0, 0, 0, 0}};
}

// Four neighbouring values of the output, WIDE as one store.
template <int ODT, bool WIDE>
__device__ __forceinline__ void store4(const AttendParams& p, long long at, dkv_f32x4 v) {
  typedef __attribute__((ext_vector_type(2))) float f32x2;
  if constexpr (!WIDE) {
#pragma unroll
    for (int u = 0; u < 4; ++u) dkv_store_f32<ODT>(p.out, at + u, v[u]);
  } else if constexpr (ODT == DKV_F32) {
    *(dkv_f32x4*)((float*)p.out + at) = v;
  } else if constexpr (ODT == DKV_BF16) {
    *(dkv_u32x2*)((uint16_t*)p.out + at) = dkv_u32x2{
        __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{v[0], v[1]}, dkv_bf16x2)),
        __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{v[2], v[3]}, dkv_bf16x2))};
  } else {
    // (the quotient in fp32 first, as the fp32 output has it: not one instruction to fp16)
#pragma unroll
    for (int u = 0; u < 4; ++u) asm("" : "+v"(v[u]));
    *(dkv_u32x2*)((uint16_t*)p.out + at) =
        dkv_u32x2{dkv_pack_f16x2(v[0], v[1]), dkv_pack_f16x2(v[2], v[3])};
  }
}
// f(db) at dims 16 db + 0 .. 3 from `at` on, by wide stores where the output's rows allow it
template <int ODT, class F>
__device__ __forceinline__ void store_dims(const AttendParams& p, long long at, F&& f) {
  if (p.out_wide) {
#pragma unroll
    for (int db = 0; db < 8; ++db) store4<ODT, true>(p, at + 16 * db, f(db));
  } else {
#pragma unroll
    for (int db = 0; db < 8; ++db) store4<ODT, false>(p, at + 16 * db, f(db));
  }
}

__device__ __forceinline__ float pg_max4(float x) {  // over lanes n, n + 16, n + 32, n + 48
  return dkv_lane_max16(dkv_lane_max32(x));
}

// One row over keys k0 .. k1 - 1, by a wave, key by key: for rows whose values came out as infinity or
// NaN, or whose scores are too large for one fused multiplication and subtraction. A product of
// matrices takes a masked key's value times 0, which is NaN for an infinite one; here
// a masked key is not touched. Lane l returns dims 2l, 2l + 1. Slow, and for every row that attends such
// a value: one NaN in the first value of a KV head makes 512 tokens at 8192 take 16 ms (80 us without), a
// prompt of 2048 8.8 ms (59 us).
template <int DT>
__device__ __forceinline__ void attend_row_apart(const AttendParams& p, int b, int kvh,
                                              const uint16_t* qr, int k0, int k1, int lane,
                                              float& m, float& l, float& o0, float& o1) {
  m = PG_NO_MAX;
  l = o0 = o1 = 0.f;
  for (int t0 = k0; t0 < k1; t0 += 64) {
    const int key = t0 + lane;
    const int page = key < k1 ? paged_page(p.pool, b, key) : -1;
    const long long at = (long long)max(page, 0) * p.pool.page_stride +
                         (long long)kvh * p.pool.head_stride +
                         (long long)(key & (p.pool.page_size - 1)) * PG_DH;
    float s = -INFINITY;
    if (page >= 0) {
      s = 0.f;
      for (int d = 0; d < PG_DH; d += 8) {
        float kv[8], qv[8];
        load8<DT>(p.k + at + d, kv);
        load8<DT>(qr + d, qv);
#pragma unroll
        for (int e = 0; e < 8; ++e) s = fmaf(qv[e], kv[e], s);
      }
      s *= p.scale_log2;
    }
    const float mt = fmaxf(m, dkv_wave_max(s));
    const float alpha = exp2f(m - mt), w = page >= 0 ? exp2f(s - mt) : 0.f;
    l = l * alpha + dkv_wave_sum(w);
    o0 *= alpha;
    o1 *= alpha;
    m = mt;
    for (int j = 0; j < 64 && t0 + j < k1; ++j) {
      if (__builtin_amdgcn_readlane(page, j) < 0) continue;
      const float wj = __shfl(w, j, 64);
      const long long vj = __shfl(at, j, 64);
      o0 = fmaf(wj, dkv_load_f32<DT>(p.v + vj, 2 * lane), o0);
      o1 = fmaf(wj, dkv_load_f32<DT>(p.v + vj, 2 * lane + 1), o1);
    }
  }
}

// Workgroup `wg`; `sKV`: 4 * CTILE_BYTES of LDS, 1 KB aligned (the operand reads form their
// addresses by exclusive-or): two K tiles, two V tiles.
template <int DT, int ODT, int QB, int NW>
__device__ __forceinline__ void many_rows(const ChunkParams& c, int wg, uint8_t* sKV) {
  constexpr int QW = 16 * QB;            // rows per wave
  constexpr int BQ = NW * QW;            // rows per workgroup
  constexpr int LW = CK / 4 / NW;        // K (or V) loads per wave and tile, 4 keys each
  auto sK = [&](int i) { return sKV + i * CTILE_BYTES; };
  auto sV = [&](int i) { return sKV + (2 + i) * CTILE_BYTES; };
  const AttendParams& p = c.a;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, g = lane >> 4;
  // the KV head runs fastest: workgroups go to the 8 XCDs in turn, so that a head's keys and values
  // stay in one L2 (for 8 heads, or a multiple)
  const int rest = __builtin_amdgcn_readfirstlane(quot(p.by_hkv, wg));
  const int kvh = wg - rest * p.Hkv;
  const bool cut = rest < c.items * c.splits;
  const int splits = cut ? c.splits : 1;
  const int item = cut ? __builtin_amdgcn_readfirstlane(quot(c.by_splits, rest))
                       : rest - c.items * (c.splits - 1);
  const int split = cut ? rest - item * c.splits : 0;
  const ChunkItem it = chunk_item(c, item, lane);
  const int b = __builtin_amdgcn_readfirstlane(it.b);
  if (b < 0) return;
  const PagedRequest r = uniform(it.r);
  const int rows = r.n * p.hpg;
  const int q0 = __builtin_amdgcn_readfirstlane(it.rt) * BQ;
  const int wq0 = q0 + QW * wave;  // the wave's first row

  // keys up to the last row's; the wave's first and last row's limits
  const int k_end = __builtin_amdgcn_readfirstlane(
      max(0, min(r.len, r.pos0 + quot(p.by_hpg, min(q0 + BQ, rows) - 1) + 1)));
  const int w_first = r.pos0 + quot(p.by_hpg, min(wq0, rows - 1));
  const int w_end = wq0 < rows ? r.pos0 + quot(p.by_hpg, min(wq0 + QW, rows) - 1) + 1 : 0;
  const int all_tiles = (k_end + CK - 1) / CK;
  const int per = cut ? quot(c.by_splits, all_tiles + c.splits - 1) : all_tiles;
  const int t0 = min(all_tiles, split * per), n_tiles = min(all_tiles, t0 + per);

  // pages of the 64 blocks of 16 keys from tile tb on (16 tiles); the next 64 fetched ahead
  int ids = -1, ids_next = -1;
  auto fetch_ids = [&](int tb) {
    const int key = (tb * 4 + lane) * 16;
    return key < k_end ? paged_page(p.pool, b, key) : -1;
  };
  int ids_base = t0;
  ids = fetch_ids(t0);  // (before the queries, which the first tiles' loads need not wait for)
  if (t0 + 16 < n_tiles) ids_next = fetch_ids(t0 + 16);
  // this lane's rows (operand columns): token and last key
  dkv_u32x4 qop[QB][4];
  int limit[QB];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    const int R = min(wq0 + 16 * qb + n, rows - 1);
    const int i = quot(p.by_hpg, R), h = R - i * p.hpg;
    const uint16_t* qp = p.q + (long long)(r.row0 + i) * p.q_st +
                         (long long)(kvh * p.hpg + h) * p.q_sh + 8 * g;
#pragma unroll
    for (int s = 0; s < 4; ++s) qop[qb][s] = *(const dkv_u32x4*)(qp + 32 * s);
    limit[qb] = min(r.pos0 + i, r.len - 1);
  }
  // blocks with keys but no page
  auto absent_of = [&](int tb) {
    return __ballot(ids < 0 && (tb * 4 + lane) * 16 < k_end);
  };
  unsigned long long absent = absent_of(t0);

  // tile loads: wave w, instruction i stores keys 64 / NW * w + 4 i + lane / 16 of the tile, LDS piece
  // lane % 16, which holds the key's 16-byte piece (lane % 16) ^ (key % 16)
  const int blk = wave * (CK / NW) / 16;              // the wave's block of the tile
  const int sub = (wave * (CK / NW)) & 15;            // its first key in the block
  uint32_t voff[LW];
#pragma unroll
  for (int i = 0; i < LW; ++i) {
    const int kk = 4 * i + (lane >> 4);
    voff[i] = (uint32_t)((lane >> 4) * 256 + 16 * ((lane & 15) ^ ((sub + kk) & 15)));
  }
  const uint16_t* k_head = p.k + (long long)kvh * p.pool.head_stride;
  const uint16_t* v_head = p.v + (long long)kvh * p.pool.head_stride;
  const int key_in_tile = blk * 16 + sub, slot_mask = p.pool.page_size - 1;
  auto issue = [&](int t, int page) {  // (scalar work, a wave's by itself: every instruction counts)
    const int key = t * CK + key_in_tile;
    const long long at = (long long)max(page, 0) * p.pool.page_stride +
                         (long long)((key & slot_mask) * PG_DH);
    int keys;  // as scalar instructions: the compiler would clamp in a vector register
    asm("s_max_i32 %0, %1, 0" : "=s"(keys) : "s"(k_end - key) : "scc");
    asm("s_min_i32 %0, %1, %2" : "=s"(keys) : "s"(keys), "n"(CK / NW) : "scc");
    const uint32_t bytes = page < 0 ? 0u : (uint32_t)keys * (PG_DH * 2);
    pg_lds_loads<false>(dkv_make_rsrc(k_head + at, bytes),
                        dkv_lds_addr(sK(t & 1)) + CK / NW * wave * 256, voff);
    pg_lds_loads<false>(dkv_make_rsrc(v_head + at, bytes),
                        dkv_lds_addr(sV(t & 1)) + CK / NW * wave * 256, voff);
  };

  dkv_f32x4 acc[QB][8];
#pragma unroll
  for (int qb = 0; qb < QB; ++qb)
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[qb][i] = dkv_f32x4{0.f, 0.f, 0.f, 0.f};
  // the rows' references (log2 units), and the sums of the weights as one more row of P V: a product
  // with ones, of the weights as they were rounded (every element holds it)
  float m_run[QB];
  dkv_f32x4 sum[QB];
  constexpr uint32_t one2 = DT == DKV_BF16 ? 0x3f803f80u : 0x3c003c00u;
  const dkv_u32x4 ones = {one2, one2, one2, one2};
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    m_run[qb] = PG_NO_MAX;
    sum[qb] = dkv_f32x4{0.f, 0.f, 0.f, 0.f};
  }

  // S^T of key block kb: A = K rows (lane: key 16kb + n, dims 32s + 8g .. +8), B = Q^T; lane (row n,
  // g) then holds keys 16kb + 4g + u, unscaled
  const uint32_t krd = n * 256 + 16 * (g ^ n);
  typedef __attribute__((address_space(3))) dkv_u32x4 lds_u32x4;
  // transposed V reads: lane 4i + q of each 16 reads key 16kb + 4g + i, dims 16db + 4q .. +3; lane i
  // then holds dim 16db + i of keys 4g .. 4g + 3
  const uint32_t vrd =
      (4 * g + (n >> 2)) * 256 + 16 * (((n & 3) >> 1) ^ (4 * g + (n >> 2))) + 8 * (n & 1);

  if (t0 < n_tiles) issue(t0, __builtin_amdgcn_readlane(ids, blk));
  // settled here, not inside the loop, where the compiler's waits for them would be waits for the next
  // tile, which it does not know of
#pragma unroll
  for (int qb = 0; qb < QB; ++qb)
#pragma unroll
    for (int s = 0; s < 4; ++s) asm volatile("" : "+v"(qop[qb][s]));
  for (int t = t0; t < n_tiles; ++t) {
    pg_wait_vm();
    __syncthreads();  // tile t is in LDS for every wave; tile t - 1's buffer is free
    const uint32_t gone = (uint32_t)(absent >> (4 * (t - ids_base))) & 15u;
    if (t + 1 < n_tiles) {
      if (t + 1 == ids_base + 16) {
        ids_base += 16;
        ids = ids_next;
        absent = absent_of(ids_base);
        if (ids_base + 16 < n_tiles) ids_next = fetch_ids(ids_base + 16);
      }
      issue(t + 1, __builtin_amdgcn_readlane(ids, 4 * (t + 1 - ids_base) + blk));
    }
    const int key0 = t * CK;
    if (key0 >= w_end) continue;  // every key of the tile is past the wave's rows
    const uint32_t kt = dkv_lds_addr(sK(t & 1));
    const uint32_t vt = dkv_lds_addr(sV(t & 1)) + vrd;
    dkv_f32x4 z[QB][4];
    __builtin_amdgcn_s_setprio(1);  // (the SIMD's other wave has its vector work meanwhile)
#pragma unroll
    for (int kb = 0; kb < 4; ++kb) {
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) z[qb][kb] = dkv_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const dkv_u32x4 a = *(const lds_u32x4*)(((kt + krd) ^ (64 * s)) + 4096 * kb);
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) z[qb][kb] = dkv_mfma32<DT>(a, qop[qb][s], z[qb][kb]);
      }
    }
    __builtin_amdgcn_s_setprio(0);
    if (key0 + CK - 1 > w_first || key0 + CK > r.len || gone) {
#pragma unroll
      for (int qb = 0; qb < QB; ++qb)
#pragma unroll
        for (int kb = 0; kb < 4; ++kb) {
          const int last = (gone >> kb) & 1u ? -1 : limit[qb] - key0 - 16 * kb - 4 * g;
#pragma unroll
          for (int u = 0; u < 4; ++u)
            if (u > last) z[qb][kb][u] = -INFINITY;
        }
    }
    // V operands of key blocks 0 and 1: read ahead of the softmax
    dkv_u32x2 vx[8][2];
    auto vread = [&](int j, int db) {
      const uint32_t src = (vt ^ (32 * db)) + 8192 * j;
#pragma unroll
      for (int kk = 0; kk < 2; ++kk)
        vx[db][kk] = __builtin_bit_cast(
            dkv_u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((pg_lds_i16x4*)(src + 4096 * kk)));
    };
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int db = 0; db < 8; ++db) vread(0, db);
    __builtin_amdgcn_sched_barrier(0);
    float tmax[QB];
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      float m[4];
#pragma unroll
      for (int kb = 0; kb < 4; ++kb)
        m[kb] = dkv_max3(dkv_max3(z[qb][kb][0], z[qb][kb][1], z[qb][kb][2]), z[qb][kb][3],
                         z[qb][kb][3]);
      tmax[qb] = pg_max4(dkv_max3(dkv_max3(m[0], m[1], m[2]), m[3], m[3])) * p.scale_log2;
    }
    constexpr float RAISE = PG_BIAS<DT> + C_RESCALE<DT>;
    if (__ballot(tmax[0] > m_run[0] + RAISE || tmax[QB - 1] > m_run[QB - 1] + RAISE)) {
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) {
        const float m_new = dkv_max2(m_run[qb], tmax[qb] - PG_BIAS<DT>);
        const float alpha = __builtin_amdgcn_exp2f(m_run[qb] - m_new);
        m_run[qb] = m_new;
#pragma unroll
        for (int u = 0; u < 4; ++u) sum[qb][u] *= alpha;
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int u = 0; u < 4; ++u) acc[qb][i][u] *= alpha;
      }
    }
    // P of key blocks 2j and 2j + 1: the products' k = 8g .. 8g + 3 are key block 2j's keys 4g .. 4g
    // + 3, k = 8g + 4 .. 8g + 7 key block 2j + 1's
    dkv_u32x4 bp[2][QB];
    auto probs = [&](int j, int kk, int qb) {
      float pu[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        pu[u] = __builtin_amdgcn_exp2f(
            __builtin_fmaf(z[qb][2 * j + kk][u], p.scale_log2, -m_run[qb]));
      }
      typedef __attribute__((ext_vector_type(2))) float f32x2;
      if constexpr (DT == DKV_BF16) {
        bp[j][qb][2 * kk] = __builtin_bit_cast(
            uint32_t, __builtin_convertvector(f32x2{pu[0], pu[1]}, dkv_bf16x2));
        bp[j][qb][2 * kk + 1] = __builtin_bit_cast(
            uint32_t, __builtin_convertvector(f32x2{pu[2], pu[3]}, dkv_bf16x2));
      } else {
        bp[j][qb][2 * kk] = dkv_pack_f16x2(pu[0], pu[1]);
        bp[j][qb][2 * kk + 1] = dkv_pack_f16x2(pu[2], pu[3]);
      }
    };
#pragma unroll
    for (int i = 0; i < 2 * QB; ++i) probs(0, i & 1, i >> 1);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int db = 0; db < 8; ++db) {
        __builtin_amdgcn_sched_barrier(0);
        const dkv_u32x4 aop = {vx[db][0].x, vx[db][0].y, vx[db][1].x, vx[db][1].y};
        if (j == 0) vread(1, db);
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) acc[qb][db] = dkv_mfma32<DT>(aop, bp[j][qb], acc[qb][db]);
        if (db == 7) {
#pragma unroll
          for (int qb = 0; qb < QB; ++qb) sum[qb] = dkv_mfma32<DT>(ones, bp[j][qb], sum[qb]);
        }
        if (j == 0 && db % (4 / QB) == 4 / QB - 1)
          probs(1, db / (4 / QB) % 2, db / (8 / QB));
      }
    }
  }

  // acc rows are dims, columns rows of the request: lane (row n, g) holds dims 16db + 4g + u. A
  // range's record: acc[BQ][128], then m and l of each row.
  float* rec = c.records + ((long long)(item * p.Hkv + kvh) * c.splits + split) * BQ *
                               (PG_DH + 2);
#pragma unroll
  for (int qb = 0; qb < QB; ++qb) {
    const float l = sum[qb][0];
    const int R = wq0 + 16 * qb + n;
    const int i = quot(p.by_hpg, R), h = R - i * p.hpg;
    // 0, or NaN where a value is infinite or NaN
    float od[4] = {l * 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int db = 0; db < 8; ++db)
#pragma unroll
      for (int u = 0; u < 4; ++u) od[u] = fmaf(acc[qb][db][u], 0.f, od[u]);
    const float odd = (od[0] + od[1]) + (od[2] + od[3]);
    // (Or a sum below that of the largest score's weight alone, which is at least 2^PG_BIAS as rounded:
    // scores past 2^24, whose product with the scale and the rounded maximum differ by more than their sum.)
    constexpr float LOW = DT == DKV_F16 ? 2048.f : 0.5f;  // half of it
    static_assert(PG_BIAS<DKV_F16> == 12.f && PG_BIAS<DKV_BF16> == 0.f, "");
    const bool low = l < LOW && min(limit[qb] + 1, n_tiles * CK) > t0 * CK;
    unsigned long long bad = __ballot(R < rows && (!(odd == 0.f) || low));
    bad = (bad | (bad >> 16) | (bad >> 32) | (bad >> 48)) & 0xffffull;  // by row
    const bool good = R < rows && !((bad >> n) & 1);
    if (splits == 1) {
      if (good) {
        const float inv = l > 0.f ? 1.f / l : 0.f;
        const long long ob = (long long)(r.row0 + i) * p.o_st +
                             (long long)(kvh * p.hpg + h) * p.o_sh;
        store_dims<ODT>(p, ob + 4 * g, [&](int db) { return acc[qb][db] * inv; });
      }
    } else if (good) {
      const int x = QW * wave + 16 * qb + n;
      if (g == 0) *(float2*)(rec + BQ * PG_DH + 2 * x) = float2{m_run[qb], l};
#pragma unroll
      for (int db = 0; db < 8; ++db)
        *(dkv_f32x4*)(rec + x * PG_DH + 16 * db + 4 * g) = acc[qb][db];
    }
    while (bad) {  // key by key
      const int x = __ffsll((long long)bad) - 1;
      bad &= bad - 1;
      const int Rx = wq0 + 16 * qb + x, ix = quot(p.by_hpg, Rx), hx = Rx - ix * p.hpg;
      const uint16_t* qx = p.q + (long long)(r.row0 + ix) * p.q_st +
                           (long long)(kvh * p.hpg + hx) * p.q_sh;
      float mx, lx, o0, o1;
      attend_row_apart<DT>(p, b, kvh, qx, t0 * CK, min(n_tiles * CK, min(r.pos0 + ix + 1, r.len)),
                           lane, mx, lx, o0, o1);
      if (splits == 1) {
        const float inv = lx > 0.f ? 1.f / lx : (lx == 0.f ? 0.f : lx);
        const long long ob = (long long)(r.row0 + ix) * p.o_st +
                             (long long)(kvh * p.hpg + hx) * p.o_sh + 2 * lane;
        dkv_store_f32<ODT>(p.out, ob, o0 * inv);
        dkv_store_f32<ODT>(p.out, ob + 1, o1 * inv);
      } else {
        const int y = QW * wave + 16 * qb + x;
        if (lane == 0) *(float2*)(rec + BQ * PG_DH + 2 * y) = float2{mx, lx};
        *(float2*)(rec + y * PG_DH + 2 * lane) = float2{o0, o1};
      }
    }
  }
}

template <int DT, int ODT, int QB, int NW>
__global__ __launch_bounds__(64 * NW, NW == 8 ? 4 : 2) void paged_chunk_kernel(ChunkParams c) {
  __shared__ __attribute__((aligned(1024))) uint8_t sKV[4 * CTILE_BYTES];
  many_rows<DT, ODT, QB, NW>(c, blockIdx.x, sKV);
}

// Both kinds of requests in one launch: the ones of few rows, bound by memory, beside the others,
// bound by their products. Workgroups of the two kinds are handed out in turn, so that a CU has one of
// each.
template <int DT, int ODT, int QB>
__global__ __launch_bounds__(256, 2) void paged_mixed_kernel(ChunkParams c, int few, int many) {
  static_assert(4 * DSLOT * DSLOT_BYTES <= 4 * CTILE_BYTES, "one workgroup shape");
  __shared__ __attribute__((aligned(1024))) uint8_t smem[4 * CTILE_BYTES];
  __shared__ int sLast;
  const int x = blockIdx.x, both = 2 * min(few, many);
  const int i = x < both ? x >> 1 : x - both / 2;
  if (x < both ? (x & 1) == 0 : few > many)
    few_rows<DT, ODT, 4>(c.a, i, few, smem, &sLast);
  else
    many_rows<DT, ODT, QB, 4>(c, i, smem);
}

// The key ranges' records of a row joined: 32 rows per workgroup, 8 threads of 16 dims each.
template <int DT, int ODT>
__global__ __launch_bounds__(256) void paged_join_kernel(ChunkParams c) {
  const AttendParams& p = c.a;
  const int groups = c.bq / 32;  // workgroups per (item, KV head)
  const int ik = blockIdx.x / groups;
  const int row = blockIdx.x % groups * 32 + (threadIdx.x >> 3), d0 = 4 * (threadIdx.x & 7);
  const float* rec = c.records + (long long)ik * c.splits * c.bq * (PG_DH + 2);
  const long long step = (long long)c.bq * (PG_DH + 2);
  const int kvh = ik % p.Hkv;
  const ChunkItem it = chunk_item(c, ik / p.Hkv, threadIdx.x & 63);
  if (it.b < 0) return;
  const PagedRequest& r = it.r;
  const int R = it.rt * c.bq + row;
  if (R >= r.n * p.hpg) return;
  float M = PG_NO_MAX, L = 0.f;
  dkv_f32x4 a[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) a[q] = dkv_f32x4{0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < c.splits; ++s) {
    const float2 ml = *(const float2*)(rec + s * step + c.bq * PG_DH + 2 * row);
    dkv_f32x4 x[4];
#pragma unroll
    for (int q = 0; q < 4; ++q)
      x[q] = *(const dkv_f32x4*)(rec + s * step + row * PG_DH + 32 * q + d0);
    if (ml.y == 0.f) continue;  // a range without keys for the row
    const float Mn = fmaxf(M, ml.x), so = exp2f(M - Mn), sn = exp2f(ml.x - Mn);
    M = Mn;
    L = L * so + ml.y * sn;
#pragma unroll
    for (int q = 0; q < 4; ++q) a[q] = a[q] * so + x[q] * sn;
  }
  const float inv = L > 0.f ? 1.f / L : (L == 0.f ? 0.f : L);
  const int i = quot(p.by_hpg, R), h = R - i * p.hpg;
  const long long ob = (long long)(r.row0 + i) * p.o_st +
                       (long long)(kvh * p.hpg + h) * p.o_sh + d0;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    if (p.out_wide)
      store4<ODT, true>(p, ob + 32 * q, a[q] * inv);
    else
      store4<ODT, false>(p, ob + 32 * q, a[q] * inv);
  }
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// T x H segments of `len` bytes, segment (i, h) at `at` + i st + h sh; a stride of a size of one is any.
struct Segments {
  long long at, st, sh, len;
  int T, H;
  long long end() const { return at + (T - 1) * st + (H - 1) * sh + len; }
};
// Whether a segment of a and one of b, of the same strides, have a byte in common (of one array with
// itself: two of its segments).
bool segments_meet(const Segments& a, const Segments& b, bool itself = false) {
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
bool output_apart(const Segments& out, const Segments& in, bool in_place) {
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

int fill_pool(PagedPool& pool, long long page_stride, long long head_stride, int num_pages,
              int page_size, const int* table, long long table_ld, int cols, int Hkv) {
  if (num_pages < 0 || cols < 0 || table_ld < cols) return DKV_E_ARG;
  if (page_size < 16 || (page_size & (page_size - 1))) return DKV_E_UNSUPPORTED;
  if (head_stride < (long long)page_size * PG_DH && Hkv > 1) return DKV_E_ARG;
  if (page_stride < 0 || head_stride < 0) return DKV_E_ARG;
  if ((page_stride & 7) || (head_stride & 7)) return DKV_E_UNSUPPORTED;
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

extern "C" int dkv_paged_append(void* stream, int dtype, const void* qkv, long long qkv_ld,
                                void* q_out, long long q_st, long long q_sh, void* k_pages,
                                void* v_pages, long long page_stride, long long head_stride,
                                int num_pages, int page_size, const int* page_table,
                                long long table_ld, int table_cols, const int* q_start,
                                const int* lens, int B, int T, int Hq, int Hkv, int Dh,
                                const void* q_norm, const void* k_norm, float eps,
                                const double* inv_freq) {
  if (dtype != DKV_F16 && dtype != DKV_BF16) return DKV_E_UNSUPPORTED;
  if (B < 0 || T < 0 || Hq <= 0 || Hkv <= 0) return DKV_E_ARG;
  if (Dh != PG_DH || Hq % Hkv != 0) return DKV_E_UNSUPPORTED;
  AppendParams p;
  const int rc = fill_pool(p.pool, page_stride, head_stride, num_pages, page_size, page_table,
                           table_ld, table_cols, Hkv);
  if (rc != DKV_OK) return rc;
  if (B == 0 || T == 0) return DKV_OK;
  if (!qkv || !q_out || !k_pages || !v_pages || !q_start || !lens || !inv_freq) return DKV_E_ARG;
  if (qkv_ld < (long long)(Hq + 2 * Hkv) * PG_DH || q_sh < PG_DH || q_st < PG_DH) return DKV_E_ARG;
  const bool in_place =
      qkv == q_out && (T == 1 || q_st == qkv_ld) && (Hq == 1 || q_sh == PG_DH);
  if (!output_apart({(long long)(uintptr_t)q_out, 2 * q_st, 2 * q_sh, 2 * PG_DH, T, Hq},
                    {(long long)(uintptr_t)qkv, 2 * qkv_ld, 0,
                     2LL * (Hq + 2 * Hkv) * PG_DH, T, 1},
                    in_place))
    return DKV_E_ARG;
  if (!aligned16(qkv) || !aligned16(q_out) || !aligned16(k_pages) || !aligned16(v_pages) ||
      (qkv_ld & 7) || (q_st & 7) || (q_sh & 7) || (q_norm && !aligned16(q_norm)) ||
      (k_norm && !aligned16(k_norm)))
    return DKV_E_UNSUPPORTED;
  p.qkv = (const uint16_t*)qkv;
  p.qkv_ld = qkv_ld;
  p.q_out = (uint16_t*)q_out;
  p.q_st = q_st;
  p.q_sh = q_sh;
  p.k = (uint16_t*)k_pages;
  p.v = (uint16_t*)v_pages;
  p.q_start = q_start;
  p.lens = lens;
  p.B = B;
  p.T = T;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.q_norm = (const uint16_t*)q_norm;
  p.k_norm = (const uint16_t*)k_norm;
  p.eps = eps;
  for (int j = 0; j < PG_DH / 2; ++j) p.rev[j] = inv_freq[j] * 0.15915494309189533577;
  const long long items = (long long)T * ((Hq + 2 * Hkv + 7) / 8);
  const long long wgs = (items + AP_WAVES - 1) / AP_WAVES;
  if (wgs > 0x7fffffffLL) return DKV_E_UNSUPPORTED;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == DKV_BF16)
    hipLaunchKernelGGL(paged_append_kernel<DKV_BF16>, dim3((unsigned)wgs), dim3(64 * AP_WAVES), 0,
                       st, p);
  else
    hipLaunchKernelGGL(paged_append_kernel<DKV_F16>, dim3((unsigned)wgs), dim3(64 * AP_WAVES), 0,
                       st, p);
  DKV_HIP_CHECK_LAUNCH();
  return DKV_OK;
}

namespace {

// The launches of a call, from its bounds alone.
struct AttendPlan {
  bool few, many;          // kernels that run
  int few_wgs, few_split;
  int qb, nw, bq, splits;
  int items, more;         // row tiles cut into key ranges, and further ones that are not
  long long many_at;       // the many-row kind's records, in floats from the others'
  long long floats;        // workspace (0: none)
};

// The shape of the many-row kernel, by the workgroups that the rows fill (rows that the host counts
// as if requests' tiles were full; 512 workgroups fit the chip at a time, 256 of 8 waves), and the key
// tiles of the longest request. us on MI355X, bf16, 32 query and 8 KV heads; shape: row blocks x
// waves / key ranges (workgroups):
//  * more than 1024 of 128 rows: 2x4, each key operand read from LDS serves two products. Four
//    2048-token prompts 158 2x4/1, 167 1x8/1, 188 1x4/1.
//  * up to 256 of 128 rows and long keys: ranges that fill the chip once, at least 24 tiles each.
//    512 tokens at 8192: 77.7 2x4/4 (512), 87 2x4/3, 89.4 1x4/2, 125 1x4/1. 846 tokens of two
//    requests at up to 6001: 87.3 2x4/2, 89.4 2x4/4, 101 1x4/1.
//  * so few rows that 64-row tiles, too, leave half the chip idle: those, ranges of 8 tiles or more.
//    64 tokens at 32768: 61.9 1x4/16, 65.1 2x4/16. 200 at 2000: 26.7 1x4/4, 27.5 1x4/2, 31.7 1x4/5
//    (520).
//  * otherwise one range: above 256 of 128 rows 1x8 (eight 300-token prompts 22.7, against 23.5 1x4,
//    25.5 2x4), else 1x4 (512 tokens at 1024: 20.1, against 24.4 1x8 and 29 2x4/2: a range more
//    costs its records, 66 KB a workgroup, written and read).
AttendPlan attend_plan(int B, int T, int Hq, int Hkv, int max_new, int min_new, int max_len) {
  AttendPlan a = {};
  const int hpg = Hq / Hkv;
  const long long units = (long long)B * Hkv;
  a.few = (long long)(min_new > 1 ? min_new : 1) * hpg <= DROWS;
  long long floats = 0;
  a.many = (long long)max_new * hpg > DROWS;
  if (a.few) {
    const long long tiles = ((long long)max_len + DTILE - 1) / DTILE;
    const long long most = units * ((tiles + D_MIN_TILES - 1) / D_MIN_TILES);
    long long wgs = units;
    if (wgs < D_WGS) wgs = most < D_WGS ? (most > units ? most : units) : D_WGS;
    a.few_split = wgs > units;
    a.few_wgs = (int)wgs;
    if (a.few_split) floats = wgs * DREC;
  }
  if (a.many) {
    auto items = [&](int bq) {  // sum over requests of ceil(rows / bq), at most
      const long long rows = (long long)T * hpg, each = ((long long)max_new * hpg + bq - 1) / bq;
      const long long x = rows / bq + B, y = each * B;
      return x < y ? x : y;
    };
    const long long tiles = ((long long)max_len + CK - 1) / CK;
    auto full = [&](int bq) {  // workgroups of full tiles
      const long long x = ((long long)T * hpg + bq - 1) / bq, y = items(bq);
      return (x < y ? x : y) * Hkv;
    };
    const long long wg128 = full(128), wg64 = full(64);
    auto ranges = [&](long long wgs, long long least) {
      // (beside the other kind, about half the chip: 12 single tokens and 512 at 2048, 16 and 4
      // heads: 30 us with two ranges; 42 with one or three and 49 in a launch of its own, where two
      // took 34. How many workgroups the other kind has does not count: 512 at 8192 beside one token,
      // or with a least number of new tokens that allows one, 128 us, alone 80)
      const long long n = a.few ? (256 + wgs / 2) / wgs : 512 / wgs, most = (tiles + least / 2) / least;
      return (int)(n < most ? n : most);
    };
    a.splits = 1;
    if (wg128 > 1024) {
      a.qb = 2, a.nw = 4;
    } else if (wg64 >= 256 && wg128 <= 256 && ranges(wg128, 24) > 1) {
      a.qb = 2, a.nw = 4, a.splits = ranges(wg128, 24);
    } else if (wg64 < 256 && ranges(wg64, 8) > 1) {
      a.qb = 1, a.nw = 4, a.splits = ranges(wg64, 8);
    } else {
      a.qb = 1, a.nw = wg128 > 256 && !a.few ? 8 : 4;
    }
    a.bq = 16 * a.qb * a.nw;
    a.items = (int)items(a.bq);
    if (a.splits > 1) {  // its records behind the other kind's
      // Of tiles that requests of min_new tokens (and more rows than the other kind's) can have: a step's
      // other requests have no token. The tiles that only a step which breaks min_new has come after them.
      const long long least = a.few ? DROWS / hpg + 1 : min_new;
      const long long n = T / least < B ? (T >= least ? T / least : 1) : B;
      const long long x = (long long)T * hpg / a.bq + n;
      const long long y = ((long long)max_new * hpg + a.bq - 1) / a.bq * n;
      const int all = a.items;
      a.items = (int)(x < y ? x : y);
      a.more = all - a.items;
      a.many_at = (floats + 3) / 4 * 4;
      floats = a.many_at + (long long)a.items * Hkv * a.splits * a.bq * (PG_DH + 2);
    }
  }
  a.floats = floats ? D_COUNTERS + floats : 0;
  return a;
}

// The lock of a workspace, under which every call that has one makes its launches: of two, the second
// reads what the first left, and threads may make calls on one stream, in whose workspace they follow
// each other.
std::mutex& launch_lock(const void* workspace) {
  static std::mutex locks[16];
  return locks[((uintptr_t)workspace >> 9) % 16];
}

template <int DT, int ODT>
void launch_attend(const AttendPlan& a, const ChunkParams& c, hipStream_t st) {
  const int many = (a.items * a.splits + a.more) * c.a.Hkv;
  std::unique_lock<std::mutex> together(launch_lock(c.a.counters), std::defer_lock);
  if (a.floats > 0) together.lock();
  if (a.few && a.many) {
    const dim3 grid((unsigned)(a.few_wgs + many));
    if (a.qb == 2)
      hipLaunchKernelGGL((paged_mixed_kernel<DT, ODT, 2>), grid, dim3(256), 0, st, c, a.few_wgs,
                         many);
    else
      hipLaunchKernelGGL((paged_mixed_kernel<DT, ODT, 1>), grid, dim3(256), 0, st, c, a.few_wgs,
                         many);
  } else if (a.few) {
    hipLaunchKernelGGL((paged_few_kernel<DT, ODT>), dim3((unsigned)a.few_wgs), dim3(512), 0, st, c.a);
  } else {
    const dim3 grid((unsigned)many);
    if (a.qb == 2)
      hipLaunchKernelGGL((paged_chunk_kernel<DT, ODT, 2, 4>), grid, dim3(256), 0, st, c);
    else if (a.nw == 8)
      hipLaunchKernelGGL((paged_chunk_kernel<DT, ODT, 1, 8>), grid, dim3(512), 0, st, c);
    else
      hipLaunchKernelGGL((paged_chunk_kernel<DT, ODT, 1, 4>), grid, dim3(256), 0, st, c);
  }
  if (a.many && a.splits > 1)
    hipLaunchKernelGGL((paged_join_kernel<DT, ODT>),
                       dim3((unsigned)(a.items * c.a.Hkv * (a.bq / 32))), dim3(256), 0, st, c);
}

bool attend_sizes_ok(int B, int T, int Hq, int Hkv, int max_new) {
  // rows and work items are counted in 32 bits
  return (long long)T * (Hq / Hkv) + 4096 < 0x7fffffffLL &&
         (long long)max_new * (Hq / Hkv) + 4096 < 0x7fffffffLL &&
         (((long long)T * (Hq / Hkv)) / 64 + B) * Hkv * 32 < 0x7fffffffLL;
}

}  // namespace

extern "C" long long dkv_paged_workspace_floats(int B, int T, int Hq, int Hkv, int max_new,
                                                int min_new, int max_len) {
  if (B <= 0 || T <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || max_new <= 0 || max_len < 0)
    return 0;
  if (!attend_sizes_ok(B, T, Hq, Hkv, max_new)) return 0;
  return attend_plan(B, T, Hq, Hkv, max_new, min_new, max_len).floats;
}

extern "C" int dkv_paged_attention(void* stream, int dtype, const void* q, long long q_st,
                                   long long q_sh, const void* k_pages, const void* v_pages,
                                   long long page_stride, long long head_stride, int num_pages,
                                   int page_size, const int* page_table, long long table_ld,
                                   int table_cols, const int* q_start, const int* lens, int B,
                                   int T, int Hq, int Hkv, int Dh, int max_new, int min_new,
                                   int max_len, float scale, float* workspace,
                                   long long workspace_floats, void* out, int out_dtype,
                                   long long o_st, long long o_sh) {
  if (!(scale > 0.f) || !(scale * 1.4426950408889634f < INFINITY)) return DKV_E_UNSUPPORTED;
  if (dtype != DKV_F16 && dtype != DKV_BF16) return DKV_E_UNSUPPORTED;
  if (out_dtype != dtype && out_dtype != DKV_F32) return DKV_E_ARG;
  if (B < 0 || T < 0 || Hq <= 0 || Hkv <= 0 || max_new < 0 || min_new < 0 || max_len < 0)
    return DKV_E_ARG;
  if (Dh != PG_DH || Hq % Hkv != 0 || Hq / Hkv > 16) return DKV_E_UNSUPPORTED;
  ChunkParams c;
  AttendParams& p = c.a;
  const int rc = fill_pool(p.pool, page_stride, head_stride, num_pages, page_size, page_table,
                           table_ld, table_cols, Hkv);
  if (rc != DKV_OK) return rc;
  if (B == 0 || T == 0 || max_new == 0) return DKV_OK;
  if (!q || !k_pages || !v_pages || !q_start || !lens || !out || num_pages == 0) return DKV_E_ARG;
  if (q_st < 0 || q_sh < 0 || o_st < 0 || o_sh < PG_DH) return DKV_E_ARG;
  const int oz = dkv_elt_size(out_dtype);
  const bool in_place = q == out && out_dtype == dtype && (T == 1 || q_st == o_st) &&
                        (Hq == 1 || q_sh == o_sh);
  if (!output_apart({(long long)(uintptr_t)out, oz * o_st, oz * o_sh, oz * PG_DH, T, Hq},
                    {(long long)(uintptr_t)q, 2 * q_st, 2 * q_sh, 2 * PG_DH, T, Hq}, in_place))
    return DKV_E_ARG;
  if (!aligned16(q) || !aligned16(k_pages) || !aligned16(v_pages) || (q_st & 7) || (q_sh & 7))
    return DKV_E_UNSUPPORTED;
  if (!attend_sizes_ok(B, T, Hq, Hkv, max_new)) return DKV_E_UNSUPPORTED;
  const AttendPlan plan = attend_plan(B, T, Hq, Hkv, max_new, min_new, max_len);
  if (!aligned16(workspace)) return DKV_E_UNSUPPORTED;
  if (plan.floats > 0 && (!workspace || workspace_floats < plan.floats)) return DKV_E_WORKSPACE;
  p.q = (const uint16_t*)q;
  p.q_st = q_st;
  p.q_sh = q_sh;
  p.k = (const uint16_t*)k_pages;
  p.v = (const uint16_t*)v_pages;
  p.q_start = q_start;
  p.lens = lens;
  p.out = out;
  p.o_st = o_st;
  p.o_sh = o_sh;
  p.B = B;
  p.T = T;
  p.Hq = Hq;
  p.Hkv = Hkv;
  p.hpg = Hq / Hkv;
  p.by_hpg = divisor(p.hpg);
  p.by_hkv = divisor(Hkv);
  p.scale_log2 = scale * 1.4426950408889634f;
  p.counters = reinterpret_cast<int*>(workspace);
  p.records = workspace ? workspace + D_COUNTERS : nullptr;
  p.split = plan.few_split;
  p.out_wide = !(((uintptr_t)out | (uintptr_t)o_st * dkv_elt_size(out_dtype) |
                  (uintptr_t)o_sh * dkv_elt_size(out_dtype)) &
                 (uintptr_t)(4 * dkv_elt_size(out_dtype) - 1));
  c.records = workspace ? workspace + D_COUNTERS + plan.many_at : nullptr;
  c.bq = plan.bq;
  c.bq_shift = plan.many ? __builtin_ctz((unsigned)plan.bq) : 0;
  c.items = plan.items;
  c.splits = plan.splits;
  c.by_splits = divisor(plan.many ? plan.splits : 1);
  c.few_rows = plan.few ? DROWS : 0;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == DKV_BF16) {
    if (out_dtype == DKV_F32)
      launch_attend<DKV_BF16, DKV_F32>(plan, c, st);
    else
      launch_attend<DKV_BF16, DKV_BF16>(plan, c, st);
  } else {
    if (out_dtype == DKV_F32)
      launch_attend<DKV_F16, DKV_F32>(plan, c, st);
    else
      launch_attend<DKV_F16, DKV_F16>(plan, c, st);
  }
  DKV_HIP_CHECK_LAUNCH();
  return DKV_OK;
}
