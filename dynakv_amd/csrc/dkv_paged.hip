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

namespace {

constexpr int PG_DH = 128;

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
// 0 .. t; o = sum_k exp(s_k - m) v_k / sum_k exp(s_k - m), s_k = scale q . k. One wave per row and
// query head: lane l scores key l of a tile of 64, the maximum and the sum run over the tiles, and
// lane l sums dims 2l, 2l + 1 of the values.
// ---------------------------------------------------------------------------------------
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
  int B, T, Hq, Hkv;
  float scale;
};

template <int DT, int ODT>
__global__ __launch_bounds__(64) void paged_attend_kernel(AttendParams p) {
  __shared__ float sq[PG_DH];
  __shared__ float sp[64];
  __shared__ long long sv[64];
  const int lane = threadIdx.x;
  const int row = blockIdx.x, h = blockIdx.y, g = h / (p.Hq / p.Hkv);
  const int b = request_of_row(p.q_start, p.B, row, lane);
  if (b < 0) return;
  const PagedRequest r = paged_request(p.pool, p.q_start, p.lens, b, p.T);
  const int pos = r.pos0 + row - r.row0;
  const uint16_t* qr = p.q + (long long)row * p.q_st + (long long)h * p.q_sh;
  sq[2 * lane] = dkv_load_f32<DT>(qr, 2 * lane) * p.scale;
  sq[2 * lane + 1] = dkv_load_f32<DT>(qr, 2 * lane + 1) * p.scale;
  __syncthreads();
  const int end = min(pos + 1, r.len);
  float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
  for (int k0 = 0; k0 < end; k0 += 64) {
    const int key = k0 + lane;
    const int page = key < end ? paged_page(p.pool, b, key) : -1;
    const long long at = page < 0 ? -1
                                  : (long long)page * p.pool.page_stride +
                                        (long long)g * p.pool.head_stride +
                                        (long long)(key & (p.pool.page_size - 1)) * PG_DH;
    float s = -INFINITY;
    if (at >= 0) {
      s = 0.f;
      for (int d = 0; d < PG_DH; d += 8) {
        float kv[8];
        load8<DT>(p.k + at + d, kv);
#pragma unroll
        for (int e = 0; e < 8; ++e) s = fmaf(sq[d + e], kv[e], s);
      }
    }
    const float mt = fmaxf(m, dkv_wave_max(s));
    if (mt == -INFINITY) continue;
    const float alpha = expf(m - mt);
    const float pr = at >= 0 ? expf(s - mt) : 0.f;
    l = l * alpha + dkv_wave_sum(pr);
    o0 *= alpha;
    o1 *= alpha;
    m = mt;
    __syncthreads();
    sp[lane] = pr;
    sv[lane] = at;
    __syncthreads();
    const int cnt = min(64, end - k0);
    for (int j = 0; j < cnt; ++j) {
      if (sv[j] < 0) continue;
      const float w = sp[j];
      o0 = fmaf(w, dkv_load_f32<DT>(p.v + sv[j], 2 * lane), o0);
      o1 = fmaf(w, dkv_load_f32<DT>(p.v + sv[j], 2 * lane + 1), o1);
    }
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  const long long oi = (long long)row * p.o_st + (long long)h * p.o_sh + 2 * lane;
  dkv_store_f32<ODT>(p.out, oi, o0 * inv);
  dkv_store_f32<ODT>(p.out, oi + 1, o1 * inv);
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

int fill_pool(PagedPool& pool, long long page_stride, long long head_stride, int num_pages,
              int page_size, const int* table, long long table_ld, int cols, int Hkv) {
  if (num_pages < 0 || cols < 0 || table_ld < cols) return DKV_E_ARG;
  if (page_size < 16 || (page_size & (page_size - 1))) return DKV_E_UNSUPPORTED;
  if (head_stride < (long long)page_size * PG_DH && Hkv > 1) return DKV_E_ARG;
  if (page_stride < 0 || head_stride < 0) return DKV_E_ARG;
  if ((page_stride & 7) || (head_stride & 7)) return DKV_E_UNSUPPORTED;
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

extern "C" long long dkv_paged_workspace_floats(int B, int Hq, int Hkv, int max_new, int min_new,
                                                int max_len) {
  (void)B, (void)Hq, (void)Hkv, (void)max_new, (void)min_new, (void)max_len;
  return 0;
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
  if (!(scale > 0.f) || !(scale < INFINITY)) return DKV_E_UNSUPPORTED;
  if (dtype != DKV_F16 && dtype != DKV_BF16) return DKV_E_UNSUPPORTED;
  if (out_dtype != dtype && out_dtype != DKV_F32) return DKV_E_ARG;
  if (B < 0 || T < 0 || Hq <= 0 || Hkv <= 0 || max_new < 0 || min_new < 0 || max_len < 0)
    return DKV_E_ARG;
  if (Dh != PG_DH || Hq % Hkv != 0 || Hq / Hkv > 16) return DKV_E_UNSUPPORTED;
  AttendParams p;
  const int rc = fill_pool(p.pool, page_stride, head_stride, num_pages, page_size, page_table,
                           table_ld, table_cols, Hkv);
  if (rc != DKV_OK) return rc;
  if (B == 0 || T == 0 || max_new == 0) return DKV_OK;
  if (!q || !k_pages || !v_pages || !q_start || !lens || !out) return DKV_E_ARG;
  if (q_st < 0 || q_sh < 0 || o_st < 0 || o_sh < PG_DH) return DKV_E_ARG;
  if (!aligned16(q) || !aligned16(k_pages) || !aligned16(v_pages) || (q_st & 7) || (q_sh & 7))
    return DKV_E_UNSUPPORTED;
  (void)workspace, (void)workspace_floats;
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
  p.scale = scale;
  if (Hq > 65535) return DKV_E_UNSUPPORTED;
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)T, (unsigned)Hq);
#define PG_LAUNCH(DT, ODT) \
  hipLaunchKernelGGL((paged_attend_kernel<DT, ODT>), grid, dim3(64), 0, st, p)
  if (dtype == DKV_BF16) {
    if (out_dtype == DKV_F32)
      PG_LAUNCH(DKV_BF16, DKV_F32);
    else
      PG_LAUNCH(DKV_BF16, DKV_BF16);
  } else {
    if (out_dtype == DKV_F32)
      PG_LAUNCH(DKV_F16, DKV_F32);
    else
      PG_LAUNCH(DKV_F16, DKV_F16);
  }
#undef PG_LAUNCH
  DKV_HIP_CHECK_LAUNCH();
  return DKV_OK;
}
