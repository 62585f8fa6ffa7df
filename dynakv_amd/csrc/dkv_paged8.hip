// Pages of 8 bits: the append of a step's keys and values to them, and pages read back as values.
// The layout of codes and scales: dkv_paged.h. The attention over them: dkv_paged.hip.
#include "dkv_paged.h"

namespace {

constexpr float E4M3_MAX = 448.f;
// Exponents a block may get: those for which every code times 2^e is a number of the model's type (in
// bf16 a normal one), so that the attention reads exactly what was stored.
template <int DT>
constexpr int E_LOW = DT == DKV_F16 ? -15 : -110;
template <int DT>
constexpr int E_HIGH = DT == DKV_F16 ? 7 : 119;

// ---------------------------------------------------------------------------------------
// Append to 8-bit pages. Queries as in the 16-bit append. Keys y (normed, rotated) and values y of one
// block (16 tokens, one head) get one exponent
//   e = least with max |y| <= 448 2^e, within E_LOW .. E_HIGH, and at least the block's old one where it
//       holds earlier tokens of the request (its first slots), whose codes are rounded again where their
//       scale changes (it rises, or lay outside the range),
//   c = y / 2^e rounded to the nearest e4m3 (ties to even), at most 448.
// Scales are powers of two: a code moved to a larger one only loses what falls below 2^-9 of it, so
// tokens that come one by one are held as those that come at once are, but for a last bit down there.
// A value is off by at most 2^-4 of itself from 2^-6 of the scale on, below that by 2^-10 of the scale.
// The block's largest lies between 224 and 448 scales where the scale is its least, so that is from
// 2^-13.8 of the largest on; a larger scale kept from earlier tokens raises the border with it. Values
// that are infinite or NaN are held as NaN and have no say in e.
//
// Keys are computed in 64 bits: which code a value gets turns over at borders, and 32-bit arithmetic with
// the sine instruction (off by 2^-19 or so) would put some hundreds of 8 million on another side of one.
//
// 8192 tokens of 32 + 2 x 8 heads with norms 52 us by trace (49 in a row; a large copy takes 37 for the
// bytes): the waves of keys have 12 us of issue slots, at three workgroups a CU (80 registers) partly
// beside the others' traffic. 64 tokens 6.0 us, the chain of lengths, page id, scale and codes. Tried and
// left: blocks and queries in turns on each CU (11% slower: both then have half the workgroups); a wave a
// block and head, 134 registers (68 us); keys as fp32 only, computed again where that may not do (as fast,
// 3.5 us more for few tokens).
//
// Two waves have one block and head (a unit: K heads, then V heads), eight tokens each: lane (token
// lane / 8, piece c = lane % 8) holds dims 8c .. 8c + 7 and 64 + 8c .. 64 + 8c + 7. The four units of a
// workgroup share the block's sines and cosines in LDS. Queries go to further workgroups of the
// launch, a wave per row and 8 heads.
// ---------------------------------------------------------------------------------------
struct Append8Params {
  const uint16_t* qkv;
  long long qkv_ld;
  uint16_t* q_out;
  long long q_st, q_sh;
  uint8_t* k;
  uint8_t* v;
  uint8_t* k_scale;
  uint8_t* v_scale;
  long long scale_page, scale_head;  // strides of the scales
  PagedPool pool;
  const int* q_start;
  const int* lens;
  int B, T, Hq, Hkv;
  int kv_wgs;      // leading workgroups: blocks times groups of units
  int by_row;      // an item for every row, as many as for the blocks' places
  Divisor by_groups, by_q_groups;
  const uint16_t* q_norm;  // (128,), or null: no norm
  const uint16_t* k_norm;
  float eps;
  double rev[PG_DH / 2];  // revolutions per position of each pair
};

constexpr int A8_WAVES = 8, A8_UNITS = 4;  // of a workgroup
constexpr int A8_SCAN = 256;  // requests that one wave sums over (64 at a time)
constexpr int A8_ROW = 72;  // pairs of doubles a token's sines and cosines take in LDS

// A block with new tokens: tokens t_lo .. t_hi - 1 of request b, all in block [base, base + 16).
struct NewBlock {
  int b;  // < 0: none
  int base, t_lo, t_hi;
  int row_of_0;  // row of token t: row_of_0 + t
};
// The item-th block with new tokens, request by request. Of more than A8_SCAN requests the one at the item-th
// place instead (paged_block_place), or the one whose first new token is row `item`, if there is one: found
// by a search, where sums over the requests before it would make the launch's time go by their square: single
// tokens of 512 requests 15.4 us (summed 17.2), of 1024 30.8 (42.4), of 4096 123 (370); of 256 9.4 (9.2).
__device__ __forceinline__ NewBlock new_block(const Append8Params& p, int item, int lane) {
  if (p.B > A8_SCAN) {
    const NewBlock none = {-1, 0, 0, 0, 0};
    int b, first = 0;
    if (p.by_row) {
      b = request_of_row(p.q_start, p.B, item, lane);
      if (b < 0) return none;
    } else {
      b = last_request(p.B, lane,
                       [&](int i) { return paged_block_place(max(p.q_start[i], 0), i) <= item; });
      first = paged_block_place(max(p.q_start[b], 0), b);
      if (first > item) return none;
    }
    b = __builtin_amdgcn_readfirstlane(b);
    const PagedRequest r = uniform(paged_request(p.pool, p.q_start, p.lens, b, p.T));
    const int lo = max(r.pos0, 0);
    const int hi = (int)min((long long)r.pos0 + r.n, (long long)p.pool.cols << p.pool.page_shift);
    if (r.n <= 0 || hi <= lo) return none;
    NewBlock n = {b, 0, 0, 0, r.row0 - r.pos0};
    if (p.by_row) {
      const int t = item - n.row_of_0;
      if (t < lo || t >= hi || (t != lo && t % PG_BLOCK)) return none;
      n.base = t / PG_BLOCK * PG_BLOCK;
    } else {
      const long long base = (lo / PG_BLOCK + (long long)(item - first)) * PG_BLOCK;
      if (base >= hi) return none;
      n.base = (int)base;
    }
    n.t_lo = max(lo, n.base);
    n.t_hi = min(hi, n.base + PG_BLOCK);
    return n;
  }
  int before = 0;
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    int count = 0, lo = 0, hi = 0, off = 0;
    if (b0 + lane < p.B) {
      const PagedRequest r = paged_request(p.pool, p.q_start, p.lens, b0 + lane, p.T);
      lo = max(r.pos0, 0);
      hi = (int)min((long long)r.pos0 + r.n, (long long)p.pool.cols << p.pool.page_shift);
      off = r.row0 - r.pos0;
      if (r.n > 0 && hi > lo) count = (hi - 1) / PG_BLOCK - lo / PG_BLOCK + 1;
    }
    const int run = pg_wave_scan(count);
    const unsigned long long hit = __ballot(item < before + run);
    if (hit) {
      const int l = __ffsll((long long)hit) - 1;
      NewBlock n;
      n.b = b0 + l;
      const int first = __builtin_amdgcn_readlane(lo, l);
      const int j = item - before - __builtin_amdgcn_readlane(run - count, l);
      n.base = (first / PG_BLOCK + j) * PG_BLOCK;
      n.t_lo = max(first, n.base);
      n.t_hi = min(__builtin_amdgcn_readlane(hi, l), n.base + PG_BLOCK);
      n.row_of_0 = __builtin_amdgcn_readlane(off, l);
      return n;
    }
    before += __builtin_amdgcn_readlane(run, 63);
  }
  return NewBlock{-1, 0, 0, 0, 0};
}

// cos and sin of f revolutions, 0 <= f < 1: reduced to an eighth of one, then the series (the first term
// left out is below 2^-53).
__device__ __forceinline__ double2 cos_sin_rev(double f) {
  const double q = rint(4.0 * f);
  const double x = (f - 0.25 * q) * 6.283185307179586477, z = x * x;
  double s = -1.0 / 1307674368000.0, c = 1.0 / 20922789888000.0;
  s = fma(s, z, 1.0 / 6227020800.0);
  s = fma(s, z, -1.0 / 39916800.0);
  s = fma(s, z, 1.0 / 362880.0);
  s = fma(s, z, -1.0 / 5040.0);
  s = fma(s, z, 1.0 / 120.0);
  s = fma(s, z, -1.0 / 6.0);
  s = fma(s * z, x, x);
  c = fma(c, z, -1.0 / 87178291200.0);
  c = fma(c, z, 1.0 / 479001600.0);
  c = fma(c, z, -1.0 / 3628800.0);
  c = fma(c, z, 1.0 / 40320.0);
  c = fma(c, z, -1.0 / 720.0);
  c = fma(c, z, 1.0 / 24.0);
  c = fma(c, z, -0.5);
  c = fma(c, z, 1.0);
  const int n = (int)q & 3;
  const double a = n & 1 ? s : c, b = n & 1 ? c : s;
  return double2{n == 1 || n == 2 ? -a : a, n >= 2 ? -b : b};
}

// The least e with m <= 448 2^e = 1.75 2^(e + 8) (m = 0: very low).
__device__ __forceinline__ int exponent_of(double m) {
  const unsigned long long bits = __builtin_bit_cast(unsigned long long, m);
  const bool above = (bits & 0xfffffffffffffULL) > 0xc000000000000ULL;
  return (int)(bits >> 52) - 1023 - 8 + above;
}
__device__ __forceinline__ double pow2(int e) {
  return __builtin_bit_cast(double, (unsigned long long)(1023 + e) << 52);
}

// Eight numbers rounded to e4m3. ANY: what is past 448 is 448, what is not finite becomes NaN (else they
// are neither).
template <bool ANY>
__device__ __forceinline__ dkv_u32x2 encode8(const float* f) {
  uint32_t w[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    float x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      x[i] = ANY ? __builtin_amdgcn_fmed3f(f[4 * k + i], -E4M3_MAX, E4M3_MAX) : f[4 * k + i];
    w[k] = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
    w[k] = __builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], w[k], true);
    if constexpr (ANY) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (!(fabsf(f[4 * k + i]) < INFINITY))
          w[k] = (w[k] & ~(0xffu << (8 * i))) | (0x7fu << (8 * i));
    }
  }
  return dkv_u32x2{w[0], w[1]};
}

// Workgroup `wg`: one block, four units; wave w has unit w / 2, the tokens of half w % 2 of the block.
template <int DT>
__device__ __forceinline__ void append8_block(const Append8Params& p, int wg, double2* sTrig,
                                              int* sNeed) {
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 7, slot = (wave & 1) * 8 + (lane >> 3);  // slot of the block
  const int groups = (int)p.by_groups.d;
  const int item = __builtin_amdgcn_readfirstlane(quot(p.by_groups, wg));
  const int unit0 = (wg - item * groups) * A8_UNITS, unit = unit0 + (wave >> 1);
  const NewBlock n = new_block(p, item, lane);
  if (n.b < 0) return;
  const bool is_k = unit < p.Hkv, there = unit < 2 * p.Hkv;
  const int t = n.base + slot;
  const bool isnew = there && t >= n.t_lo && t < n.t_hi, isold = there && t < n.t_lo;
  // the new row (before the page is known), then the earlier token's codes and the block's scale
  dkv_u32x4 xa = {0u, 0u, 0u, 0u}, xb = {0u, 0u, 0u, 0u};
  if (isnew) {
    const uint16_t* src = p.qkv + (long long)(n.row_of_0 + t) * p.qkv_ld +
                          (long long)(p.Hq + unit) * PG_DH + 8 * c;
    xa = *(const dkv_u32x4*)src;
    xb = *(const dkv_u32x4*)(src + 64);
  }
  const int page = __builtin_amdgcn_readfirstlane(paged_page(p.pool, n.b, n.base));
  if (page < 0) return;
  const int head = is_k ? unit : unit - p.Hkv, slot0 = n.base & (p.pool.page_size - 1);
  uint8_t* codes = (is_k ? p.k : p.v) + (long long)page * p.pool.page_stride +
                   (long long)head * p.pool.head_stride + (long long)(slot0 + slot) * PG_DH + 8 * c;
  uint8_t* scale = (is_k ? p.k_scale : p.v_scale) + (long long)page * p.scale_page +
                   (long long)head * p.scale_head + slot0 / PG_BLOCK;
  const bool has_old = n.t_lo > n.base;
  dkv_u32x2 oa = {0u, 0u}, ob = {0u, 0u};
  uint32_t old_byte = 127;
  if (has_old) {
    if (there) old_byte = *scale;
    if (isold) {
      oa = *(const dkv_u32x2*)codes;
      ob = *(const dkv_u32x2*)(codes + 64);
    }
  }
  if (unit0 < p.Hkv) {  // some of the waves have keys
    const int first = n.t_lo - n.base, pairs = (n.t_hi - n.t_lo) * (PG_DH / 2);
    for (int x = tid; x < pairs; x += 64 * A8_WAVES) {
      const int s = first + x / (PG_DH / 2), j = x % (PG_DH / 2);
      const double r = (double)(n.base + s) * p.rev[j];
      // (read below by piece j / 8 of the lanes, element j % 8)
      sTrig[s * A8_ROW + (j % 8) * 8 + j / 8] = cos_sin_rev(r - floor(r));
    }
    __syncthreads();
  }

  float f[16];  // y, then y scaled
  double y[16], big = 0.0, zeros = 0.0;
  bool odd = false;  // something is not finite
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    f[2 * e] = dkv_elt_to_f32<DT>(xa[e] & 0xffffu);
    f[2 * e + 1] = dkv_elt_to_f32<DT>(xa[e] >> 16);
    f[8 + 2 * e] = dkv_elt_to_f32<DT>(xb[e] & 0xffffu);
    f[8 + 2 * e + 1] = dkv_elt_to_f32<DT>(xb[e] >> 16);
  }
  if (is_k) {
#pragma unroll
    for (int e = 0; e < 16; ++e) y[e] = (double)f[e];
    if (p.k_norm) {
      double ss = 0.0;
#pragma unroll
      for (int e = 0; e < 16; ++e) ss = fma(y[e], y[e], ss);
#pragma unroll
      for (int o = 1; o <= 4; o <<= 1) ss += __shfl_xor(ss, o, 64);
      const double inv = 1.0 / sqrt(ss * (1.0 / PG_DH) + (double)p.eps);
      float wx[8], wy[8];
      load8<DT>(p.k_norm + 8 * c, wx);
      load8<DT>(p.k_norm + 64 + 8 * c, wy);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        y[e] = y[e] * inv * (double)wx[e];
        y[8 + e] = y[8 + e] * inv * (double)wy[e];
      }
    }
    if (isnew) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const double2 cs = sTrig[slot * A8_ROW + 8 * e + c];
        const double u = y[e], w = y[8 + e];
        y[e] = fma(u, cs.x, -(w * cs.y));
        y[8 + e] = fma(w, cs.x, u * cs.y);
        big = fmax(big, fmax(fabs(y[e]), fabs(y[8 + e])));
        zeros = fma(y[e], 0.0, fma(y[8 + e], 0.0, zeros));
      }
      odd = !(zeros == 0.0);  // (a NaN, which is no maximum)
      if (!(big < INFINITY)) {  // without what is not finite
        odd = true;
        big = 0.0;
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (fabs(y[e]) < INFINITY) big = fmax(big, fabs(y[e]));
      }
    }
  } else {
    float m = 0.f, none = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      m = fmaxf(m, fabsf(f[e]));
      none = fmaf(f[e], 0.f, none);
    }
    if (!(none == 0.f)) {
      odd = true;
      m = 0.f;
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (fabsf(f[e]) < INFINITY) m = fmaxf(m, fabsf(f[e]));
    }
    big = (double)m;
  }
  // the block's exponent, from both halves
  int need = (int)dkv_wave_max_fast((float)exponent_of(big));  // (small whole numbers)
  if (lane == 0) sNeed[wave] = need;
  __syncthreads();
  if (!there) return;
  need = max(need, sNeed[wave ^ 1]);
  // (the block's own exponent may lie outside the range: pages of another type's, or a user's)
  const int old_e = __builtin_amdgcn_readfirstlane((int)old_byte) - 127;
  int e_new = min(max(need, E_LOW<DT>), E_HIGH<DT>);
  if (has_old) e_new = max(e_new, min(max(old_e, E_LOW<DT>), E_HIGH<DT>));
  e_new = __builtin_amdgcn_readfirstlane(e_new);
  const bool again = has_old && e_new != old_e;  // earlier codes are rounded to the new scale

  const bool any = __ballot(odd) || need > E_HIGH<DT> || (again && old_e > e_new);
  if (isnew) {
    if (is_k) {
      // y / 2^e as floats from which e4m3 rounds as it would from y: where rounding to fp32 landed on a
      // border between two codes (or on a code, which has no more bits), a step to y's side of it
      const double by = pow2(-e_new);
      uint32_t tie = 0xffffffffu;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        y[e] *= by;
        f[e] = (float)y[e];
        tie = min(tie, __float_as_uint(f[e]) & 0x7ffffu);
      }
      if (tie == 0) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const uint32_t bits = __float_as_uint(f[e]);
          if ((bits & 0x7ffffu) == 0 && (double)f[e] != y[e])  // (a NaN stays one)
            f[e] = __uint_as_float(fabs(y[e]) < fabs((double)f[e]) ? bits - 1 : bits + 1);
        }
      }
    } else {
      const float by = __uint_as_float((uint32_t)(127 - e_new) << 23);
#pragma unroll
      for (int e = 0; e < 16; ++e) f[e] *= by;
    }
  } else if (isold && again) {
    // 2^(old_e - e_new), from 2^18 on as 2^18: every code but 0 is then past 448. Byte 255 is NaN.
    const int up = min(max(old_e - e_new, -127), 18);
    const float by = old_e == 128 ? NAN : __uint_as_float((uint32_t)(127 + up) << 23);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      f[4 * h] = __builtin_amdgcn_cvt_f32_fp8(oa[h], 0) * by;
      f[4 * h + 1] = __builtin_amdgcn_cvt_f32_fp8(oa[h], 1) * by;
      f[4 * h + 2] = __builtin_amdgcn_cvt_f32_fp8(oa[h], 2) * by;
      f[4 * h + 3] = __builtin_amdgcn_cvt_f32_fp8(oa[h], 3) * by;
      f[8 + 4 * h] = __builtin_amdgcn_cvt_f32_fp8(ob[h], 0) * by;
      f[8 + 4 * h + 1] = __builtin_amdgcn_cvt_f32_fp8(ob[h], 1) * by;
      f[8 + 4 * h + 2] = __builtin_amdgcn_cvt_f32_fp8(ob[h], 2) * by;
      f[8 + 4 * h + 3] = __builtin_amdgcn_cvt_f32_fp8(ob[h], 3) * by;
    }
  }
  if (isnew || (isold && again)) {
    if (any) {
      *(dkv_u32x2*)codes = encode8<true>(f);
      *(dkv_u32x2*)(codes + 64) = encode8<true>(f + 8);
    } else {
      *(dkv_u32x2*)codes = encode8<false>(f);
      *(dkv_u32x2*)(codes + 64) = encode8<false>(f + 8);
    }
  }
  if (lane == 0 && !(wave & 1)) *scale = (uint8_t)(127 + e_new);
}

template <int DT>
__global__ __launch_bounds__(64 * A8_WAVES, 6) void paged_append8_kernel(Append8Params p) {
  __shared__ double2 sTrig[PG_BLOCK * A8_ROW];
  __shared__ int sNeed[A8_WAVES];
  if ((int)blockIdx.x < p.kv_wgs) {
    append8_block<DT>(p, blockIdx.x, sTrig, sNeed);
    return;
  }
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int item = (int)(blockIdx.x - p.kv_wgs) * A8_WAVES + wave;
  const int row = quot(p.by_q_groups, item);
  const int h = (item - row * (int)p.by_q_groups.d) * 8 + (lane >> 3), c = lane & 7;
  if (row >= p.T) return;
  const int b = request_of_row(p.q_start, p.B, row, lane);
  if (b < 0) return;
  const int a0 = p.q_start[b], a1 = p.q_start[b + 1];
  const int pos = p.lens[b] - (a1 - a0) + (row - a0);
  if (pos < 0 || h >= p.Hq) return;
  float ox[8], oy[8];
  paged_turn<DT>(p.qkv + (long long)row * p.qkv_ld + (long long)h * PG_DH, p.q_norm, p.eps, pos,
                 p.rev, c, ox, oy);
  uint16_t* dst = p.q_out + (long long)row * p.q_st + (long long)h * p.q_sh;
  *(dkv_u32x4*)(dst + 8 * c) = round8<DT>(ox);
  *(dkv_u32x4*)(dst + 64 + 8 * c) = round8<DT>(oy);
}

// ---------------------------------------------------------------------------------------
// Pages read back: value = code * scale, of all pages or of those that `ids` names (one outside the pool
// gives zeros), keys and values to (pages, heads, page_size, 128) each. Bound by memory.
// ---------------------------------------------------------------------------------------
struct ValuesParams {
  const uint8_t* k;
  const uint8_t* v;
  PagedScales scales;
  long long page_stride, head_stride;
  int num_pages, page_shift, Hkv;
  const int* ids;  // null: page i
  Divisor by_hkv;
  long long pieces;  // V_CODES each
  void* k_out;
  void* v_out;
};
// A thread's codes of one access: a wave's stores are whole lines (16 codes, two stores of every other 16
// bytes: 50 us instead of 44 for 512 pages of 64 tokens, through the caches)
template <int ODT>
constexpr int V_CODES = ODT == DKV_F32 ? 4 : 8;
constexpr int V_THREADS = 256, V_EACH = 8;

template <int ODT>
__global__ __launch_bounds__(V_THREADS) void paged_values_kernel(ValuesParams p) {
  constexpr int CODES = V_CODES<ODT>, PIECES = PG_DH / CODES;  // of a token
  const bool is_v = blockIdx.y != 0;
  const uint8_t* pool = is_v ? p.v : p.k;
  const uint8_t* scales = is_v ? p.scales.v : p.scales.k;
  uint8_t* out = (uint8_t*)(is_v ? p.v_out : p.k_out);
  const long long at0 = (long long)blockIdx.x * (V_THREADS * V_EACH) + threadIdx.x;
  dkv_u32x2 codes[V_EACH];
  uint32_t byte[V_EACH];
#pragma unroll
  for (int u = 0; u < V_EACH; ++u) {
    const long long at = at0 + u * V_THREADS;
    codes[u] = dkv_u32x2{0u, 0u};
    byte[u] = 127;
    if (at >= p.pieces) continue;
    const PagedPiece x = paged_piece<PIECES>(at, p.page_shift);  // (row: page and head)
    const int i = quot(p.by_hkv, x.row), h = x.row - i * p.Hkv;
    const int page = p.ids ? p.ids[i] : i;
    if (page < 0 || page >= p.num_pages) continue;
    const uint8_t* src = pool + (long long)page * p.page_stride + (long long)h * p.head_stride +
                         paged_slot_at(x.slot) + CODES * x.piece;
    if constexpr (CODES == 8)
      codes[u] = *(const dkv_u32x2*)src;
    else
      codes[u].x = *(const uint32_t*)src;
    byte[u] = scales[(long long)page * p.scales.page_stride + (long long)h * p.scales.head_stride +
                     x.slot / PG_BLOCK];
  }
#pragma unroll
  for (int u = 0; u < V_EACH; ++u) {
    const long long at = at0 + u * V_THREADS;
    if (at >= p.pieces) continue;
    dkv_u32x4 x;
    if constexpr (ODT == DKV_F32) {
      const float s = pg_factor(byte[u]);
      x[0] = __float_as_uint(__builtin_amdgcn_cvt_f32_fp8(codes[u].x, 0) * s);
      x[1] = __float_as_uint(__builtin_amdgcn_cvt_f32_fp8(codes[u].x, 1) * s);
      x[2] = __float_as_uint(__builtin_amdgcn_cvt_f32_fp8(codes[u].x, 2) * s);
      x[3] = __float_as_uint(__builtin_amdgcn_cvt_f32_fp8(codes[u].x, 3) * s);
    } else {
      const float s = pg_scale(byte[u]);
      x = dkv_u32x4{pg_pair<ODT, false>(codes[u].x, s), pg_pair<ODT, true>(codes[u].x, s),
                    pg_pair<ODT, false>(codes[u].y, s), pg_pair<ODT, true>(codes[u].y, s)};
    }
    // (past the caches: 35 us for 512 pages of 64 tokens, 44 through them)
    __builtin_nontemporal_store(x, (dkv_u32x4*)(out + at * 16));
  }
}

bool ranges_meet(const void* a, long long an, const void* b, long long bn) {
  return (uintptr_t)a < (uintptr_t)b + bn && (uintptr_t)b < (uintptr_t)a + an;
}

}  // namespace

extern "C" int dkv_paged_append8(void* stream, int dtype, const void* qkv, long long qkv_ld,
                                 void* q_out, long long q_st, long long q_sh, void* k_pages,
                                 void* v_pages, long long page_stride, long long head_stride,
                                 int num_pages, int page_size, void* k_scale, void* v_scale,
                                 long long scale_page_stride, long long scale_head_stride,
                                 const int* page_table, long long table_ld, int table_cols,
                                 const int* q_start, const int* lens, int B, int T, int Hq, int Hkv,
                                 int Dh, const void* q_norm, const void* k_norm, float eps,
                                 const double* inv_freq) {
  if (dtype != DKV_F16 && dtype != DKV_BF16) return DKV_E_UNSUPPORTED;
  if (B < 0 || T < 0 || Hq <= 0 || Hkv <= 0) return DKV_E_ARG;
  if (Dh != PG_DH || Hq % Hkv != 0) return DKV_E_UNSUPPORTED;
  Append8Params p;
  int rc = fill_pool(p.pool, page_stride, head_stride, num_pages, page_size, page_table, table_ld,
                     table_cols, Hkv, 16);
  if (rc != DKV_OK) return rc;
  if (B == 0 || T == 0) return DKV_OK;
  if (!qkv || !q_out || !k_pages || !v_pages || !q_start || !lens || !inv_freq) return DKV_E_ARG;
  rc = check_scales({(const uint8_t*)k_scale, (const uint8_t*)v_scale, scale_page_stride,
                     scale_head_stride},
                    num_pages, page_size, Hkv);
  if (rc != DKV_OK) return rc;
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
  p.k = (uint8_t*)k_pages;
  p.v = (uint8_t*)v_pages;
  p.k_scale = (uint8_t*)k_scale;
  p.v_scale = (uint8_t*)v_scale;
  p.scale_page = scale_page_stride;
  p.scale_head = scale_head_stride;
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
  // n new tokens touch at most n blocks and at most n / 16 + 2
  const long long some = T / PG_BLOCK + 2LL * (B < T ? B : T), blocks = some < T ? some : T;
  const int groups = (2 * Hkv + A8_UNITS - 1) / A8_UNITS, q_groups = (Hq + 7) / 8;
  const long long q_items = (long long)T * q_groups;
  const long long wgs = blocks * groups + (q_items + A8_WAVES - 1) / A8_WAVES;
  if (wgs > 0x7fffffffLL || q_items > 0x7fffffffLL - A8_WAVES) return DKV_E_UNSUPPORTED;
  p.kv_wgs = (int)(blocks * groups);
  p.by_row = blocks == T;
  p.by_groups = divisor(groups);
  p.by_q_groups = divisor(q_groups);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == DKV_BF16)
    hipLaunchKernelGGL(paged_append8_kernel<DKV_BF16>, dim3((unsigned)wgs), dim3(64 * A8_WAVES), 0, st,
                       p);
  else
    hipLaunchKernelGGL(paged_append8_kernel<DKV_F16>, dim3((unsigned)wgs), dim3(64 * A8_WAVES), 0, st,
                       p);
  DKV_HIP_CHECK_LAUNCH();
  return DKV_OK;
}

extern "C" int dkv_paged_values(void* stream, int out_dtype, const void* k_pages, const void* v_pages,
                                long long page_stride, long long head_stride, int num_pages,
                                int page_size, int Hkv, int Dh, const void* k_scale,
                                const void* v_scale, long long scale_page_stride,
                                long long scale_head_stride, const int* ids, int n, void* k_out,
                                void* v_out) {
  if (out_dtype != DKV_F16 && out_dtype != DKV_BF16 && out_dtype != DKV_F32) return DKV_E_UNSUPPORTED;
  if (Hkv <= 0 || n < 0 || (!ids && n > num_pages)) return DKV_E_ARG;
  if (Dh != PG_DH) return DKV_E_UNSUPPORTED;
  PagedPool pool;
  int rc = fill_pool(pool, page_stride, head_stride, num_pages, page_size, nullptr, 0, 0, Hkv, 16);
  if (rc != DKV_OK) return rc;
  if (n == 0) return DKV_OK;
  if (!k_pages || !v_pages || !k_out || !v_out) return DKV_E_ARG;
  rc = check_scales({(const uint8_t*)k_scale, (const uint8_t*)v_scale, scale_page_stride,
                     scale_head_stride},
                    num_pages, page_size, Hkv);
  if (rc != DKV_OK) return rc;
  if (!aligned16(k_pages) || !aligned16(v_pages) || !aligned16(k_out) || !aligned16(v_out))
    return DKV_E_UNSUPPORTED;
  const long long bytes = (long long)n * Hkv * page_size * PG_DH * dkv_elt_size(out_dtype);
  if (ranges_meet(k_out, bytes, v_out, bytes)) return DKV_E_ARG;
  if ((long long)n * Hkv > 0x7fffffffLL) return DKV_E_UNSUPPORTED;
  ValuesParams p;
  p.k = (const uint8_t*)k_pages;
  p.v = (const uint8_t*)v_pages;
  p.scales = {(const uint8_t*)k_scale, (const uint8_t*)v_scale, scale_page_stride, scale_head_stride};
  p.page_stride = page_stride;
  p.head_stride = head_stride;
  p.num_pages = num_pages;
  p.page_shift = pool.page_shift;
  p.Hkv = Hkv;
  p.ids = ids;
  p.by_hkv = divisor(Hkv);
  p.pieces = (long long)n * Hkv * page_size *
             (PG_DH / (out_dtype == DKV_F32 ? V_CODES<DKV_F32> : V_CODES<DKV_BF16>));
  p.k_out = k_out;
  p.v_out = v_out;
  const long long wgs = (p.pieces + V_THREADS * V_EACH - 1) / (V_THREADS * V_EACH);
  if (wgs > 0x7fffffffLL) return DKV_E_UNSUPPORTED;
  const dim3 grid((unsigned)wgs, 2);
  hipStream_t st = (hipStream_t)stream;
  if (out_dtype == DKV_BF16)
    hipLaunchKernelGGL(paged_values_kernel<DKV_BF16>, grid, dim3(V_THREADS), 0, st, p);
  else if (out_dtype == DKV_F16)
    hipLaunchKernelGGL(paged_values_kernel<DKV_F16>, grid, dim3(V_THREADS), 0, st, p);
  else
    hipLaunchKernelGGL(paged_values_kernel<DKV_F32>, grid, dim3(V_THREADS), 0, st, p);
  DKV_HIP_CHECK_LAUNCH();
  return DKV_OK;
}
