// Sampling of a token per row of logits, from a given uniform number per row.
//
// With weights w_i = exp((l_i - max l) / t) and the tokens in the order of their logits (largest
// first, of equal ones the lowest index first):
//   top-k keeps the first k; top-p keeps, of those, the ones before which less than p of their mass
//   lies; min-p keeps, of those, the ones with w_i >= min_p. The first token is always kept.
// Each of them keeps a prefix of that order, so what is kept is given by the smallest logit kept
// and how many of its equals are (the lowest indices). The answer is the first token, in the
// vocabulary's order, up to which the kept mass exceeds u times all of it.
//
// Weights are held in 64-bit fixed point, 44 bits after the point: sums of them are the same in any
// order (the histogram adds by atomics), and a token is decided by u * mass against a running sum,
// where 32 bits would pick another token than the formula's in one draw of a few thousand. With
// x = 64 log2(e) (max l - l) / t as a sum of two 32-bit numbers p + r, i = floor(p):
//   w = 2^(-i/64) (1 - d),  d = 1 - 2^(-(x - i)/64) < 0.011,
// d to 31 bits after the point, 2^(-j/64) from a table of 64.
//
// Two ways through a row:
//  * 16-bit logits, a workgroup per row: by their values. A bin for each value (those next to 0 share
//    one), so the row is read twice: for the counts, from which the borders follow with one weight a
//    bin, and for the mass of every 512 tokens, by a table of the weights. Then the 512 and the token in
//    which u times the mass lies are known. us, 256 rows of 128256 bf16 with top-p: 34.5, of which the
//    first reading takes 10 at the rate of the memory, the second 9 (11 vector instructions a token and
//    a table read); 90 by bins of the weights' logarithm as below. fp16: 52, as more bins are cleared and
//    looked through, and more tokens are next to 0, for which the row is read once more.
//  * otherwise by the logarithm of the weights: for the maximum; for a histogram of the tokens by i,
//    counts and sums of d in one 64-bit number, so that a bin's mass is known and with it the bins of the
//    borders; for the mass of every 512 tokens (256 in fp32) above those bins, and the tokens inside
//    them, which are sorted and those kept added. A bin of too many tokens (equal logits, a border 64
//    halvings down) goes through a search by the digits of the logits instead. Bound by vector
//    instructions where a row has one CU (17 a token for the histogram), else by latency. Few rows are
//    cut into parts, a launch for each of the three passes; 37 rows of 50257 fp32: 28.9 us; 256 rows of
//    128256 fp32, uncut, 93.
// Rows in which one logit stands many times are slow, as its additions go to one place: us, 256 rows of
// 128256 with top-p, 95% of them 0: bf16 133, fp16 804 (the border is among what is next to 0, so that the
// row goes the other way), fp32 647; 95% of them -100: 124, 48, 73; all equal: 253, 257, 661. -1e4 and
// -infinity lie below all bins and cost nothing: 31, 48, 74.
#include "dkv_common.h"

namespace {

typedef unsigned long long u64;

constexpr int SM_THREADS = 1024;
constexpr int SM_WAVES = SM_THREADS / 64;
constexpr int SM_POINT = 44;             // bits after the point of a weight
constexpr int SM_MAX_V = 1 << 19;        // weights of at most 1: sums below 2^63
constexpr int SM_AHEAD = 2;              // 16-byte pieces that a thread has in flight
constexpr int SM_BINS = 4096;            // bins of 1/64 in log2 of the weight; the last: the rest
constexpr int SM_CAND = 2048;            // tokens of a border's bin that are sorted
constexpr int SM_CHUNKS = SM_MAX_V / 4 / 64 + 2;  // rows of 64 pieces (1 KB) of a row of logits
constexpr int SM_COUNT = 44;             // a bin: the count from this bit on, below it the sum of d
constexpr uint32_t SM_OFF = 1u << 13;    // added to d, which may be as low as -2^-19
constexpr double SM_ONE = 17592186044416.0;  // 2^44
constexpr int SM_KEYS = 1 << 15;         // bins of one logit value each (16-bit types)
constexpr int SM_TABLE = SM_KEYS / 2 - 2;  // weights of such values that a table holds
constexpr int SM_TIES = 54;              // a chunk: the tokens at the border from this bit on, below it mass
constexpr u64 SM_MASS = (1ULL << SM_TIES) - 1;

struct SampleParams {
  const void* logits;
  long long ld;
  int V;
  const float* u;
  const float* temperature;  // per row, or null: the value below for every row (and so on)
  const int* top_k;
  const float* top_p;
  const float* min_p;
  float temperature_all, top_p_all, min_p_all;
  int top_k_all;
  long long* out;
  u64* ws;    // SM_WS words a row where rows are cut
  int parts;  // workgroups of a row
};

// A cut row's words in the workspace: the parts' maxima, the number of listed tokens and of parts that
// are done, the histogram, the tokens of the borders' bins, the masses of the rows of pieces.
constexpr int SM_PARTS = 16;
constexpr int SM_WS_N = SM_PARTS, SM_WS_HIST = 32, SM_WS_CAND = SM_WS_HIST + SM_BINS,
              SM_WS_CHUNK = SM_WS_CAND + SM_CAND, SM_WS = SM_WS_CHUNK + SM_CHUNKS;
static_assert(SM_WS % 2 == 0 && SM_WS_HIST % 2 == 0, "16-byte accesses");

template <int DT>
struct SampleShared {
  union {
    struct {
      __attribute__((aligned(16))) u64 hist[SM_BINS + 64];  // and 64 that catch the rest
      u64 cand[SM_CAND], sort[SM_CAND];
    };
    __attribute__((aligned(16))) uint32_t bins[DT == DKV_F32 ? 4 : SM_KEYS];
    u64 table[DT == DKV_F32 ? 2 : SM_KEYS / 2];
  };
  u64 chunk[SM_CHUNKS];
  u64 wave[SM_WAVES], wave2[SM_WAVES], pick[4];
  uint32_t root[64];
  int n, last;
};

// 2^(31 - j/64), rounded
__device__ const uint32_t sm_root[64] = {
    0x80000000u, 0x7e9f0606u, 0x7d41d96eu, 0x7be86fbau, 0x7a92be8bu, 0x7940bb9eu, 0x77f25cceu,
    0x76a7980fu, 0x75606374u, 0x741cb528u, 0x72dc8374u, 0x719fc4b9u, 0x70666f76u, 0x6f307a41u,
    0x6dfddbccu, 0x6cce8ae1u, 0x6ba27e65u, 0x6a79ad56u, 0x69540ec9u, 0x683199edu, 0x6712460bu,
    0x65f60a7fu, 0x64dcdec3u, 0x63c6ba64u, 0x62b39509u, 0x61a3666du, 0x60962665u, 0x5f8bccdbu,
    0x5e8451d0u, 0x5d7fad59u, 0x5c7dd7a4u, 0x5b7ec8f2u, 0x5a82799au, 0x5988e209u, 0x5891fac1u,
    0x579dbc57u, 0x56ac1f75u, 0x55bd1cdbu, 0x54d0ad5au, 0x53e6c9dau, 0x52ff6b55u, 0x521a8ad7u,
    0x51382182u, 0x50582888u, 0x4f7a9930u, 0x4e9f6cd4u, 0x4dc69cddu, 0x4cf022cau, 0x4c1bf829u,
    0x4b4a169cu, 0x4a7a77d4u, 0x49ad1598u, 0x48e1e9bau, 0x4818ee22u, 0x47521cc6u, 0x468d6faeu,
    0x45cae0f2u, 0x450a6abbu, 0x444c0740u, 0x438fb0cbu, 0x42d561b4u, 0x421d1462u, 0x4166c34cu,
    0x40b268fau,
};

// A logit as a number that orders as the logits do (-0 as +0).
__device__ __forceinline__ uint32_t sm_key(float f) {
  const uint32_t b = __float_as_uint(f + 0.0f);
  return b ^ ((int)b < 0 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float sm_unkey(uint32_t k) {
  return __uint_as_float(k ^ ((int)k < 0 ? 0x80000000u : 0xffffffffu));
}

template <int CTRL>
__device__ __forceinline__ u64 sm_dpp(u64 v) {
  return (uint32_t)dkv_dpp_i32<CTRL>((int)(uint32_t)v) |
         ((u64)(uint32_t)dkv_dpp_i32<CTRL>((int)(uint32_t)(v >> 32)) << 32);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 sm_dpp_rows(u64 v) {  // 0 into the rows that are not meant
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xf, false) |
         ((u64)(uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROWS, 0xf,
                                                     false)
          << 32);
}
__device__ __forceinline__ u64 sm_wave_scan(u64 v) {  // inclusive, as dkv_wave_scan_fast
  v += sm_dpp<0x111>(v);
  v += sm_dpp<0x112>(v);
  v += sm_dpp<0x114>(v);
  v += sm_dpp<0x118>(v);
  v += sm_dpp_rows<0x142, 0xa>(v);
  v += sm_dpp_rows<0x143, 0xc>(v);
  return v;
}
__device__ __forceinline__ u64 sm_wave_sum(u64 v) {  // as dkv_wave_sum_fast
  v += sm_dpp<0xb1>(v);
  v += sm_dpp<0x4e>(v);
  v += sm_dpp<0x141>(v);
  v += sm_dpp<0x140>(v);
  {
    const uint32_t lo = (uint32_t)v, hi = (uint32_t)(v >> 32);
    const auto a = __builtin_amdgcn_permlane16_swap(lo, lo, false, false);
    const auto b = __builtin_amdgcn_permlane16_swap(hi, hi, false, false);
    v = (a[0] | ((u64)b[0] << 32)) + (a[1] | ((u64)b[1] << 32));
  }
  {
    const uint32_t lo = (uint32_t)v, hi = (uint32_t)(v >> 32);
    const auto a = __builtin_amdgcn_permlane32_swap(lo, lo, false, false);
    const auto b = __builtin_amdgcn_permlane32_swap(hi, hi, false, false);
    v = (a[0] | ((u64)b[0] << 32)) + (a[1] | ((u64)b[1] << 32));
  }
  return v;
}

// lane `lane`'s value, for all (the lane is the whole wave's)
__device__ __forceinline__ u64 sm_lane(u64 v, int lane) {
  return (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane) |
         ((u64)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), lane) << 32);
}
__device__ __forceinline__ u64 sm_first(u64 v) { return sm_lane(v, 0); }

// the sums of two waves' values, halfway: of lanes l and l + 32 (a in the lower half, b in the upper);
// of rows of 16 lanes 2r and 2r + 1 (a in row 2r, b in row 2r + 1)
__device__ __forceinline__ u64 sm_meet32(u64 a, u64 b) {
  const auto x = __builtin_amdgcn_permlane32_swap((uint32_t)a, (uint32_t)b, false, false);
  const auto y =
      __builtin_amdgcn_permlane32_swap((uint32_t)(a >> 32), (uint32_t)(b >> 32), false, false);
  return (x[0] | ((u64)y[0] << 32)) + (x[1] | ((u64)y[1] << 32));
}
__device__ __forceinline__ u64 sm_meet16(u64 a, u64 b) {
  const auto x = __builtin_amdgcn_permlane16_swap((uint32_t)a, (uint32_t)b, false, false);
  const auto y =
      __builtin_amdgcn_permlane16_swap((uint32_t)(a >> 32), (uint32_t)(b >> 32), false, false);
  return (x[0] | ((u64)y[0] << 32)) + (x[1] | ((u64)y[1] << 32));
}

// What is kept: every token above `at`, and those at it up to index `last`.
struct Border {
  float at;
  int last;
};

__device__ __forceinline__ u64 sm_get(const u64* a) {
  return __hip_atomic_load(a, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void sm_put(u64* a, u64 v) {
  __hip_atomic_store(a, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// One workgroup's work on a row.
template <int DT>
struct RowSampler {
  static constexpr int E = DT == DKV_F32 ? 4 : 8;  // elements of a 16-byte piece
  const SampleParams& p;
  SampleShared<DT>& s;
  const int row, tid, lane, wave, V;
  const char* base;
  int head, rows64;  // elements of the first aligned piece before the row; its rows of 64 pieces
  int r0, r1;        // the wave's rows of pieces
  float t, tp, mp, u;
  uint32_t root;
  int k;
  bool by_k, by_p;
  bool infinite = false;
  float m, c_hi, c_lo;  // largest logit; 64 log2(e) / t
  u64 floor_w;
  Border keep = {-INFINITY, -1};
  u64 kept = 0;  // the mass of what is kept so far
  // the histogram's running counts and masses before the thread's bins 4 tid .. 4 tid + 3, and theirs
  u64 n_run, m_run, cnt[4], mass[4];

  __device__ __forceinline__ RowSampler(const SampleParams& p_, SampleShared<DT>& s_, int row_)
      : p(p_), s(s_), row(row_), tid(threadIdx.x), lane(threadIdx.x & 63),
        wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)), V(p_.V) {
    base = (const char*)p.logits + (long long)row * p.ld * (16 / E);
    head = (int)((uintptr_t)base & 15) / (16 / E);
    rows64 = (V + head + E * 64 - 1) / (E * 64);
    t = p.temperature ? p.temperature[row] : p.temperature_all;
    k = p.top_k ? p.top_k[row] : p.top_k_all;
    tp = p.top_p ? p.top_p[row] : p.top_p_all;
    mp = p.min_p ? p.min_p[row] : p.min_p_all;
    u = p.u[row];
    by_k = k > 0 && k < V;
    by_p = tp < 1.f;
    floor_w = mp > 0.f && mp <= 1.f ? (u64)ceil((double)mp * SM_ONE) : 0;
    root = sm_root[lane];
  }
  // (after the first loads are under way; seen after the next barrier)
  __device__ __forceinline__ void keep_root() {
    if (wave == 0) s.root[lane] = root;
  }
  // only the first token is kept
  __device__ __forceinline__ bool greedy() const {
    return !(t > 0.f) || k == 1 || tp <= 0.f || mp > 1.f;
  }
  // the workgroup takes part `part` of `parts` of the row
  __device__ __forceinline__ void take(int part, int parts) {
    const int per = (rows64 + parts - 1) / parts;
    const int a = min(rows64, part * per), b = min(rows64, a + per);
    const int pw = (b - a + SM_WAVES - 1) / SM_WAVES;
    r0 = min(b, a + wave * pw);
    r1 = min(b, r0 + pw);
  }

  // ---- the row: pieces of 16 aligned bytes, 64 to a row of pieces ----
  __device__ __forceinline__ int first_of(int R) const { return (R * 64 + lane) * E - head; }
  // the lane's piece of row R as its words; elements outside the row of logits are -infinity
  __device__ __forceinline__ dkv_u32x4 load(int R) const {
    const int i0 = first_of(R);
    constexpr uint32_t none = DT == DKV_F32 ? 0xff800000u
                              : DT == DKV_BF16 ? 0xff80ff80u
                                               : 0xfc00fc00u;
    dkv_u32x4 v = {none, none, none, none};
    if (i0 >= 0 && i0 + E <= V) {
      v = *(const dkv_u32x4*)(base + (long long)i0 * (16 / E));
    } else if (i0 + E > 0 && i0 < V) {  // the first or the last piece
      uint32_t w[4] = {none, none, none, none};
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if (i0 + e < 0 || i0 + e >= V) continue;
        if constexpr (E == 4) {
          w[e] = ((const uint32_t*)base)[i0 + e];
        } else {
          const uint32_t x = ((const uint16_t*)base)[i0 + e];
          w[e / 2] = e & 1 ? (w[e / 2] & 0xffffu) | (x << 16) : (w[e / 2] & 0xffff0000u) | x;
        }
      }
      v = dkv_u32x4{w[0], w[1], w[2], w[3]};
    }
    if (infinite) {  // logits of +infinity share the mass: they are read as 0, the others as -infinity
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (DT == DKV_F32) {
          v[i] = v[i] == 0x7f800000u ? 0u : 0xff800000u;
        } else {
          constexpr uint32_t inf = DT == DKV_BF16 ? 0x7f80u : 0x7c00u;
          v[i] = ((v[i] & 0xffffu) == inf ? 0u : inf | 0x8000u) |
                 ((v[i] >> 16) == inf ? 0u : (inf | 0x8000u) << 16);
        }
      }
    }
    return v;
  }
  static __device__ __forceinline__ float value(const dkv_u32x4& v, int e) {
    if constexpr (DT == DKV_F32)
      return __uint_as_float(v[e]);
    else if constexpr (DT == DKV_BF16)
      return __uint_as_float(e & 1 ? v[e / 2] & 0xffff0000u : v[e / 2] << 16);
    else
      return dkv_f16_bits_to_f32(e & 1 ? v[e / 2] >> 16 : v[e / 2] & 0xffffu);
  }
  // f(R, first token of the lane's piece, the piece) for each of the wave's rows of pieces, in order
  template <class F>
  __device__ __forceinline__ void each(F&& f) const {
#pragma unroll 1
    for (int R = r0; R < r1; R += SM_AHEAD) {
      dkv_u32x4 v[SM_AHEAD];
#pragma unroll
      for (int q = 0; q < SM_AHEAD; ++q)
        if (R + q < r1) v[q] = load(R + q);
#pragma unroll
      for (int q = 0; q < SM_AHEAD; ++q)
        if (R + q < r1) f(R + q, first_of(R + q), v[q]);
    }
  }

  // ---- the largest logit of the workgroup's part, or for a greedy row that and its first index, as
  // (key, ~index) ----
  __device__ __forceinline__ u64 largest() {
    float x = -INFINITY;
    each([&](int, int, const dkv_u32x4& v) {
#pragma unroll
      for (int e = 0; e < E; ++e) x = fmaxf(x, value(v, e));  // (a NaN is passed over)
    });
    x = dkv_wave_max(x);
    u64 best = (u64)sm_key(x) << 32;
    if (greedy()) {  // of the waves with the largest, each the first index of its own
      int at = 0x7fffffff;
      each([&](int, int i0, const dkv_u32x4& v) {
#pragma unroll
        for (int e = E - 1; e >= 0; --e)
          if (value(v, e) == x) at = min(at, i0 + e);
      });
#pragma unroll
      for (int o = 32; o >= 1; o >>= 1) at = min(at, __shfl_xor(at, o, 64));
      best |= (uint32_t)~at;
    }
    keep_root();
    if (lane == 0) s.wave[wave] = best;
    __syncthreads();
    best = s.wave[lane & (SM_WAVES - 1)];
    best = max(best, sm_dpp<0xb1>(best));
    best = max(best, sm_dpp<0x4e>(best));
    best = max(best, sm_dpp<0x141>(best));
    best = max(best, sm_dpp<0x140>(best));
    return sm_first(best);
  }
  // Takes the row's largest logit; false where that decides the row (the answer is written, by one).
  __device__ __forceinline__ bool begin(u64 best, bool write) {
    m = sm_unkey((uint32_t)(best >> 32));
    if (m == -INFINITY || greedy()) {
      if (write && tid == 0) p.out[row] = m == -INFINITY ? -1 : (long long)~(uint32_t)best;
      return false;
    }
    if (m == INFINITY) {
      infinite = true;
      m = 0.f;
    }
    set_scale();
    return true;
  }
  __device__ __forceinline__ void set_scale() {
    const double c64 = 64.0 * 1.4426950408889634074 / (double)fminf(fmaxf(t, 1e-30f), 1e30f);
    c_hi = (float)c64;
    c_lo = (float)(c64 - (double)c_hi);
  }

  // x of a logit, up to that of the last bin (that of a NaN); `dl`: max l - l as it was rounded
  __device__ __forceinline__ float x_of(float l, float& dl) const {
    dl = m - l;
    return fminf(dl * c_hi, (float)(SM_BINS - 1));
  }
  // The bin of a logit; `d`: 2^31 d + SM_OFF. Of max l - l fp32 logits take what the rounding left;
  // 16-bit ones are exact but for some next to 0.
  __device__ __forceinline__ int split(float l, uint32_t& d) const {
    float dl;
    const float x = x_of(l, dl);
    float r = fmaf(dl, c_lo, fmaf(dl, c_hi, -x));
    if constexpr (DT == DKV_F32) r = fmaf((m - dl) - l, c_hi, r);
    const float f = __builtin_amdgcn_fractf(x) + r;
    // 2^31 (1 - 2^(-f/64)) by the cubic of least error over 0 .. 1 through 0 (0.02 of a unit; the
    // coefficients' own rounding 0.4)
    const float y = fmaf(f, fmaf(f, fmaf(f, 452.14603f, -125946.242f), 23258160.f), (float)SM_OFF);
    d = (uint32_t)y;
    return (int)x;
  }
  // the weight of a logit, in 2^-44
  __device__ __forceinline__ u64 weight(float l) const {
    uint32_t d;
    const int i = split(l, d);
    const u64 w = (u64)s.root[i & 63] * (u64)(uint32_t)((1u << 31) + SM_OFF - d);  // 2^62 w
    return i == SM_BINS - 1 ? 0ULL : w >> min((62 - SM_POINT) + (i >> 6), 63);
  }
  __device__ __forceinline__ u64 floored(u64 w) const { return w >= floor_w ? w : 0ULL; }
  // the mass of a bin
  __device__ __forceinline__ u64 bin_mass(int i, u64 h) const {
    const double n = (double)(h >> SM_COUNT);
    const double d = (double)(h & ((1ULL << SM_COUNT) - 1)) - n * (double)SM_OFF;
    const double w = (double)s.root[i & 63] * (n - d * (1.0 / 2147483648.0));  // 2^31 w
    return i == SM_BINS - 1 ? 0ULL : (u64)rint(ldexp(w, SM_POINT - 31 - (i >> 6)));
  }
  __device__ __forceinline__ bool is_kept(float l, int i) const {
    return l > keep.at || (l == keep.at && i <= keep.last);
  }

  // ---- the histogram of the workgroup's part ----
  // The last bin, the rest, stays empty: such a token goes to its lane's bin behind it (a branch around
  // the addition keeps the eight tokens of a piece from being worked on together).
  __device__ __forceinline__ void histogram() {
    for (int i = tid; i < SM_BINS; i += SM_THREADS) s.hist[i] = 0;
    __syncthreads();
    each([&](int, int, const dkv_u32x4& v) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        uint32_t d;
        const int i = split(value(v, e), d);
        atomicAdd(&s.hist[i < SM_BINS - 1 ? i : SM_BINS + lane], (1ULL << SM_COUNT) | d);
      }
    });
    __syncthreads();
  }
  // running counts and masses over the histogram; the total mass is what is kept at first
  __device__ __forceinline__ void run_sums() {
    u64 n_sum = 0, m_sum = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const u64 h = s.hist[4 * tid + q];
      cnt[q] = h >> SM_COUNT;
      mass[q] = h ? bin_mass(4 * tid + q, h) : 0ULL;  // (most waves have none)
      n_sum += cnt[q];
      m_sum += mass[q];
    }
    u64 n_all;
    n_run = before(n_sum, s.wave, n_all);
    m_run = before(m_sum, s.wave2, kept);
  }
  // the threads' sums before the thread's own, and that of all; `at`: a word for each wave
  __device__ __forceinline__ u64 before(u64 own, u64* at, u64& all) const {
    const u64 run = sm_wave_scan(own);
    if (lane == 63) at[wave] = run;
    __syncthreads();
    u64 x = at[lane & (SM_WAVES - 1)];  // (a row of 16 lanes: each wave's)
    x += sm_dpp<0x111>(x);
    x += sm_dpp<0x112>(x);
    x += sm_dpp<0x114>(x);
    x += sm_dpp<0x118>(x);
    all = sm_lane(x, SM_WAVES - 1);
    return (wave ? sm_lane(x, wave - 1) : 0ULL) + run - own;
  }
  // The bin of a border: where the k-th token is (want), or the last one before which less than P lies;
  // the count and the mass above it. SM_BINS: none.
  __device__ __forceinline__ int find(u64 want, double P, u64& n_above, u64& m_above) {
    __syncthreads();
    if (tid == 0) s.pick[0] = want ? SM_BINS - 1 : SM_BINS, s.pick[1] = s.pick[2] = 0;
    __syncthreads();
    u64 n = n_run, x = m_run;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const bool rest = 4 * tid + q == SM_BINS - 1;
      const bool here = want ? n < want && (rest || want <= n + cnt[q])
                             : cnt[q] && (double)x < P && P <= (double)(x + mass[q]);
      if (here) {
        s.pick[0] = (u64)(4 * tid + q);
        s.pick[1] = n;
        s.pick[2] = x;
      }
      n += cnt[q];
      x += mass[q];
    }
    __syncthreads();
    n_above = s.pick[1];
    m_above = s.pick[2];
    return (int)s.pick[0];
  }
  // The bins b0 .. b1 in which the borders lie, and the count and the mass above them, if one list can
  // hold their tokens. Both borders: what top-k keeps has a mass between that above its bin and that
  // with it, which bounds top-p's bin from above.
  __device__ __forceinline__ bool bins(int& b0, int& b1, u64& n_above, u64& m_above) {
    if (!by_k) {
      b0 = b1 = find(0, (double)tp * (double)kept, n_above, m_above);
      return b0 < SM_BINS && (s.hist[b0] >> SM_COUNT) <= SM_CAND;
    }
    u64 n_k, m_k;
    b0 = b1 = find((u64)k, 0.0, n_k, m_k);
    if (b1 == SM_BINS - 1) return false;
    const u64 n_end = n_k + (s.hist[b1] >> SM_COUNT);
    n_above = n_k;
    m_above = m_k;
    if (by_p) {
      b0 = find(0, (double)tp * (double)max(m_k, 1ULL), n_above, m_above);
      if (b0 > b1) return false;
    }
    return n_end - n_above <= SM_CAND;
  }

  // ---- the mass of each row of pieces, to put(R, mass) ----
  // LISTED: of the tokens above bin b0; those of bins b0 .. b1 go to list(key and ~index). Otherwise of
  // the tokens that are kept.
  template <bool LISTED, class Put, class List>
  __device__ __forceinline__ void masses(int b0, int b1, Put&& put, List&& list) {
    const float x0 = (float)b0, x1 = b1 == SM_BINS - 1 ? INFINITY : (float)(b1 + 1);
    each([&](int R, int i0, const dkv_u32x4& v) {
      u64 sum = 0;
      if (!by_k && !by_p) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float l = value(v, e);
          sum += l > -INFINITY ? floored(weight(l)) : 0ULL;
        }
      } else {
        // bit E - 1 - e of a mask: token e; a bit is the sign of a difference
        uint32_t mask = 0, in = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float l = value(v, e);
          if constexpr (LISTED) {
            float dl;
            const float x = x_of(l, dl);
            mask = __builtin_amdgcn_alignbit(mask, __float_as_uint(x - x0), 31);
            in = __builtin_amdgcn_alignbit(in, __float_as_uint(x - x1), 31);
          } else {
            mask = mask << 1 | (l >= keep.at && is_kept(l, i0 + e) ? 1u : 0u);
          }
        }
        auto token = [&](uint32_t bits) { return E - 1 - (__ffs((int)bits) - 1); };
        auto pick = [&](uint32_t bits) {
          const int e = bits ? token(bits) : 0, w = DT == DKV_F32 ? e : e >> 1;
          const uint32_t a = w & 1 ? v[1] : v[0], b = w & 1 ? v[3] : v[2], x = w & 2 ? b : a;
          if constexpr (DT == DKV_F32)
            return __uint_as_float(x);
          else if constexpr (DT == DKV_BF16)
            return __uint_as_float(e & 1 ? x & 0xffff0000u : x << 16);
          else
            return dkv_f16_bits_to_f32((e & 1 ? x >> 16 : x) & 0xffffu);
        };
        in &= ~mask;
        while (__ballot(mask != 0)) {  // one of each lane's at a time
          const u64 w = floored(weight(pick(mask)));
          sum += mask ? w : 0ULL;
          mask &= mask - 1;
        }
        if constexpr (LISTED) {
          while (in) {
            const float l = pick(in);
            const int i = i0 + token(in);
            if (i >= 0 && i < V && l == l) list(((u64)sm_key(l) << 32) | (uint32_t)~i);
            in &= in - 1;
          }
        }
      }
      sum = sm_wave_sum(sum);
      if (lane == 0) put(R, sum);
    });
  }
  // u times the mass, in whole units of it
  __device__ __forceinline__ u64 target_of(u64 all) const {
    const double U = u > 0.f ? (double)u * (double)all : 0.0;
    return U < (double)all ? min((u64)U, all - 1) : all - 1;
  }
  // the n tokens of s.cand in order
  __device__ __forceinline__ void sort(int n) {
    for (int a = tid; a < n; a += SM_THREADS) {
      const u64 x = s.cand[a];
      int rank = 0;
      for (int b = 0; b < n; ++b) rank += s.cand[b] > x;
      s.sort[rank] = x;
    }
    __syncthreads();
  }
  // Up to the j-th of the n sorted tokens (j > 0), or those before which, with `before`, less than P
  // lies; returns their mass.
  __device__ __forceinline__ u64 border_in(int n, u64 j, u64 before, double P) {
    __syncthreads();
    if (wave == 0) {
      u64 run = 0;
      int last = -1;
      for (int a = 0; a < n; a += 64) {
        const int at = a + lane;
        const u64 w = at < n ? weight(sm_unkey((uint32_t)(s.sort[at] >> 32))) : 0;
        const u64 sum = sm_wave_scan(w);
        const bool in = at < n && (j ? (u64)at < j : (double)(before + run + sum - w) < P);
        const u64 hit = __ballot(in);
        if (!hit) break;
        const int l = 63 - __clzll((long long)hit);
        last = a + l;
        run += __shfl(sum, l, 64);
        if (l < 63) break;
      }
      if (lane == 0) {
        s.pick[0] = last >= 0 ? s.sort[last] : 0;
        s.pick[1] = run;
      }
    }
    __syncthreads();
    // (no token at all: the j-th is a NaN; everything above them is kept)
    keep.at = s.pick[0] ? sm_unkey((uint32_t)(s.pick[0] >> 32)) : -INFINITY;
    keep.last = (int)~(uint32_t)s.pick[0];
    return s.pick[1];
  }
  // The borders among the n sorted tokens, above which count and mass are given; the kept ones' masses
  // join their rows of pieces.
  __device__ __forceinline__ void borders(int n, u64 n_above, u64 m_above) {
    if (by_k) kept = m_above + border_in(n, (u64)k - n_above, 0, 0.0);
    if (by_p) kept = m_above + border_in(n, 0, m_above, (double)tp * (double)kept);
    for (int a = tid; a < n; a += SM_THREADS) {
      const float l = sm_unkey((uint32_t)(s.sort[a] >> 32));
      const int i = (int)~(uint32_t)s.sort[a];
      if (is_kept(l, i)) atomicAdd(&s.chunk[(i + head) / (E * 64)], floored(weight(l)));
    }
    __syncthreads();
  }

  // ---- the border by digits of the keys (11, 11, 10 bits): for a bin of too many tokens ----
  // Level by level the bin in which the border lies, among the tokens that share the digits found so
  // far; then the index of the last of the equal ones that are kept. Clears the histogram.
  __device__ __forceinline__ void by_digits(u64 want, double P) {
    u64 above = 0, m_above = 0;
    uint32_t found = 0;
    u64 ties = 0;
#pragma unroll 1
    for (int level = 0; level < 3; ++level) {
      const int shift = level == 0 ? 21 : level == 1 ? 10 : 0;
      const int bits = level == 2 ? 10 : 11;
      __syncthreads();
      for (int i = tid; i < SM_BINS; i += SM_THREADS) s.hist[i] = 0;
      __syncthreads();
      each([&](int, int i0, const dkv_u32x4& v) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float l = fmaxf(value(v, e), -INFINITY);
          const int i = i0 + e;
          const uint32_t key = sm_key(l);
          const bool on = i >= 0 && i < V && (!level || (key >> (shift + bits)) == found);
          const int bin = (int)((key >> shift) & ((1u << bits) - 1));
          const u64 w = on ? weight(l) : 0ULL;
          // many in one bin (this is where logits are equal) are added up first, as additions to one place
          // wait for each other: 256 rows of 128256 equal fp32 logits 0.65 ms, 1.48 without
          const unsigned long long act = __ballot(on);
          if (!act) continue;
          const int lead = __ffsll((long long)act) - 1;
          const bool same = on && bin == __builtin_amdgcn_readlane(bin, lead);
          const int n = __popcll(__ballot(same));
          const bool many = n > 8;
          if (many) {
            const u64 all = sm_wave_sum(same ? w : 0ULL);
            if (lane == lead) {
              atomicAdd(&s.hist[bin], all);
              atomicAdd(&s.hist[2048 + bin], (u64)n);
            }
          }
          if (on && !(many && same)) {
            atomicAdd(&s.hist[bin], w);
            atomicAdd(&s.hist[2048 + bin], 1ULL);
          }
        }
      });
      if (tid == 0) s.n = -1, s.pick[0] = s.pick[1] = s.pick[2] = s.pick[3] = 0;
      __syncthreads();
      // the bins from the top, two a thread: the last one before which less than wanted lies
      const int top = (1 << bits) - 1;
      u64 c[2], x[2], all;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int bin = top - 2 * tid - q;
        c[q] = bin >= 0 ? s.hist[2048 + bin] : 0ULL;
        x[q] = bin >= 0 ? s.hist[bin] : 0ULL;
      }
      u64 n = above + before(c[0] + c[1], s.wave, all), m = m_above + before(x[0] + x[1], s.wave2, all);
      u64 n_at = 0, m_at = 0, ties_at = 0;
      int at = -1;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        if (c[q] && (want ? n < want : (double)m < P)) {
          at = 2 * tid + q;
          n_at = n;
          m_at = m;
          ties_at = c[q];
        }
        n += c[q];
        m += x[q];
      }
      if (at >= 0) atomicMax(&s.n, at);
      __syncthreads();
      if (at >= 0 && at == s.n) {
        s.pick[0] = (u64)(top - at);
        s.pick[1] = n_at;
        s.pick[2] = m_at;
        s.pick[3] = ties_at;
      }
      __syncthreads();
      found = (found << bits) | (uint32_t)s.pick[0];
      above = s.pick[1];
      m_above = s.pick[2];
      ties = s.pick[3];
    }
    keep.at = sm_unkey(found);
    const u64 w = weight(keep.at);
    if (want) {
      ties = min(ties, want - above);
    } else if (w > 0) {
      u64 lo = 1, hi = ties;  // the equal ones before which less than P lies
      while (lo < hi) {
        const u64 mid = (lo + hi + 1) / 2;
        if ((double)(m_above + (mid - 1) * w) < P)
          lo = mid;
        else
          hi = mid - 1;
      }
      ties = lo;
    }
    kept = m_above + ties * w;
    // the index of the last of them: equal ones by row of pieces, in order
    auto equal = [&](int i0, const dkv_u32x4& v) {
      uint32_t mask = 0;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int i = i0 + e;
        if (i >= 0 && i < V && fmaxf(value(v, e), -INFINITY) == keep.at) mask |= 1u << e;
      }
      return mask;
    };
    __syncthreads();
    for (int i = tid; i < rows64; i += SM_THREADS) s.chunk[i] = 0;
    __syncthreads();
    each([&](int R, int i0, const dkv_u32x4& v) {
      const uint32_t mask = equal(i0, v);
      if (mask) atomicAdd(&s.chunk[R], (u64)__popc(mask));
    });
    __syncthreads();
    if (tid == 0) {
      u64 n = 0;
      int at = 0;
      for (; at < rows64 - 1 && n + s.chunk[at] < ties; ++at) n += s.chunk[at];
      s.pick[0] = (u64)at;
      s.pick[1] = ties - n;  // the one of them in that row of pieces
    }
    __syncthreads();
    if (wave == 0) {
      const int R = (int)s.pick[0], i0 = first_of(R);
      uint32_t mask = equal(i0, load(R));
      const u64 run = sm_wave_scan((u64)__popc(mask)), at = s.pick[1];
      const u64 before = run - (u64)__popc(mask);
      if (before < at && at <= run) {
        for (u64 x = before + 1; x < at; ++x) mask &= mask - 1;
        s.pick[2] = (u64)(i0 + __ffs((int)mask) - 1);
      }
    }
    __syncthreads();
    keep.last = (int)s.pick[2];
    __syncthreads();
  }

  // ---- the borders one after the other, and the masses of what is kept: where one list does not
  // do. The workgroup has the whole row and its histogram. ----
  __device__ __forceinline__ void one_by_one() {
    bool digits = false;
#pragma unroll 1
    for (int step = 0; step < 2; ++step) {  // top-k, then top-p of what it keeps
      if (step == 0 ? !by_k : !by_p) continue;
      const u64 want = step == 0 ? (u64)k : 0;
      const double P = step == 0 ? 0.0 : (double)tp * (double)kept;
      u64 n_above = 0, m_above = 0;
      const int bin = digits ? SM_BINS : find(want, P, n_above, m_above);
      if (bin < SM_BINS) {
        __syncthreads();
        if (tid == 0) s.n = 0;
        __syncthreads();
        masses<true>(bin, bin, [](int, u64) {}, [&](u64 x) {
          const int at = atomicAdd(&s.n, 1);
          if (at < SM_CAND) s.cand[at] = x;
        });
        __syncthreads();
      }
      if (bin < SM_BINS && s.n <= SM_CAND) {
        const int n = s.n;
        sort(n);
        kept = m_above + border_in(n, want ? want - n_above : 0, m_above, P);
      } else {
        by_digits(want, P);
        digits = true;
      }
    }
    __syncthreads();
    masses<false>(0, 0, [&](int R, u64 w) { s.chunk[R] = w; }, [](u64) {});
    __syncthreads();
  }

  // ---- the token in which u times the mass lies ----
  // s.chunk: the masses of the rows of pieces, and from bit SM_TIES on the tokens at a border, the first
  // `ties` of which are kept, of weight tie_w each. weights(piece, its first token, w): the same of a
  // piece's tokens. One wave's work: lane l has rows share * l .. share * (l + 1) - 1.
  template <class F>
  __device__ __forceinline__ void finish(u64 ties, u64 tie_w, F&& weights) const {
    if (wave != 0) return;
    const int share = (rows64 + 63) / 64, c0 = lane * share, c1 = min(rows64, c0 + share);
    u64 own = 0, at = 0;
    for (int i = c0; i < c1; ++i) {
      own += s.chunk[i] & SM_MASS;
      at += s.chunk[i] >> SM_TIES;
    }
    u64 tie0 = 0;  // tokens at the border before the lane's
    if (ties) {
      tie0 = sm_wave_scan(at) - at;
      own += (min(tie0 + at, ties) - min(tie0, ties)) * tie_w;
    }
    u64 run = sm_wave_scan(own);
    const u64 target = target_of(sm_lane(run, 63));
    const int who = __ffsll((long long)__ballot(run > target)) - 1;
    run = sm_lane(run - own, who);
    tie0 = sm_lane(tie0, who);
    int R = who * share;
    for (;; ++R) {
      const u64 c = s.chunk[R], t = c >> SM_TIES;
      const u64 x = (c & SM_MASS) + (min(tie0 + t, ties) - min(tie0, ties)) * tie_w;
      if (run + x > target || R == rows64 - 1) break;
      run += x;
      tie0 += t;
    }
    R = __builtin_amdgcn_readfirstlane(R);
    const int i0 = first_of(R);
    u64 w[E], t = 0, sum = 0;
    weights(load(R), i0, w);
    if (ties) {
#pragma unroll
      for (int e = 0; e < E; ++e) t += w[e] >> SM_TIES;
      tie0 += sm_wave_scan(t) - t;
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (w[e] >> SM_TIES) w[e] = tie0++ < ties ? tie_w : 0ULL;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) sum += w[e];
    run += sm_wave_scan(sum) - sum;
    if (run <= target && target < run + sum) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if (run <= target && target < run + w[e]) p.out[row] = (long long)(i0 + e);
        run += w[e];
      }
    }
  }
  __device__ __forceinline__ void finish() const {
    finish(0, 0, [&](const dkv_u32x4& v, int i0, u64 (&w)[E]) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float l = value(v, e);
        w[e] = is_kept(l, i0 + e) ? floored(weight(l)) : 0ULL;
      }
    });
  }

  // ---- 16-bit logits, the row in one workgroup: by their values ----
  // A row has few distinct logits, so a bin each: its tokens are counted, its weight is worked out once
  // and, for the masses, read from a table; a border is a bin and the tokens at it (the first of them in
  // the vocabulary's order are kept), and nothing is sorted.
  // A bin is the logit's key: its bits without the sign, up to 2^-20 (bf16) or 2^-8 (fp16) all 0, signed.
  // What is next to 0 thus shares a bin with it (halvings of the logit down to 2^-126 would be most of
  // the bins): its tokens' weights differ from that of 0 and are put right one by one.
  static constexpr int NEAR = DT == DKV_BF16 ? (127 - 20) << 7 : (15 - 8) << 10;
  static constexpr int INF = DT == DKV_BF16 ? 0x7f80 : 0x7c00;
  typedef short s2 __attribute__((ext_vector_type(2)));
  typedef unsigned short u2 __attribute__((ext_vector_type(2)));
  // keys of 4096 (bf16) or 64 (fp16): rows without larger logits are counted before their largest is
  // known
  static constexpr int LIMIT = DT == DKV_BF16 ? ((127 + 12) << 7) - NEAR : ((15 + 6) << 10) - NEAR;
  int k_max, k_lo;   // the largest logit's key, and the key of bin 0; bins 0 .. 63 catch what lies below
  int k_low;         // the lowest key that has a weight, or less
  int near_n = 0;    // tokens next to 0
  u64 near_m = 0;    // what their weights are above those of as many at 0 (modulo 2^64)
  static __device__ __forceinline__ s2 keys(uint32_t v) {
    const u2 t = __builtin_bit_cast(u2, v & 0x7fff7fffu);
    const u2 u = __builtin_elementwise_sub_sat(t, u2{(unsigned short)NEAR, (unsigned short)NEAR});
    const s2 sign = __builtin_bit_cast(s2, v) >> 15;
    return (__builtin_bit_cast(s2, u) ^ sign) - sign;
  }
  static __device__ __forceinline__ float of_key(int key) {
    const uint32_t b = (key < 0 ? 0x8000u : 0u) | (key ? (uint32_t)(abs(key) + NEAR) : 0u);
    return DT == DKV_BF16 ? __uint_as_float(b << 16) : dkv_f16_bits_to_f32(b);
  }
  static __device__ __forceinline__ int key_of(float l) {  // (towards 0)
    uint32_t b = __float_as_uint(l) >> 16;
    if constexpr (DT == DKV_F16)
      b = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(fmaxf(l, -65504.f), 0.f));
    return keys(b)[0];
  }
  __device__ __forceinline__ void set_low() {
    // no weight at x = SM_BINS - 1; the key is off by less than 2
    const int low = key_of(fmaxf(m - (float)SM_BINS / c_hi, -3.4028234663852886e38f)) - 2;
    k_low = max(low, -(INF - NEAR) + 1);
  }
  // Whether the row's range of logits has bins, below its largest logit.
  __device__ __forceinline__ bool by_values_fits() {
    k_max = key_of(m);
    set_low();
    k_lo = k_low - 64;
    return k_max - k_lo <= SM_KEYS - 2;
  }
  static __device__ __forceinline__ bool is_near(const dkv_u32x4& v, int e) {
    return ((v[e / 2] >> (16 * (e & 1))) & 0x7fffu) - 1 < (uint32_t)NEAR;
  }
  // f(logit) for the tokens of the piece that are next to 0 and not 0
  template <class F>
  __device__ __forceinline__ void next_to_0(const dkv_u32x4& v, F&& f) const {
    u2 least = {0xffff, 0xffff};
#pragma unroll
    for (int i = 0; i < 4; ++i)  // (0 itself wraps)
      least = __builtin_elementwise_min(
          least, __builtin_bit_cast(u2, v[i] & 0x7fff7fffu) - u2{1, 1});
    if (min(least[0], least[1]) >= NEAR) return;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (is_near(v, e)) f(value(v, e));
  }
  // The tokens by their key, from k_lo on; what is above bin `top` goes to it.
  __device__ __forceinline__ void count_values(int top) {
    for (int i = 4 * tid; i <= top; i += 4 * SM_THREADS)
      *(dkv_u32x4*)&s.bins[i] = dkv_u32x4{0u, 0u, 0u, 0u};
    __syncthreads();
    const s2 lo = {(short)k_lo, (short)k_lo}, own = {(short)lane, (short)lane},
             end = {(short)top, (short)top};
    each([&](int, int, const dkv_u32x4& v) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const s2 k = __builtin_elementwise_min(
            __builtin_elementwise_max(__builtin_elementwise_sub_sat(keys(v[i]), lo), own), end);
        const uint32_t b = __builtin_bit_cast(uint32_t, k);
        atomicAdd(&s.bins[b & 0xffffu], 1u);
        atomicAdd(&s.bins[b >> 16], 1u);
      }
    });
    __syncthreads();
  }
  // The same before the row's largest logit is known, which is then the last bin that is not empty;
  // false where it has to be found by itself.
  __device__ __forceinline__ bool count_first() {
    constexpr int TOP = 2 * LIMIT + 65;  // above LIMIT: too large, infinite or NaN
    k_lo = -LIMIT - 64;
    keep_root();
    count_values(TOP);
    int best = 0;
    for (int i = 64 + tid; i < TOP; i += SM_THREADS) best = s.bins[i] ? i : best;
    best = (int)dkv_wave_max_fast((float)best);
    if (lane == 0) s.wave[wave] = (u64)best;
    __syncthreads();
    best = (int)dkv_wave_max_fast((float)s.wave[lane & (SM_WAVES - 1)]);
    const uint32_t over = s.bins[TOP];
    __syncthreads();
    best = __builtin_amdgcn_readfirstlane(best);
    k_max = best + k_lo;
    if (over || best < 64 || k_max == 0) return false;
    m = of_key(k_max);
    set_scale();
    set_low();
    return k_low >= -LIMIT;
  }
  // the weights of tokens next to 0
  __device__ __forceinline__ void weigh_near() {
    if (!count_at(-k_lo) || k_low > 0) return;
    const u64 w0 = weight(0.f);
    __syncthreads();
    if (tid == 0) s.n = 0, s.pick[3] = 0;
    __syncthreads();
    each([&](int, int, const dkv_u32x4& v) {
      next_to_0(v, [&](float l) {
        atomicAdd(&s.pick[3], weight(l) - w0);
        atomicAdd(&s.n, 1);
      });
    });
    __syncthreads();
    near_n = s.n;
    near_m = s.pick[3];
  }
  __device__ __forceinline__ uint32_t count_at(int bin) const {
    return bin >= 64 && bin <= k_max - k_lo ? s.bins[bin] : 0u;
  }
  __device__ __forceinline__ u64 mass_at(int bin, uint32_t n) const {
    return (u64)n * weight(of_key(bin + k_lo)) + (bin == -k_lo ? near_m : 0ULL);
  }
  // Bins in order: d of them below the largest logit's. `end`, `end_n`: the last of them that are taken
  // and its tokens that are (top-k's border).
  __device__ __forceinline__ uint32_t count_d(int d, int end, uint32_t end_n) const {
    const uint32_t n = count_at(k_max - k_lo - d);
    return d < end ? n : d == end ? min(n, end_n) : 0u;
  }
  __device__ __forceinline__ u64 mass_d(int d, uint32_t n) const {
    return n ? mass_at(k_max - k_lo - d, n) : 0ULL;
  }
  // A border among the bins up to `end`, which is moved to it: thread t has bins per * t .. per * (t +
  // 1) - 1 (per odd: no two lanes in a bank); the one whose counts (BY_MASS: masses) the border lies in
  // writes its number, and its bins are looked at by lane.
  template <bool BY_MASS>
  __device__ __forceinline__ bool border(int& end, uint32_t& end_n) {
    const int per = ((end + SM_THREADS) / SM_THREADS) | 1;
    u64 own = 0, all;
    for (int d = per * tid; d < min(per * (tid + 1), end + 1); ++d) {
      const uint32_t n = count_d(d, end, end_n);
      own += BY_MASS ? mass_d(d, n) : (u64)n;
    }
    if (tid == 0) s.pick[0] = ~0ULL;
    const u64 run = before(own, BY_MASS ? s.wave2 : s.wave, all);
    const double P = (double)tp * (double)all;
    auto early = [&](u64 x) { return BY_MASS ? (double)x < P : x < (u64)k; };
    if (own && early(run) && !early(run + own)) {
      s.pick[0] = (u64)tid;
      s.pick[1] = run;
    }
    __syncthreads();
    const u64 who = s.pick[0], run0 = s.pick[1];
    if (who == ~0ULL) return false;
    __syncthreads();
    if (wave == 0) {
      const int d = per * (int)who + lane;
      const uint32_t n = lane < per ? count_d(d, end, end_n) : 0u;
      const u64 x = BY_MASS ? mass_d(d, n) : (u64)n;
      const u64 first = run0 + sm_wave_scan(x) - x;
      const unsigned long long hit = __ballot(n && early(first));
      if (lane == 63 - __clzll((long long)hit)) {
        u64 j = n;
        if constexpr (BY_MASS) {
          const u64 w = weight(of_key(k_max - d));
          if (w) {  // those before which less than P lies
            j = min(j, (u64)fmax((P - (double)first) / (double)w, 1.0));
            while (j > 1 && !early(first + (j - 1) * w)) --j;
            while (j < n && early(first + j * w)) ++j;
          }
        } else {
          j = min(j, (u64)k - first);
        }
        s.pick[2] = (u64)d;
        s.pick[3] = j;
      }
    }
    __syncthreads();
    end = (int)s.pick[2];
    end_n = (uint32_t)s.pick[3];
    return true;
  }
  // The piece's tokens less than n keys below the largest: their masses, and those at n as at_border.
  template <bool TABLE, class F>
  __device__ __forceinline__ void value_weights(const dkv_u32x4& v, uint32_t n, u64 at_border,
                                                F&& f) const {
    const u2 top = {(unsigned short)k_max, (unsigned short)k_max};
    const u2 end = {(unsigned short)(n + 1), (unsigned short)(n + 1)};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // (a NaN's is larger than n)
      const u2 d = top - __builtin_bit_cast(u2, keys(v[i]));
      if constexpr (TABLE) {
        const uint32_t b = __builtin_bit_cast(uint32_t, __builtin_elementwise_min(d, end));
        f(2 * i, s.table[b & 0xffffu]);
        f(2 * i + 1, s.table[b >> 16]);
      } else {
#pragma unroll
        for (int q = 0; q < 2; ++q)
          f(2 * i + q,
            d[q] < n ? floored(weight(value(v, 2 * i + q))) : d[q] == n ? at_border : 0ULL);
      }
    }
  }
  // The masses of the rows of pieces, and the number of tokens at the border (`ties` of which are kept,
  // of weight tie_w), then the token in which u times the mass lies.
  template <bool TABLE>
  __device__ __forceinline__ void by_weights(uint32_t n, u64 ties, u64 tie_w) {
    const u64 at_border = ties ? 1ULL << SM_TIES : 0ULL, w0 = floored(weight(0.f));
    if constexpr (TABLE) {
      __syncthreads();  // (the bins' memory)
      for (uint32_t i = tid; i < n; i += SM_THREADS)
        s.table[i] = floored(weight(of_key(k_max - (int)i)));
      if (tid < 2) s.table[n + tid] = tid ? 0ULL : at_border;
      __syncthreads();
    }
    const bool near = TABLE && near_n && k_max >= 0 && (uint32_t)k_max < n;
    auto sum_of = [&](const dkv_u32x4& v) {
      u64 sum = 0;
      value_weights<TABLE>(v, n, at_border, [&](int, u64 w) { sum += w; });
      if (near) next_to_0(v, [&](float l) { sum += floored(weight(l)) - w0; });
      return sum;
    };
    // four rows' sums are brought together in a step of two halves, one of two rows of 16, four within
    // those: row R + 2 ((lane / 16) % 2) + lane / 32 of the four
#pragma unroll 1
    for (int R = r0; R < r1; R += 4) {
      dkv_u32x4 v[4];
      u64 x[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] = load(min(R + q, r1 - 1));
#pragma unroll
      for (int q = 0; q < 4; ++q) x[q] = R + q < r1 ? sum_of(v[q]) : 0ULL;
      u64 sum = sm_meet16(sm_meet32(x[0], x[1]), sm_meet32(x[2], x[3]));
      sum += sm_dpp<0xb1>(sum);
      sum += sm_dpp<0x4e>(sum);
      sum += sm_dpp<0x141>(sum);
      sum += sm_dpp<0x140>(sum);
      const int at = R + (lane >> 4 & 1) * 2 + (lane >> 5);
      if ((lane & 15) == 0 && at < r1) s.chunk[at] = sum;
    }
    __syncthreads();
    finish(ties, tie_w, [&](const dkv_u32x4& v, int, u64 (&w)[E]) {
      value_weights<TABLE>(v, n, at_border, [&](int e, u64 x) { w[e] = x; });
      if (near) {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (is_near(v, e)) w[e] = floored(weight(value(v, e)));
      }
    });
  }
  // The whole of it, of a row that is counted; false where the borders are among the tokens next to 0.
  __device__ __forceinline__ bool by_values() {
    int end = k_max - k_low;  // the last bin that has a weight
    uint32_t end_n = 0;       // its tokens that are kept, where it is a border
    bool found = false;
    if (by_k || by_p) {
      weigh_near();
      end_n = ~0u;
      if (by_k && border<false>(end, end_n)) {
        found = true;
        if (end == k_max && near_n) return false;
      }
      if (by_p && border<true>(end, end_n)) {
        found = true;
        if (end == k_max && near_n) return false;
      }
    } else {
      near_n = 1;  // (unknown)
    }
    const uint32_t n = found ? (uint32_t)end : (uint32_t)(end + 1);
    const u64 ties = found ? end_n : 0ULL, tie_w = floored(weight(of_key(k_max - end)));
    if (n <= (uint32_t)min(SM_TABLE, V))
      by_weights<true>(n, ties, tie_w);
    else
      by_weights<false>(n, ties, tie_w);
    return true;
  }
};

// A row per workgroup.
template <int DT>
__global__ __launch_bounds__(SM_THREADS) void sample_rows_kernel(SampleParams p) {
  __shared__ SampleShared<DT> s;
  RowSampler<DT> r(p, s, blockIdx.x);
  r.take(0, 1);
  if constexpr (DT != DKV_F32)
    if ((r.by_k || r.by_p) && !r.greedy() && r.count_first() && r.by_values()) return;
  if (!r.begin(r.largest(), true)) return;
  if constexpr (DT != DKV_F32) {
    if (r.by_values_fits()) {
      if (r.by_k || r.by_p) r.count_values(r.k_max - r.k_lo + 1);
      if (r.by_values()) return;
    }
  }
  if (r.by_k || r.by_p) {
    r.histogram();
    r.run_sums();
    int b0, b1;
    u64 n_above, m_above;
    if (r.bins(b0, b1, n_above, m_above)) {
      if (threadIdx.x == 0) s.n = 0;
      __syncthreads();
      r.template masses<true>(b0, b1, [&](int R, u64 w) { s.chunk[R] = w; },
                              [&](u64 x) { s.cand[atomicAdd(&s.n, 1)] = x; });
      __syncthreads();
      const int n = s.n;
      r.sort(n);
      r.borders(n, n_above, m_above);
    } else {
      r.one_by_one();
    }
  } else {
    r.template masses<false>(0, 0, [&](int R, u64 w) { s.chunk[R] = w; }, [](u64) {});
    __syncthreads();
  }
  r.finish();
}

// A part of a row per workgroup, a launch per pass: 0 the maxima (and a clear workspace), 1 the
// histogram, 2 the masses, after which the row's last workgroup to arrive ends it.
template <int DT, int PASS>
__global__ __launch_bounds__(SM_THREADS) void sample_parts_kernel(SampleParams p) {
  __shared__ SampleShared<DT> s;
  const int row = blockIdx.x / p.parts, part = blockIdx.x % p.parts, tid = threadIdx.x;
  u64* ws = p.ws + (long long)row * SM_WS;
  RowSampler<DT> r(p, s, row);
  r.take(part, p.parts);
  if constexpr (PASS == 0) {
    const u64 best = r.largest();
    if (tid == 0) ws[part] = best;
    if (part == 0 && tid == 0) ws[SM_WS_N] = 0;
    for (int i = part * SM_THREADS + tid; i < SM_BINS; i += p.parts * SM_THREADS)
      ws[SM_WS_HIST + i] = 0;
    return;
  }
  u64 best = (tid & 63) < p.parts ? ws[tid & 63] : 0;
  dkv_u64x2 h[2];  // the histogram's bins 4 tid .. 4 tid + 3
  if constexpr (PASS == 2) {
#pragma unroll
    for (int q = 0; q < 2; ++q) h[q] = ((const dkv_u64x2*)(ws + SM_WS_HIST))[2 * tid + q];
  }
  r.keep_root();
#pragma unroll
  for (int o = 8; o >= 1; o >>= 1) best = max(best, __shfl_xor(best, o, 64));
  best = __shfl(best, 0, 64);
  __syncthreads();  // (the table of roots)
  if (!r.begin(best, PASS == 1 && part == 0)) return;
  const bool filters = r.by_k || r.by_p;
  if constexpr (PASS == 1) {
    if (!filters) return;
    r.histogram();
    for (int i = tid; i < SM_BINS; i += SM_THREADS)
      if (s.hist[i]) atomicAdd(&ws[SM_WS_HIST + i], s.hist[i]);
    return;
  }
  int b0 = 0, b1 = 0;
  u64 n_above = 0, m_above = 0;
  bool listed = false;
  if (filters) {
#pragma unroll
    for (int q = 0; q < 2; ++q) ((dkv_u64x2*)s.hist)[2 * tid + q] = h[q];
    __syncthreads();
    r.run_sums();
    listed = r.bins(b0, b1, n_above, m_above);
    if (!listed) {  // one workgroup goes on with the whole row
      if (part) return;
      r.take(0, 1);
      r.one_by_one();
      r.finish();
      return;
    }
  }
  uint32_t* counts = (uint32_t*)(ws + SM_WS_N);  // listed tokens, parts that are done
  auto put = [&](int R, u64 w) { sm_put(ws + SM_WS_CHUNK + R, w); };
  if (listed)
    r.template masses<true>(b0, b1, put, [&](u64 x) {
      sm_put(ws + SM_WS_CAND + atomicAdd(&counts[0], 1u), x);
    });
  else
    r.template masses<false>(0, 0, put, [](u64) {});
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (tid == 0) s.last = atomicAdd(&counts[1], 1u) == (uint32_t)p.parts - 1;
  __syncthreads();
  if (!s.last) return;
  const int n = listed ? (int)__hip_atomic_load(&counts[0], __ATOMIC_RELAXED,
                                                __HIP_MEMORY_SCOPE_AGENT)
                       : 0;
  for (int i = tid; i < r.rows64; i += SM_THREADS) s.chunk[i] = sm_get(ws + SM_WS_CHUNK + i);
  for (int i = tid; i < n; i += SM_THREADS) s.cand[i] = sm_get(ws + SM_WS_CAND + i);
  __syncthreads();
  if (listed) {
    r.sort(n);
    r.borders(n, n_above, m_above);
  }
  r.finish();
}

// Workgroups of a row: rows for half the CUs have one each, fewer are cut so that the workgroups fill
// the chip, if each of the 16 waves would have ten rows of pieces or more. The launches and the parts'
// meeting cost 8 us. us, top-p, cut / whole: 37 rows of 50257 fp32 27.6 / 34.5, 64 rows of 32000 fp32
// 27.4 / 25.6. 16-bit rows in one workgroup go by their values, which parts do not, and are cut into
// eight or more: bf16, top-k, top-p and both, one row of 200000 (12 parts) 20.7, 28.5, 22.3 / 33.2, 35.7,
// 35.3; of 128256 (7) 21.0, 27.5, 21.9 / 23.7, 26.4, 25.6; 16 such rows 23.2, 29.9, 25.5 / 24.3, 26.9, 26.4.
int sample_parts(int rows, int V, int dtype) {
  const int tokens = (dtype == DKV_F32 ? 4 : 8) * 64;
  const int rows64 = (V + tokens - 1) / tokens;
  if (rows64 < 10 * SM_WAVES || rows < 1) return 1;
  int n = 256 / rows;
  if (n > SM_PARTS) n = SM_PARTS;
  if (n > rows64 / (2 * SM_WAVES)) n = rows64 / (2 * SM_WAVES);
  return n < (dtype == DKV_F32 ? 2 : 8) ? 1 : n;
}

template <int DT>
void launch_sample(const SampleParams& p, int rows, hipStream_t st) {
  const dim3 block(SM_THREADS), grid((unsigned)(rows * p.parts));
  if (p.parts == 1) {
    hipLaunchKernelGGL(sample_rows_kernel<DT>, grid, block, 0, st, p);
    return;
  }
  hipLaunchKernelGGL((sample_parts_kernel<DT, 0>), grid, block, 0, st, p);
  hipLaunchKernelGGL((sample_parts_kernel<DT, 1>), grid, block, 0, st, p);
  hipLaunchKernelGGL((sample_parts_kernel<DT, 2>), grid, block, 0, st, p);
}

}  // namespace

extern "C" long long dkv_sample_workspace_bytes(int dtype, int rows, int V) {
  if (rows <= 0 || V <= 0 || V > SM_MAX_V) return 0;
  return sample_parts(rows, V, dtype) > 1 ? (long long)rows * SM_WS * (long long)sizeof(u64) : 0;
}

extern "C" int dkv_sample_tokens(void* stream, int dtype, const void* logits, long long ld,
                                 int rows, int V, const float* u, const float* temperature,
                                 float temperature_all, const int* top_k, int top_k_all,
                                 const float* top_p, float top_p_all, const float* min_p,
                                 float min_p_all, void* workspace, long long workspace_bytes,
                                 long long* out) {
  if (dtype != DKV_F16 && dtype != DKV_BF16 && dtype != DKV_F32) return DKV_E_UNSUPPORTED;
  if (rows < 0 || V <= 0) return DKV_E_ARG;
  if (V > SM_MAX_V) return DKV_E_UNSUPPORTED;
  if (rows == 0) return DKV_OK;
  if (!logits || !u || !out || ld < 0 || (rows > 1 && ld < V)) return DKV_E_ARG;
  const long long need = dkv_sample_workspace_bytes(dtype, rows, V);
  if (need > 0 && (!workspace || workspace_bytes < need)) return DKV_E_WORKSPACE;
  if ((uintptr_t)workspace & 15) return DKV_E_UNSUPPORTED;
  SampleParams p;
  p.logits = logits;
  p.ld = ld;
  p.V = V;
  p.u = u;
  p.temperature = temperature;
  p.top_k = top_k;
  p.top_p = top_p;
  p.min_p = min_p;
  p.temperature_all = temperature_all;
  p.top_k_all = top_k_all;
  p.top_p_all = top_p_all;
  p.min_p_all = min_p_all;
  p.out = out;
  p.ws = (u64*)workspace;
  p.parts = sample_parts(rows, V, dtype);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == DKV_F32)
    launch_sample<DKV_F32>(p, rows, st);
  else if (dtype == DKV_BF16)
    launch_sample<DKV_BF16>(p, rows, st);
  else
    launch_sample<DKV_F16>(p, rows, st);
  DKV_HIP_CHECK_LAUNCH();
  return DKV_OK;
}
