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
// One workgroup of 1024 threads per row, which goes over the row four times (from the caches after the
// first): the maximum; a histogram of the tokens by i (counts and sums of d in one 64-bit number, so that a bin's mass is
// known), in which the borders' bins are found; the tokens of a border's bin sorted in LDS; the kept
// mass of every 512 tokens (256 in fp32), in the vocabulary's order; the token. Bound by vector
// instructions: a row's 128256 tokens in one CU take 0.85 us an instruction.
#include "dkv_common.h"

namespace {

typedef unsigned long long u64;

constexpr int SM_THREADS = 1024;
constexpr int SM_WAVES = SM_THREADS / 64;
constexpr int SM_POINT = 44;             // bits after the point of a weight
constexpr int SM_MAX_V = 1 << 19;        // weights of at most 1: sums below 2^63
constexpr int SM_AHEAD = 4;              // 16-byte pieces that a thread has in flight
constexpr int SM_BINS = 4096;            // bins of 1/64 in log2 of the weight; the last: the rest
constexpr int SM_CAND = 2048;            // tokens of a border's bin that are sorted
constexpr int SM_CHUNKS = SM_WAVES * (SM_MAX_V / 4 / SM_THREADS + 1);  // 1 KB pieces of a row
constexpr int SM_COUNT = 44;             // a bin: the count from this bit on, below it the sum of d
constexpr uint32_t SM_OFF = 1u << 13;    // added to d, which may be as low as -2^-19
constexpr double SM_ONE = 17592186044416.0;  // 2^44

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
};

// A logit as a number that orders as the logits do (-0 as +0).
__device__ __forceinline__ uint32_t sm_key(float f) {
  const uint32_t b = __float_as_uint(f + 0.0f);
  return b ^ ((int)b < 0 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float sm_unkey(uint32_t k) {
  return __uint_as_float(k ^ ((int)k < 0 ? 0x80000000u : 0xffffffffu));
}

__device__ __forceinline__ u64 sm_wave_scan(u64 v, int lane) {  // inclusive
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const u64 x = __shfl_up(v, o, 64);
    if (lane >= o) v += x;
  }
  return v;
}
template <int CTRL>
__device__ __forceinline__ u64 sm_dpp(u64 v) {
  return (uint32_t)dkv_dpp_i32<CTRL>((int)(uint32_t)v) |
         ((u64)(uint32_t)dkv_dpp_i32<CTRL>((int)(uint32_t)(v >> 32)) << 32);
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

// What is kept: every token above `key`, and those at it up to index `last`.
struct Border {
  float at;
  int last;
};

template <int DT>
__global__ __launch_bounds__(SM_THREADS) void sample_kernel(SampleParams p) {
  constexpr int E = DT == DKV_F32 ? 4 : 8;  // elements of a 16-byte piece
  __shared__ u64 sHist[SM_BINS];
  __shared__ u64 sCand[SM_CAND];
  __shared__ u64 sSort[SM_CAND];
  __shared__ u64 sChunk[SM_CHUNKS];
  __shared__ uint32_t sRoot[64];
  __shared__ u64 sWave[SM_WAVES];
  __shared__ u64 sWave2[SM_WAVES];
  __shared__ float sMax[SM_WAVES];
  __shared__ u64 sPick[4];
  __shared__ int sN;
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int V = p.V;
  const char* base = (const char*)p.logits + (long long)row * p.ld * (DT == DKV_F32 ? 4 : 2);
  const float t = p.temperature ? p.temperature[row] : p.temperature_all;
  const int k = p.top_k ? p.top_k[row] : p.top_k_all;
  const float tp = p.top_p ? p.top_p[row] : p.top_p_all;
  const float mp = p.min_p ? p.min_p[row] : p.min_p_all;

  // ---- the row: pieces of 16 aligned bytes, a wave's consecutive ----
  const int head = (int)((uintptr_t)base & 15) / (16 / E);  // elements of the first piece before it
  const int pieces = (V + head + E - 1) / E;
  const int per_wave = (pieces + SM_THREADS - 1) / SM_THREADS;  // of 64 pieces each
  auto first_of = [&](int c) { return ((wave * per_wave + c) * 64 + lane) * E - head; };
  // piece c of the thread as its words; elements outside the row are -infinity
  auto load = [&](int c) {
    const int i0 = first_of(c);
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
    return v;
  };
  // In a row with logits of +infinity those share the mass: they are read as 0, the others as
  // -infinity.
  bool infinite = false;
  auto remap = [&](dkv_u32x4 v) {
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
    return v;
  };
  auto value = [&](const dkv_u32x4& v, int e) {
    if constexpr (DT == DKV_F32)
      return __uint_as_float(v[e]);
    else if constexpr (DT == DKV_BF16)
      return __uint_as_float(e & 1 ? v[e / 2] & 0xffff0000u : v[e / 2] << 16);
    else
      return dkv_f16_bits_to_f32(e & 1 ? v[e / 2] >> 16 : v[e / 2] & 0xffffu);
  };
  auto load_again = [&](int c) {
    const dkv_u32x4 v = load(c);
    return infinite ? remap(v) : v;
  };
  // f(c, its first token, the piece) for each of the thread's pieces, in order
  auto each = [&](auto&& f) {
#pragma unroll 1
    for (int c = 0; c < per_wave; c += SM_AHEAD) {
      dkv_u32x4 v[SM_AHEAD];
#pragma unroll
      for (int q = 0; q < SM_AHEAD; ++q)
        if (c + q < per_wave) v[q] = load_again(c + q);
#pragma unroll
      for (int q = 0; q < SM_AHEAD; ++q)
        if (c + q < per_wave) f(c + q, first_of(c + q), v[q]);
    }
  };

  // ---- the largest logit ----
  float m = -INFINITY;
  each([&](int, int, const dkv_u32x4& v) {
#pragma unroll
    for (int e = 0; e < E; ++e) m = fmaxf(m, value(v, e));  // (a NaN is passed over)
  });
  m = dkv_wave_max(m);
  if (lane == 0) sMax[wave] = m;
  if (tid == 0) sN = 0x7fffffff;
  if (tid < 64) sRoot[tid] = (uint32_t)rint(exp2(31.0 - (double)tid / 64.0));
  __syncthreads();
  for (int w = 0; w < SM_WAVES; ++w) m = fmaxf(m, sMax[w]);
  if (m == -INFINITY) {
    if (tid == 0) p.out[row] = -1;
    return;
  }
  if (!(t > 0.f) || k == 1 || tp <= 0.f || mp > 1.f) {  // the first token alone
    int at = 0x7fffffff;
    each([&](int c, int i0, const dkv_u32x4& v) {
#pragma unroll
      for (int e = E - 1; e >= 0; --e)
        if (value(v, e) == m) at = min(at, i0 + e);
    });
    if (at != 0x7fffffff) atomicMin(&sN, at);
    __syncthreads();
    if (tid == 0) p.out[row] = sN;
    return;
  }
  if (m == INFINITY) {
    infinite = true;
    m = 0.f;
  }
  const double c64 = 64.0 * 1.4426950408889634074 / (double)fminf(fmaxf(t, 1e-30f), 1e30f);

  const float c_hi = (float)c64, c_lo = (float)(c64 - (double)c_hi);

  // The bin of a logit; `d`: 2^31 d + SM_OFF. (NaN: the last bin.) Of max l - l, which is rounded,
  // fp32 logits take what the rounding left; 16-bit ones are exact but for some next to 0.
  auto bin_at = [&](float l, float& dl, float& x) {
    dl = m - l;
    x = fminf(dl * c_hi, (float)(SM_BINS - 1));
    return (int)x;
  };
  auto bin_of = [&](float l) {
    float dl, x;
    return bin_at(l, dl, x);
  };
  auto split = [&](float l, int& i, uint32_t& d) {
    float dl, x;
    i = bin_at(l, dl, x);
    float r = fmaf(dl, c_lo, fmaf(dl, c_hi, -x));
    if constexpr (DT == DKV_F32) r = fmaf((m - dl) - l, c_hi, r);
    const float f = __builtin_amdgcn_fractf(x) + r;
    // 2^31 (1 - 2^(-f/64)): with g = ln2 / 64, g f - (g f)^2 / 2 + (g f)^3 / 6 - (g f)^4 / 24
    constexpr double g = 0.69314718055994530942 / 64, one = 2147483648.0;
    const float s = fmaf(
        f, fmaf(f, fmaf(f, fmaf(f, (float)(-g * g * g * g / 24 * one), (float)(g * g * g / 6 * one)),
                        (float)(-g * g / 2 * one)),
                (float)(g * one)),
        (float)SM_OFF);
    d = (uint32_t)s;
  };
  // the weight of a logit, in 2^-44
  auto weight = [&](float l) {
    int i;
    uint32_t d;
    split(l, i, d);
    const u64 w = (u64)sRoot[i & 63] * (u64)(uint32_t)((1u << 31) + SM_OFF - d);  // 2^62 w
    return i == SM_BINS - 1 ? 0ULL : w >> min((62 - SM_POINT) + (i >> 6), 63);
  };
  // the mass of a bin
  auto bin_mass = [&](int i, u64 h) {
    const double n = (double)(h >> SM_COUNT);
    const double d = (double)(h & ((1ULL << SM_COUNT) - 1)) - n * (double)SM_OFF;
    const double w = (double)sRoot[i & 63] * (n - d * (1.0 / 2147483648.0));  // 2^31 w
    return i == SM_BINS - 1 ? 0ULL : (u64)rint(ldexp(w, SM_POINT - 31 - (i >> 6)));
  };

  const bool by_k = k > 0 && k < V, by_p = tp < 1.f;
  Border keep = {-INFINITY, -1};
  u64 kept = 0;  // the mass of what is kept so far

  // ---- the borders inside bins: the n tokens of bins b0 .. b1 (at most SM_CAND) sorted ----
  int sorted = 0;
  auto sort_bins = [&](int b0, int b1) {
    __syncthreads();
    if (tid == 0) sN = 0;
    __syncthreads();
    each([&](int c, int i0, const dkv_u32x4& v) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float l = value(v, e);
        const int bin = bin_of(l);
        if (bin >= b0 && bin <= b1) {
          const int i = i0 + e;
          if (i >= 0 && i < V && l == l) {
            const int at = atomicAdd(&sN, 1);
            if (at < SM_CAND) sCand[at] = ((u64)sm_key(l) << 32) | (uint32_t)~i;
          }
        }
      }
    });
    __syncthreads();
    sorted = sN;
    if (sorted > SM_CAND) return false;
    for (int a = tid; a < sorted; a += SM_THREADS) {
      const u64 x = sCand[a];
      int rank = 0;
      for (int b = 0; b < sorted; ++b) rank += sCand[b] > x;
      sSort[rank] = x;
    }
    __syncthreads();
    return true;
  };
  // Up to the j-th of the sorted tokens (j > 0), or those before which, with `before`, less than P
  // lies; `mass`: theirs.
  auto border_in = [&](u64 j, u64 before, double P, Border& r, u64& mass) {
    __syncthreads();
    if (wave == 0) {
      u64 run = 0;
      int last = -1;
      for (int a = 0; a < sorted; a += 64) {
        const int at = a + lane;
        const u64 w = at < sorted ? weight(sm_unkey((uint32_t)(sSort[at] >> 32))) : 0;
        const u64 sum = sm_wave_scan(w, lane);
        const bool in = at < sorted && (j ? (u64)at < j : (double)(before + run + sum - w) < P);
        const u64 hit = __ballot(in);
        if (!hit) break;
        const int l = 63 - __clzll((long long)hit);
        last = a + l;
        run += __shfl(sum, l, 64);
        if (l < 63) break;
      }
      if (lane == 0) {
        sPick[0] = last >= 0 ? sSort[last] : 0;
        sPick[1] = run;
      }
    }
    __syncthreads();
    // (no token at all: the j-th is a NaN; everything above them is kept)
    r.at = sPick[0] ? sm_unkey((uint32_t)(sPick[0] >> 32)) : -INFINITY;
    r.last = (int)~(uint32_t)sPick[0];
    mass = sPick[1];
  };

  // ---- the border by digits of the keys (11, 11, 10 bits): for a bin of too many tokens ----
  // Level by level the bin in which the border lies, among the tokens that share the digits found so
  // far; then the index of the last of the equal ones that are kept. Clears the histogram.
  auto by_digits = [&](u64 want, double P, Border& r, u64& mass_kept) {
    u64 above = 0, m_above = 0;
    uint32_t found = 0;
    u64 ties = 0;
    for (int level = 0; level < 3; ++level) {
      const int shift = level == 0 ? 21 : level == 1 ? 10 : 0;
      const int bits = level == 2 ? 10 : 11;
      __syncthreads();
      for (int i = tid; i < SM_BINS; i += SM_THREADS) sHist[i] = 0;
      __syncthreads();
      each([&](int c, int i0, const dkv_u32x4& v) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float l = fmaxf(value(v, e), -INFINITY);
          const int i = i0 + e;
          if (i < 0 || i >= V) continue;
          const uint32_t key = sm_key(l);
          if (level && (key >> (shift + bits)) != found) continue;
          const int bin = (int)((key >> shift) & ((1u << bits) - 1));
          atomicAdd(&sHist[bin], weight(l));
          atomicAdd(&sHist[2048 + bin], 1ULL);
        }
      });
      __syncthreads();
      if (tid == 0) {  // the bins from the top
        u64 cnt = above, mass = m_above, cnt_at = 0, mass_at = 0;
        int at = 0;
        for (int bin = (1 << bits) - 1; bin >= 0; --bin) {
          if (!sHist[2048 + bin]) continue;
          if (!(want ? cnt < want : (double)mass < P)) break;
          at = bin;
          cnt_at = cnt;
          mass_at = mass;
          cnt += sHist[2048 + bin];
          mass += sHist[bin];
        }
        sPick[0] = (u64)at;
        sPick[1] = cnt_at;
        sPick[2] = mass_at;
        sPick[3] = sHist[2048 + at];
      }
      __syncthreads();
      found = (found << bits) | (uint32_t)sPick[0];
      above = sPick[1];
      m_above = sPick[2];
      ties = sPick[3];
    }
    r.at = sm_unkey(found);
    const u64 w = weight(r.at);
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
    mass_kept = m_above + ties * w;
    // the index of the last of them: equal ones by piece row, in order
    __syncthreads();
    for (int i = tid; i < SM_CHUNKS; i += SM_THREADS) sChunk[i] = 0;
    __syncthreads();
    each([&](int c, int i0, const dkv_u32x4& v) {
      int n = 0;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int i = i0 + e;
        n += i >= 0 && i < V && fmaxf(value(v, e), -INFINITY) == r.at;
      }
      if (n) atomicAdd(&sChunk[wave * per_wave + c], (u64)n);
    });
    __syncthreads();
    if (tid == 0) {
      u64 cnt = 0;
      int at = 0;
      for (; at < SM_WAVES * per_wave - 1 && cnt + sChunk[at] < ties; ++at) cnt += sChunk[at];
      sPick[0] = (u64)at;
      sPick[1] = ties - cnt;  // the one of them in that piece row
    }
    __syncthreads();
    if ((int)sPick[0] / per_wave == wave) {
      const int c = (int)sPick[0] % per_wave;
      const dkv_u32x4 v = load_again(c);
      const int i0 = first_of(c);
      uint32_t mask = 0;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int i = i0 + e;
        if (i >= 0 && i < V && fmaxf(value(v, e), -INFINITY) == r.at) mask |= 1u << e;
      }
      const u64 run = sm_wave_scan((u64)__popc(mask), lane), want_at = sPick[1];
      const u64 before = run - (u64)__popc(mask);
      if (before < want_at && want_at <= run) {
        for (u64 x = before + 1; x < want_at; ++x) mask &= mask - 1;
        sPick[2] = (u64)(i0 + __ffs((int)mask) - 1);
      }
    }
    __syncthreads();
    r.last = (int)sPick[2];
    __syncthreads();
  };

  if (by_k || by_p) {
    // ---- the histogram ----
    for (int i = tid; i < SM_BINS; i += SM_THREADS) sHist[i] = 0;
    __syncthreads();
    each([&](int c, int i0, const dkv_u32x4& v) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        int i;
        uint32_t d;
        split(value(v, e), i, d);
        if (i < SM_BINS - 1) atomicAdd(&sHist[i], (1ULL << SM_COUNT) | d);
      }
    });
    __syncthreads();
    // running counts and masses: thread i has bins 4i .. 4i + 3 (the last bin is the rest)
    u64 cnt[4], mass[4], nsum = 0, msum = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const u64 h = sHist[4 * tid + q];
      cnt[q] = h >> SM_COUNT;
      mass[q] = bin_mass(4 * tid + q, h);
      nsum += cnt[q];
      msum += mass[q];
    }
    u64 nrun = sm_wave_scan(nsum, lane), mrun = sm_wave_scan(msum, lane);
    if (lane == 63) {
      sWave[wave] = nrun;
      sWave2[wave] = mrun;
    }
    __syncthreads();
    u64 total = 0;
    nrun -= nsum;
    mrun -= msum;
    for (int w = 0; w < SM_WAVES; ++w) {
      if (w < wave) {
        nrun += sWave[w];
        mrun += sWave2[w];
      }
      total += sWave2[w];
    }
    kept = total;
    // The bin of a border: where the k-th token is (want), or the last one before which less than P
    // lies; the count and the mass above it. SM_BINS: none.
    auto find = [&](u64 want, double P, u64& n_above, u64& m_above) {
      __syncthreads();
      if (tid == 0) sPick[0] = want ? SM_BINS - 1 : SM_BINS, sPick[1] = sPick[2] = 0;
      __syncthreads();
      u64 n = nrun, s = mrun;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const bool rest = 4 * tid + q == SM_BINS - 1;
        const bool here = want ? n < want && (rest || want <= n + cnt[q])
                               : cnt[q] && (double)s < P && P <= (double)(s + mass[q]);
        if (here) {
          sPick[0] = (u64)(4 * tid + q);
          sPick[1] = n;
          sPick[2] = s;
        }
        n += cnt[q];
        s += mass[q];
      }
      __syncthreads();
      n_above = sPick[1];
      m_above = sPick[2];
      return (int)sPick[0];
    };
    bool digits = false, done = false;
    u64 n_k = 0, m_k = 0;
    const int bin_k = by_k ? find((u64)k, 0.0, n_k, m_k) : SM_BINS;
    if (by_k && by_p && bin_k < SM_BINS - 1) {
      // What top-k keeps has a mass between m_k and that with its bin's; the bins in which the border
      // of top-p can lie then, sorted with top-k's where they are few: one pass for both.
      u64 n_p, m_p;
      const int bin_p = find(0, (double)tp * (double)max(m_k, 1ULL), n_p, m_p);
      const u64 h = sHist[bin_k] >> SM_COUNT;
      if (bin_p <= bin_k && n_k + h - n_p <= SM_CAND && sort_bins(bin_p, bin_k)) {
        u64 in;
        border_in((u64)k - n_p, 0, 0.0, keep, in);
        kept = m_p + in;
        const double P = (double)tp * (double)kept;
        border_in(0, m_p, P, keep, in);
        kept = m_p + in;
        done = true;
      }
    }
#pragma unroll 1
    for (int step = 0; step < 2 && !done; ++step) {  // top-k, then top-p of what it keeps
      if (step == 0 ? !by_k : !by_p) continue;
      const u64 want = step == 0 ? (u64)k : 0;
      const double P = step == 0 ? 0.0 : (double)tp * (double)kept;
      u64 n_above = 0, above = 0;
      const int bin = digits ? SM_BINS : find(want, P, n_above, above);
      if (bin < SM_BINS && sort_bins(bin, bin)) {
        u64 in;
        border_in(want ? want - n_above : 0, above, P, keep, in);
        kept = above + in;
      } else {
        by_digits(want, P, keep, kept);
        digits = true;
      }
    }
  }

  // ---- the kept mass of each row of 64 pieces ----
  const u64 floor_w = mp > 0.f ? (u64)ceil((double)mp * SM_ONE) : 0;
  auto is_kept = [&](float l, int i) { return l > keep.at || (l == keep.at && i <= keep.last); };
  auto floored = [&](u64 w) { return w >= floor_w ? w : 0ULL; };
  __syncthreads();
  each([&](int c, int i0, const dkv_u32x4& v) {
    u64 s = 0;
    if (!by_k && !by_p) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float l = value(v, e);
        s += l > -INFINITY ? floored(weight(l)) : 0ULL;
      }
    } else {
      // the few that are kept, one of each lane's at a time
      uint32_t mask = 0;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float l = value(v, e);
        mask |= l >= keep.at && is_kept(l, i0 + e) ? 1u << e : 0u;
      }
      while (__ballot(mask != 0)) {
        const int e = mask ? __ffs((int)mask) - 1 : 0;
        float l = value(v, 0);
#pragma unroll
        for (int x = 1; x < E; ++x) l = e == x ? value(v, x) : l;
        const u64 w = floored(weight(l));
        s += mask ? w : 0ULL;
        mask &= mask - 1;
      }
    }
    s = sm_wave_sum(s);
    if (lane == 0) sChunk[wave * per_wave + c] = s;
  });
  __syncthreads();
  // ---- the row of pieces in which u * mass lies ----
  const int rows = SM_WAVES * per_wave;
  const int share = (rows + SM_THREADS - 1) / SM_THREADS;
  u64 own = 0;
  for (int i = tid * share; i < min(rows, (tid + 1) * share); ++i) own += sChunk[i];
  u64 run = sm_wave_scan(own, lane);
  if (lane == 63) sWave[wave] = run;
  __syncthreads();
  u64 all = 0;
  run -= own;
  for (int w = 0; w < SM_WAVES; ++w) {
    if (w < wave) run += sWave[w];
    all += sWave[w];
  }
  const float uu = p.u[row];
  const double U = uu > 0.f ? (double)uu * (double)all : 0.0;
  const u64 target = U < (double)all ? min((u64)U, all - 1) : all - 1;
  for (int i = tid * share; i < min(rows, (tid + 1) * share); ++i) {
    if (run <= target && target < run + sChunk[i]) {
      sPick[0] = (u64)i;
      sPick[1] = run;
    }
    run += sChunk[i];
  }
  __syncthreads();
  // ---- and the token ----
  const int hit = (int)sPick[0];
  if (hit / per_wave == wave) {
    const int c = hit % per_wave;
    const dkv_u32x4 v = load_again(c);
    const int i0 = first_of(c);
    u64 w[E], s = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float l = value(v, e);
      w[e] = is_kept(l, i0 + e) ? floored(weight(l)) : 0ULL;
      s += w[e];
    }
    u64 at = sPick[1] + sm_wave_scan(s, lane) - s;
    if (at <= target && target < at + s) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if (at <= target && target < at + w[e]) p.out[row] = (long long)(i0 + e);
        at += w[e];
      }
    }
  }
}

}  // namespace

extern "C" int dkv_sample_tokens(void* stream, int dtype, const void* logits, long long ld,
                                 int rows, int V, const float* u, const float* temperature,
                                 float temperature_all, const int* top_k, int top_k_all,
                                 const float* top_p, float top_p_all, const float* min_p,
                                 float min_p_all, long long* out) {
  if (dtype != DKV_F16 && dtype != DKV_BF16 && dtype != DKV_F32) return DKV_E_UNSUPPORTED;
  if (rows < 0 || V <= 0) return DKV_E_ARG;
  if (V > SM_MAX_V) return DKV_E_UNSUPPORTED;
  if (rows == 0) return DKV_OK;
  if (!logits || !u || !out || ld < 0 || (rows > 1 && ld < V)) return DKV_E_ARG;
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
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)rows), block(SM_THREADS);
  if (dtype == DKV_F32)
    hipLaunchKernelGGL(sample_kernel<DKV_F32>, grid, block, 0, st, p);
  else if (dtype == DKV_BF16)
    hipLaunchKernelGGL(sample_kernel<DKV_BF16>, grid, block, 0, st, p);
  else
    hipLaunchKernelGGL(sample_kernel<DKV_F16>, grid, block, 0, st, p);
  DKV_HIP_CHECK_LAUNCH();
  return DKV_OK;
}
