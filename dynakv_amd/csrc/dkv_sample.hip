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
// Weights are held in 64-bit fixed point, 44 bits after the point, computed in 64-bit floating
// point: sums of them are the same in any order (the histograms add by atomics), and a token is
// decided by u * mass against a running sum, where 32 bits would pick another token than the
// formula's in one draw of a few thousand.
#include "dkv_common.h"

namespace {

typedef unsigned long long u64;

constexpr int SM_THREADS = 1024;
constexpr int SM_WAVES = SM_THREADS / 64;
constexpr int SM_POINT = 44;             // bits after the point of a weight
constexpr int SM_MAX_V = 1 << 19;        // weights of at most 1: sums below 2^63
constexpr int SM_BINS = 2048;

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

// A logit as a number that orders as the logits do: NaN as -infinity, -0 as +0.
__device__ __forceinline__ float sm_clean(float f) {
  return f != f ? -INFINITY : f + 0.0f;
}
__device__ __forceinline__ uint32_t sm_key(float f) {
  const uint32_t b = __float_as_uint(f);
  return b ^ ((int)b < 0 ? 0xffffffffu : 0x80000000u);
}

__device__ __forceinline__ u64 sm_weight(float l, float m, double c) {
  if (l == m) return 1ULL << SM_POINT;
  const double y = ((double)l - (double)m) * c;  // c = log2(e) / t
  if (!(y > -(double)(SM_POINT + 2))) return 0;
  const double n = rint(y), g = (y - n) * 0.69314718055994530942;
  double s = 1.0 / 479001600.0;  // sum of g^k / k!, k <= 12: |g| <= ln 2 / 2, 2e-16 left out
  s = fma(s, g, 1.0 / 39916800.0);
  s = fma(s, g, 1.0 / 3628800.0);
  s = fma(s, g, 1.0 / 362880.0);
  s = fma(s, g, 1.0 / 40320.0);
  s = fma(s, g, 1.0 / 5040.0);
  s = fma(s, g, 1.0 / 720.0);
  s = fma(s, g, 1.0 / 120.0);
  s = fma(s, g, 1.0 / 24.0);
  s = fma(s, g, 1.0 / 6.0);
  s = fma(s, g, 0.5);
  s = fma(s, g, 1.0);
  s = fma(s, g, 1.0);
  return (u64)llrint(ldexp(s, (int)n + SM_POINT));
}

__device__ __forceinline__ u64 sm_wave_sum(u64 v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
__device__ __forceinline__ u64 sm_wave_scan(u64 v, int lane) {  // inclusive
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const u64 x = __shfl_up(v, o, 64);
    if (lane >= o) v += x;
  }
  return v;
}

// What is kept: every token above `key`, and the first `ties` of those at it.
struct Border {
  uint32_t key;
  int ties;
};

template <int DT>
__global__ __launch_bounds__(SM_THREADS) void sample_kernel(SampleParams p) {
  __shared__ u64 sMass[SM_BINS];
  __shared__ uint32_t sCount[SM_BINS];
  __shared__ u64 sWave[SM_WAVES];
  __shared__ uint32_t sWaveN[SM_WAVES];
  __shared__ u64 sPick[4];
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const char* base = (const char*)p.logits + (long long)row * p.ld * (DT == DKV_F32 ? 4 : 2);
  auto logit = [&](int i) { return sm_clean(dkv_load_f32<DT>(base, i)); };
  const float t = p.temperature ? p.temperature[row] : p.temperature_all;
  const int k = p.top_k ? p.top_k[row] : p.top_k_all;
  const float tp = p.top_p ? p.top_p[row] : p.top_p_all;
  const float mp = p.min_p ? p.min_p[row] : p.min_p_all;
  const int V = p.V;

  // the largest logit and the first index of it
  u64 best = 0;
  for (int i = tid; i < V; i += SM_THREADS)
    best = max(best, ((u64)sm_key(logit(i)) << 32) | (uint32_t)~i);
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) best = max(best, __shfl_xor(best, o, 64));
  if (lane == 0) sWave[wave] = best;
  __syncthreads();
  for (int w = 0; w < SM_WAVES; ++w) best = max(best, sWave[w]);
  __syncthreads();
  const int arg = (int)~(uint32_t)best;
  const float m = logit(arg);
  if (m == -INFINITY) {
    if (tid == 0) p.out[row] = -1;
    return;
  }
  if (!(t > 0.f) || k == 1 || tp <= 0.f || mp > 1.f) {  // the first token alone
    if (tid == 0) p.out[row] = arg;
    return;
  }
  const double c = 1.4426950408889634074 / (double)t;

  // The border by digits of the keys (11, 11, 10 bits): a histogram of the tokens that share the
  // digits found so far, counts and masses, and the bin in which the k-th token (by_mass: the
  // first token before which the mass reaches P) lies. Every thread gets the same answer.
  auto find = [&](bool by_mass, u64 want, double P, u64& mass_above) {
    Border r = {0, 0};
    u64 above = 0;  // mass or count above the bins of this level
    u64 m_above = 0;
    uint32_t found = 0;
    for (int level = 0; level < 3; ++level) {
      const int shift = level == 0 ? 21 : level == 1 ? 10 : 0;
      const int bits = level == 2 ? 10 : 11;
      for (int i = tid; i < SM_BINS; i += SM_THREADS) sMass[i] = 0, sCount[i] = 0;
      __syncthreads();
      for (int i = tid; i < V; i += SM_THREADS) {
        const float l = logit(i);
        const uint32_t key = sm_key(l);
        if (level && (key >> (shift + bits)) != found) continue;
        const int bin = (int)((key >> shift) & ((1u << bits) - 1));
        atomicAdd(&sCount[bin], 1u);
        atomicAdd(&sMass[bin], sm_weight(l, m, c));
      }
      __syncthreads();
      // thread 0 walks the bins from the top
      if (tid == 0) {
        u64 cum = above, mass = m_above;
        int at = -1;
        u64 cum_at = 0, mass_at = 0;
        for (int bin = (1 << bits) - 1; bin >= 0; --bin) {
          if (!sCount[bin]) continue;
          if (by_mass ? (double)cum < P : cum < want) {
            at = bin;
            cum_at = cum;
            mass_at = mass;
          } else {
            break;
          }
          cum += by_mass ? sMass[bin] : sCount[bin];
          mass += sMass[bin];
        }
        sPick[0] = (u64)(uint32_t)at;
        sPick[1] = cum_at;
        sPick[2] = mass_at;
        sPick[3] = at >= 0 ? sCount[at] : 0;
      }
      __syncthreads();
      found = (found << bits) | (uint32_t)sPick[0];
      above = sPick[1];
      m_above = sPick[2];
      r.ties = (int)sPick[3];
      __syncthreads();
    }
    r.key = found;
    const uint32_t b = found ^ ((int)found < 0 ? 0x80000000u : 0xffffffffu);
    const u64 w = sm_weight(__uint_as_float(b), m, c);
    if (!by_mass) {
      r.ties = (int)min((u64)r.ties, want - above);
    } else if (w > 0) {
      // the ties before which less than P lies
      int lo = 1, hi = r.ties;
      while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if ((double)(above + (u64)(mid - 1) * w) < P)
          lo = mid;
        else
          hi = mid - 1;
      }
      r.ties = lo;
    }
    mass_above = m_above + (u64)r.ties * w;  // the mass kept
    return r;
  };

  Border keep = {0, 0x7fffffff};
  u64 kept = 0;
  const bool by_k = k > 0 && k < V, by_p = tp < 1.f;
  if (by_k) keep = find(false, (u64)k, 0.0, kept);
  if (by_p) {
    if (!by_k) {
      u64 s = 0;
      for (int i = tid; i < V; i += SM_THREADS) s += sm_weight(logit(i), m, c);
      s = sm_wave_sum(s);
      if (lane == 0) sWave[wave] = s;
      __syncthreads();
      for (int w = 0; w < SM_WAVES; ++w) kept += sWave[w];
      __syncthreads();
    }
    const double P = (double)tp * (double)kept;
    keep = find(true, 0, P, kept);
  }
  const double floor_w = mp > 0.f ? (double)mp * (double)(1ULL << SM_POINT) : 0.0;

  // The kept mass in the vocabulary's order: wave w takes the w-th part of the row.
  const int part = (V + SM_WAVES - 1) / SM_WAVES;
  const int i0 = min(V, wave * part), i1 = min(V, i0 + part);
  // ties up to the part
  uint32_t nt = 0;
  for (int i = i0 + lane; i < i1; i += 64) nt += sm_key(logit(i)) == keep.key;
  nt = (uint32_t)sm_wave_sum(nt);
  if (lane == 0) sWaveN[wave] = nt;
  __syncthreads();
  uint32_t ties0 = 0;
  for (int w = 0; w < wave; ++w) ties0 += sWaveN[w];
  auto part_mass = [&](u64 target, bool pick, u64 before) {
    u64 sum = before;
    uint32_t ties = ties0;
    for (int j = i0; j < i1; j += 64) {
      const int i = j + lane;
      const float l = i < i1 ? logit(i) : -INFINITY;
      const uint32_t key = i < i1 ? sm_key(l) : 0u;
      const u64 same = __ballot(i < i1 && key == keep.key);
      const uint32_t rank = ties + (uint32_t)__popcll(same & ((1ULL << lane) - 1));
      ties += (uint32_t)__popcll(same);
      u64 w = 0;
      if (i < i1 && (key > keep.key || (key == keep.key && rank < (uint32_t)keep.ties))) {
        w = sm_weight(l, m, c);
        if ((double)w < floor_w) w = 0;
      }
      const u64 run = sm_wave_scan(w, lane);
      if (pick) {
        const u64 hit = __ballot(sum + run > target);
        if (hit) return (u64)(j + __ffsll((long long)hit) - 1);
      }
      sum += __shfl(run, 63, 64);
    }
    return pick ? (u64)-1 : sum;
  };
  const u64 mine = part_mass(0, false, 0);
  if (lane == 0) sWave[wave] = mine;
  __syncthreads();
  u64 all = 0, before = 0;
  for (int w = 0; w < SM_WAVES; ++w) {
    if (w < wave) before += sWave[w];
    all += sWave[w];
  }
  const float uu = p.u[row];
  const double U = uu > 0.f ? (double)uu * (double)all : 0.0;
  const u64 target = U < (double)all ? min((u64)U, all - 1) : all - 1;
  if (before <= target && target < before + mine) {
    const u64 i = part_mass(target, true, before);
    if (lane == 0) p.out[row] = (long long)i;
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
