// What changes a row of logits before a token is drawn from it: penalties of tokens that the row's request
// has seen or generated, biases of some tokens, a mask of the allowed ones. In place.
#include "dkv_common.h"
#include "dkv_mfma_ops.h"

namespace {

// ---------------------------------------------------------------------------------------
// For token i of a row, with n_i its number among the generated tokens (tokens[prompt .. len - 1]) and
// b_i the sum of its biases in the order of their entries, in fp32 with one rounding at the end:
//   x = x > 0 ? x / r : x r   where i is among tokens[0 .. len - 1]
//   x = x - f n_i - (n_i > 0 ? p : 0)
//   x = x + b_i               where i has a bias
//   x = -inf                  where the mask's bit of i is 0
// A token that nothing of this concerns is neither read nor written: a row of 128256 logits with a history
// of a few thousand tokens is a few thousand reads and writes.
//
// A workgroup has a row and a table in LDS of the tokens that its history and its biases name: open
// addressing, at most three quarters full, a word for the token, one for its number (the generated ones
// below the bit that says it was seen) and one for the sum of its biases. What it holds at the end does not
// depend on the order of its atomics. One wave adds the biases, 64 entries at a time: of those of one token
// the first, then the second and so on, so that sums are in the entries' order and the same call gives the
// same bits (300 entries: 5 us a row, all on one token 67). A token's turn is a fourth word. The mask is for
// other workgroups of the launch, which clear the tokens that it forbids, and only those; the rows'
// workgroups look their tokens up in it.
//
// 256 rows of 128256 bf16 logits, histories of up to 4096 (400000 different tokens in all, a line of
// memory each) 17 us, where counting by vocabulary takes 59; with a mask that forbids half 31.5. Rows so
// few that they leave CUs idle are counted by vocabulary too: one row of 32000, a history of 1000, 4.4 us
// against 6.2.
//
// Histories that no table of 64 KB holds (over 6144 tokens, half of that with biases) are counted by
// vocabulary instead: a workgroup has `span` tokens of a row's vocabulary, a word each, and reads the whole
// history.
// ---------------------------------------------------------------------------------------
struct LogitParams {
  void* logits;
  long long ld;
  int rows, V;
  const void* tokens;  // null: no penalties
  long long tokens_ld;
  int wide;  // tokens of 64 bits
  int N;
  const int* prompt;
  const int* len;
  int prompt_all, len_all;
  const float* repetition;
  const float* frequency;
  const float* presence;
  float repetition_all, frequency_all, presence_all;
  const int* bias_ids;  // null: no biases
  long long bias_ids_ld;
  const float* bias;
  long long bias_ld;
  int M;
  const uint32_t* allowed;  // null: no mask
  long long allowed_ld;
  int span, slices;
  int slots_log2;  // of the table; by vocabulary: 0
  int row_wgs;     // leading workgroups, each with a row; then those of the mask
  int mask_wgs;    // of a row
};

constexpr int L_THREADS = 512;
constexpr int L_EACH = 4;            // tokens of a thread at a time
constexpr int L_SPAN = L_THREADS * L_EACH;  // least span
constexpr uint32_t L_SEEN = 0x80000000u;
constexpr uint32_t L_NONE = 0xffffffffu;  // no bias (a NaN that no sum is kept as)

constexpr int L_MASK = 8;            // tokens of a thread in a mask's workgroup

template <int DT>
__device__ __forceinline__ float load_logit(__amdgpu_buffer_rsrc_t r, int at) {
  if constexpr (DT == DKV_F32)
    return __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(r, at, 0, 0));
  else
    return dkv_elt_to_f32<DT>(__builtin_amdgcn_raw_buffer_load_b16(r, at, 0, 0));
}
template <int DT>
__device__ __forceinline__ void store_logit(__amdgpu_buffer_rsrc_t r, int at, float y) {
  if constexpr (DT == DKV_F32)
    __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(y), r, at, 0, 0);
  else if constexpr (DT == DKV_F16)
    __builtin_amdgcn_raw_buffer_store_b16((uint16_t)dkv_f32_to_f16_bits(y), r, at, 0, 0);
  else
    __builtin_amdgcn_raw_buffer_store_b16((uint16_t)dkv_f32_to_bf16_bits(y), r, at, 0, 0);
}

// A row's settings, and its biases.
struct LogitRow {
  float rep, freq, pres;
  int n, prompt;
  const int* ids;
  const float* bias;
};
__device__ __forceinline__ LogitRow logit_row(const LogitParams& p, int row) {
  LogitRow r = {1.f, 0.f, 0.f, 0, 0, nullptr, nullptr};
  if (p.tokens) {
    r.rep = p.repetition ? p.repetition[row] : p.repetition_all;
    r.freq = p.frequency ? p.frequency[row] : p.frequency_all;
    r.pres = p.presence ? p.presence[row] : p.presence_all;
    r.n = min(p.len ? p.len[row] : p.len_all, p.N);
    r.prompt = p.prompt ? p.prompt[row] : p.prompt_all;
  }
  if (p.bias_ids) {
    r.ids = p.bias_ids + (long long)row * p.bias_ids_ld;
    r.bias = p.bias + (long long)row * p.bias_ld;
  }
  return r;
}
// Entry j of the row's history, or -1 where it is no token of the vocabulary.
__device__ __forceinline__ int history(const LogitParams& p, int row, int j) {
  if (p.wide) {
    const long long t = ((const long long*)p.tokens)[(long long)row * p.tokens_ld + j];
    return t >= 0 && t < p.V ? (int)t : -1;
  }
  const int t = ((const int*)p.tokens)[(long long)row * p.tokens_ld + j];
  return t < p.V ? t : -1;
}
// What becomes of logit x of count c (0: not in the history) and biases' sum e (bits).
__device__ __forceinline__ float adjusted(const LogitRow& r, float x, uint32_t c, uint32_t e) {
  if (c) {
    const uint32_t times = c & ~L_SEEN;
    x = x > 0.f ? x / r.rep : x * r.rep;
    if (times) x = x - r.freq * (float)times - r.pres;
  }
  return e != L_NONE ? x + __uint_as_float(e) : x;
}
// The row's biases added to sums[slot(token)] (a slot below 0: none of this workgroup's), by one wave;
// `turn`: a word for each slot, L_NONE before and after.
template <class F>
__device__ __forceinline__ void add_biases(const LogitParams& p, const LogitRow& r, uint32_t* sums,
                                           uint32_t* turn, int lane, F&& slot) {
  int id = lane < p.M ? r.ids[lane] : -1;
  float b = lane < p.M ? r.bias[lane] : 0.f;
  for (int j = 0; j < p.M; j += 64) {
    const int s = id >= 0 && id < p.V ? slot(id) : -1;
    const float mine = b;
    if (j + 64 + lane < p.M) {
      id = r.ids[j + 64 + lane];
      b = r.bias[j + 64 + lane];
    } else {
      id = -1;
    }
    // of the lanes left that have a slot, the lowest is next
    for (bool left = s >= 0; __ballot(left);) {
      if (left) atomicMin(turn + s, (uint32_t)lane);
      __builtin_amdgcn_wave_barrier();
      if (left && *(volatile uint32_t*)(turn + s) == (uint32_t)lane) {
        volatile uint32_t* at = sums + s;
        const uint32_t was = *at;
        const float sum = was == L_NONE ? mine : __uint_as_float(was) + mine;
        *at = sum == sum ? __float_as_uint(sum) : 0x7fc00000u;
        *(volatile uint32_t*)(turn + s) = L_NONE;
        left = false;
      }
      __builtin_amdgcn_wave_barrier();
    }
  }
}

template <int DT>
__global__ __launch_bounds__(1024) void adjust_rows_kernel(LogitParams p) {
  extern __shared__ __attribute__((aligned(16))) uint32_t lds[];
  constexpr int SIZE = DT == DKV_F32 ? 4 : 2;
  const int tid = threadIdx.x, T = blockDim.x;
  if ((int)blockIdx.x >= p.row_wgs) {  // the mask of some tokens of a row
    const int x = blockIdx.x - p.row_wgs, row = x / p.mask_wgs;
    const int v0 = (x - row * p.mask_wgs) * (T * L_MASK), span = min(T * L_MASK, p.V - v0);
    const __amdgpu_buffer_rsrc_t r = dkv_make_rsrc(
        (uint8_t*)p.logits + ((long long)row * p.ld + v0) * SIZE, (uint32_t)span * SIZE);
    const uint32_t* words = p.allowed + (long long)row * p.allowed_ld + v0 / 32;
    uint32_t w[L_MASK];
#pragma unroll
    for (int u = 0; u < L_MASK; ++u) {
      const int i = tid + u * T;
      w[u] = i < span ? words[i >> 5] : 0xffffffffu;
    }
#pragma unroll
    for (int u = 0; u < L_MASK; ++u) {
      const int i = tid + u * T;
      store_logit<DT>(r, (w[u] >> (i & 31)) & 1u ? DKV_OOB : i * SIZE, -INFINITY);
    }
    return;
  }
  const int row = blockIdx.x, slots = 1 << p.slots_log2;
  uint32_t *key = lds, *count = lds + slots, *entry = lds + 2 * slots;
  for (int i = 4 * tid; i < 2 * slots; i += 4 * T)  // (key: the token + 1, 0 where none is)
    *(dkv_u32x4*)(lds + i) = dkv_u32x4{0u, 0u, 0u, 0u};
  if (p.bias_ids)
    for (int i = 4 * tid; i < 2 * slots; i += 4 * T)  // (and the turns behind them)
      *(dkv_u32x4*)(entry + i) = dkv_u32x4{L_NONE, L_NONE, L_NONE, L_NONE};
  // the first of the history, whose number is not known yet, beside the settings
  int first[L_EACH];
  if (p.tokens)
#pragma unroll
    for (int u = 0; u < L_EACH; ++u) {
      const int j = tid + u * T;
      first[u] = j < p.N ? history(p, row, j) : -1;
    }
  const LogitRow r = logit_row(p, row);
  __syncthreads();
  auto place = [&](int id) {  // the token's slot (there is a free one: fewer tokens than slots)
    uint32_t i = (uint32_t)id * 2654435769u >> (32 - p.slots_log2);
    for (;;) {
      uint32_t k = *(volatile uint32_t*)(key + i);
      if (k == 0) k = atomicCAS(key + i, 0u, (uint32_t)id + 1u);
      if (k == 0 || k == (uint32_t)id + 1u) return i;
      i = (i + 1) & (uint32_t)(slots - 1);
    }
  };
  if (p.bias_ids && tid < 64)
    add_biases(p, r, entry, entry + slots, tid, [&](int id) { return (int)place(id); });
  for (int j0 = tid; j0 < r.n; j0 += L_EACH * T) {
    int id[L_EACH];
#pragma unroll
    for (int u = 0; u < L_EACH; ++u) {
      const int j = j0 + u * T;
      id[u] = j >= r.n ? -1 : j0 == tid ? first[u] : history(p, row, j);
    }
#pragma unroll
    for (int u = 0; u < L_EACH; ++u) {
      if (id[u] < 0) continue;
      const uint32_t i = place(id[u]);
      if (j0 + u * T < r.prompt)
        atomicOr(count + i, L_SEEN);
      else
        atomicAdd(count + i, 1u);
    }
  }
  __syncthreads();
  const __amdgpu_buffer_rsrc_t logits =
      dkv_make_rsrc((uint8_t*)p.logits + (long long)row * p.ld * SIZE, (uint32_t)p.V * SIZE);
  for (int i0 = tid; i0 < slots; i0 += L_EACH * T) {
    int id[L_EACH];
    float x[L_EACH];
    uint32_t word[L_EACH], e[L_EACH];
#pragma unroll
    for (int u = 0; u < L_EACH; ++u) {
      const int i = i0 + u * T;
      id[u] = i < slots ? (int)key[i] - 1 : -1;
      e[u] = p.bias_ids && id[u] >= 0 ? entry[i] : L_NONE;
      x[u] = load_logit<DT>(logits, id[u] >= 0 ? id[u] * SIZE : DKV_OOB);
      word[u] = 0xffffffffu;
      if (p.allowed && id[u] >= 0)
        word[u] = p.allowed[(long long)row * p.allowed_ld + (id[u] >> 5)];
    }
#pragma unroll
    for (int u = 0; u < L_EACH; ++u) {
      if (id[u] < 0) continue;
      const int i = i0 + u * T;
      float y = adjusted(r, x[u], count[i], e[u]);
      if (!((word[u] >> (id[u] & 31)) & 1u)) y = -INFINITY;
      store_logit<DT>(logits, id[u] * SIZE, y);
    }
  }
}

template <int DT>
__global__ __launch_bounds__(L_THREADS) void adjust_vocabulary_kernel(LogitParams p) {
  extern __shared__ __attribute__((aligned(16))) uint32_t lds[];
  constexpr int SIZE = DT == DKV_F32 ? 4 : 2;
  const int tid = threadIdx.x;
  // the workgroups of a row on one XCD (they go to the eight in turn), whose L2 then has its history
  const int eight = 8 * p.slices, group = blockIdx.x / eight, in = blockIdx.x - group * eight;
  const int row = group * 8 + (in & 7), v0 = (in >> 3) * p.span;
  if (row >= p.rows) return;
  const int span = min(p.span, p.V - v0);
  uint32_t* count = lds;
  uint32_t* entry = lds + (p.tokens ? p.span : 0);
  if (p.tokens)
    for (int i = 4 * tid; i < p.span; i += 4 * L_THREADS) *(dkv_u32x4*)(count + i) = dkv_u32x4{0u, 0u, 0u, 0u};
  if (p.bias_ids)
    for (int i = 4 * tid; i < 2 * p.span; i += 4 * L_THREADS)  // (and the turns behind them)
      *(dkv_u32x4*)(entry + i) = dkv_u32x4{L_NONE, L_NONE, L_NONE, L_NONE};
  int first[L_EACH];  // (as in the kernel by rows)
  if (p.tokens)
#pragma unroll
    for (int u = 0; u < L_EACH; ++u) {
      const int j = tid + u * L_THREADS;
      first[u] = j < p.N ? history(p, row, j) : -1;
    }
  const LogitRow r = logit_row(p, row);
  if (p.tokens || p.bias_ids) __syncthreads();
  for (int j0 = tid; j0 < r.n; j0 += L_EACH * L_THREADS) {
    int at[L_EACH];
#pragma unroll
    for (int u = 0; u < L_EACH; ++u) {
      const int j = j0 + u * L_THREADS;
      at[u] = (j >= r.n ? -1 : j0 == tid ? first[u] : history(p, row, j)) - v0;
    }
#pragma unroll
    for (int u = 0; u < L_EACH; ++u) {
      if (at[u] < 0 || at[u] >= span) continue;
      if (j0 + u * L_THREADS < r.prompt)
        atomicOr(count + at[u], L_SEEN);
      else
        atomicAdd(count + at[u], 1u);
    }
  }
  if (p.bias_ids && tid < 64)
    add_biases(p, r, entry, entry + p.span, tid,
               [&](int id) { return id >= v0 && id - v0 < span ? id - v0 : -1; });
  if (p.tokens || p.bias_ids) __syncthreads();

  // the tokens that anything concerns (the others at an offset that neither loads nor stores)
  const __amdgpu_buffer_rsrc_t logits = dkv_make_rsrc(
      (uint8_t*)p.logits + ((long long)row * p.ld + v0) * SIZE, (uint32_t)span * SIZE);
  const uint32_t* words = p.allowed ? p.allowed + (long long)row * p.allowed_ld + v0 / 32 : nullptr;
  for (int i0 = tid; i0 < span; i0 += L_THREADS * L_EACH) {
    uint32_t c[L_EACH], e[L_EACH];
    bool off[L_EACH], does = false;
#pragma unroll
    for (int u = 0; u < L_EACH; ++u) {
      const int i = i0 + u * L_THREADS;
      c[u] = 0;
      e[u] = L_NONE;
      off[u] = false;
      if (i < span) {
        if (p.tokens) c[u] = count[i];
        if (p.bias_ids) e[u] = entry[i];
        if (words) off[u] = !((words[i >> 5] >> (i & 31)) & 1u);
      }
      does = does || c[u] || e[u] != L_NONE || off[u];
    }
    if (!__ballot(does)) continue;
    float x[L_EACH];
#pragma unroll
    for (int u = 0; u < L_EACH; ++u) {
      const bool reads = (c[u] || e[u] != L_NONE) && !off[u];
      x[u] = load_logit<DT>(logits, reads ? (i0 + u * L_THREADS) * SIZE : DKV_OOB);
    }
#pragma unroll
    for (int u = 0; u < L_EACH; ++u) {
      const int i = i0 + u * L_THREADS;
      const float y = off[u] ? -INFINITY : adjusted(r, x[u], c[u], e[u]);
      const bool writes = c[u] || e[u] != L_NONE || off[u];
      store_logit<DT>(logits, writes ? i * SIZE : DKV_OOB, y);
    }
  }
}

}  // namespace

extern "C" int dkv_adjust_logits(void* stream, int dtype, void* logits, long long ld, int rows, int V,
                                 const void* tokens, int token_bytes, long long tokens_ld, int N,
                                 const int* prompt_lens, int prompt_all, const int* lens, int len_all,
                                 const float* repetition, float repetition_all,
                                 const float* frequency, float frequency_all, const float* presence,
                                 float presence_all, const int* bias_ids, long long bias_ids_ld,
                                 const float* bias, long long bias_ld, int M, const int* allowed,
                                 long long allowed_ld) {
  const int size = dkv_elt_size(dtype);
  if (size == 0) return DKV_E_UNSUPPORTED;
  if (rows < 0 || V < 0 || N < 0 || M < 0) return DKV_E_ARG;
  if (rows == 0 || V == 0) return DKV_OK;
  if (V > (1 << 28)) return DKV_E_UNSUPPORTED;
  if (!logits || (rows > 1 && ld < V)) return DKV_E_ARG;
  if ((uintptr_t)logits % size) return DKV_E_UNSUPPORTED;
  if (token_bytes != 4 && token_bytes != 8) return DKV_E_ARG;
  if (tokens_ld < 0 || bias_ids_ld < 0 || bias_ld < 0 || allowed_ld < 0) return DKV_E_ARG;
  if ((M > 0 && !bias_ids != !bias)) return DKV_E_ARG;
  if (!repetition && !(repetition_all > 0.f && repetition_all < INFINITY)) return DKV_E_ARG;
  LogitParams p;
  p.logits = logits;
  p.ld = ld;
  p.rows = rows;
  p.V = V;
  p.tokens = N > 0 ? tokens : nullptr;
  p.tokens_ld = tokens_ld;
  p.wide = token_bytes == 8;
  p.N = N;
  p.prompt = prompt_lens;
  p.prompt_all = prompt_all;
  p.len = lens;
  p.len_all = len_all;
  p.repetition = repetition;
  p.repetition_all = repetition_all;
  p.frequency = frequency;
  p.frequency_all = frequency_all;
  p.presence = presence;
  p.presence_all = presence_all;
  p.bias_ids = M > 0 ? bias_ids : nullptr;
  p.bias_ids_ld = bias_ids_ld;
  p.bias = bias;
  p.bias_ld = bias_ld;
  p.M = M;
  p.allowed = (const uint32_t*)allowed;
  p.allowed_ld = allowed_ld;
  if (!p.tokens && !p.bias_ids && !p.allowed) return DKV_OK;
  hipStream_t st = (hipStream_t)stream;
  const int words = (p.tokens ? 1 : 0) + (p.bias_ids ? 2 : 0);
  auto launch = [&](auto f32, auto f16, auto bf16, long long wgs, int threads, size_t lds) {
    const dim3 grid((unsigned)wgs);
    if (dtype == DKV_F32)
      hipLaunchKernelGGL(f32, grid, dim3(threads), lds, st, p);
    else if (dtype == DKV_F16)
      hipLaunchKernelGGL(f16, grid, dim3(threads), lds, st, p);
    else
      hipLaunchKernelGGL(bf16, grid, dim3(threads), lds, st, p);
  };
  const long long named = (p.tokens ? (long long)N : 0) + M;
  int log2 = 9;
  while (log2 < 30 && 3LL << log2 < 4 * named) ++log2;
  const size_t table = ((size_t)4 << log2) * (p.bias_ids ? 4 : 2);
  const bool few = words && (long long)rows * ((V + L_SPAN - 1) / L_SPAN) <= 256;
  if (table <= 65536 && !few) {
    const int threads = named > 1024 ? 1024 : L_THREADS;
    p.slots_log2 = log2;
    p.row_wgs = words ? rows : 0;
    p.mask_wgs = (V + threads * L_MASK - 1) / (threads * L_MASK);
    const long long wgs = p.row_wgs + (p.allowed ? (long long)rows * p.mask_wgs : 0);
    if (wgs > 0x7fffffffLL) return DKV_E_UNSUPPORTED;
    launch(adjust_rows_kernel<DKV_F32>, adjust_rows_kernel<DKV_F16>, adjust_rows_kernel<DKV_BF16>, wgs,
           threads, words ? table : 0);
  } else {
    // spans of 2048 tokens to 64 KB of counts and entries (two workgroups a CU), as small as fills the chip
    int span = L_SPAN;
    const int most = words == 3 ? 4096 : words == 2 ? 8192 : 16384;
    while (span < most && (long long)rows * ((V + 2 * span - 1) / (2 * span)) >= 512) span *= 2;
    p.span = span;
    p.slices = (V + span - 1) / span;
    const long long wgs = ((long long)rows + 7) / 8 * 8 * p.slices;
    if (wgs > 0x7fffffffLL) return DKV_E_UNSUPPORTED;
    launch(adjust_vocabulary_kernel<DKV_F32>, adjust_vocabulary_kernel<DKV_F16>,
           adjust_vocabulary_kernel<DKV_BF16>, wgs, L_THREADS, (size_t)words * span * 4);
  }
  DKV_HIP_CHECK_LAUNCH();
  return DKV_OK;
}
