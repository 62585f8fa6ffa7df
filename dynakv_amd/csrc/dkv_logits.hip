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
// A workgroup has `span` tokens of a row's vocabulary and counts in LDS (a word each: the generated ones
// below the bit that says it was seen) those of the history that fall into it; every workgroup of a row
// reads the whole history. Biases go by their entries: the first one of a token claims it (least entry
// by an atomic, whatever the order), sums the token's further ones in order and applies them, so that
// the same call gives the same bits.
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
};

constexpr int L_THREADS = 512;
constexpr int L_EACH = 4;            // tokens of a thread at a time
constexpr int L_SPAN = L_THREADS * L_EACH;  // least span
constexpr uint32_t L_SEEN = 0x80000000u;
constexpr uint32_t L_NONE = 0x7fffffffu;  // no entry
constexpr uint32_t L_MORE = 0x80000000u;  // further entries of the same token

template <int DT>
__global__ __launch_bounds__(L_THREADS) void adjust_kernel(LogitParams p) {
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
    for (int i = 4 * tid; i < p.span; i += 4 * L_THREADS)
      *(dkv_u32x4*)(entry + i) = dkv_u32x4{L_NONE, L_NONE, L_NONE, L_NONE};
  float rep = 1.f, freq = 0.f, pres = 0.f;
  int n = 0, prompt = 0;
  if (p.tokens) {
    rep = p.repetition ? p.repetition[row] : p.repetition_all;
    freq = p.frequency ? p.frequency[row] : p.frequency_all;
    pres = p.presence ? p.presence[row] : p.presence_all;
    n = min(p.len ? p.len[row] : p.len_all, p.N);
    prompt = p.prompt ? p.prompt[row] : p.prompt_all;
  }
  if (p.tokens || p.bias_ids) __syncthreads();
  // history
  if (p.wide) {
    const long long* t = (const long long*)p.tokens + (long long)row * p.tokens_ld;
#pragma unroll 4
    for (int j = tid; j < n; j += L_THREADS) {
      const unsigned long long i = (unsigned long long)(t[j] - v0);
      if (i < (unsigned long long)span) {
        if (j < prompt)
          atomicOr(count + i, L_SEEN);
        else
          atomicAdd(count + i, 1u);
      }
    }
  } else {
    const int* t = (const int*)p.tokens + (long long)row * p.tokens_ld;
#pragma unroll 4
    for (int j = tid; j < n; j += L_THREADS) {
      const uint32_t i = (uint32_t)t[j] - (uint32_t)v0;
      if (t[j] >= 0 && i < (uint32_t)span) {
        if (j < prompt)
          atomicOr(count + i, L_SEEN);
        else
          atomicAdd(count + i, 1u);
      }
    }
  }
  // biases
  const int* ids = nullptr;
  const float* bias = nullptr;
  if (p.bias_ids) {
    ids = p.bias_ids + (long long)row * p.bias_ids_ld;
    bias = p.bias + (long long)row * p.bias_ld;
    for (int j = tid; j < p.M; j += L_THREADS) {
      const uint32_t i = (uint32_t)ids[j] - (uint32_t)v0;
      if (ids[j] >= 0 && i < (uint32_t)span) atomicMin(entry + i, (uint32_t)j);
    }
    __syncthreads();
    for (int j = tid; j < p.M; j += L_THREADS) {
      const uint32_t i = (uint32_t)ids[j] - (uint32_t)v0;
      if (ids[j] >= 0 && i < (uint32_t)span && (entry[i] & ~L_MORE) != (uint32_t)j)
        atomicOr(entry + i, L_MORE);
    }
  }
  if (p.tokens || p.bias_ids) __syncthreads();

  // the tokens that anything concerns (the others at an offset that neither loads nor stores)
  const __amdgpu_buffer_rsrc_t r = dkv_make_rsrc(
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
      const int at = reads ? (i0 + u * L_THREADS) * SIZE : DKV_OOB;
      if constexpr (DT == DKV_F32)
        x[u] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(r, at, 0, 0));
      else
        x[u] = dkv_elt_to_f32<DT>(__builtin_amdgcn_raw_buffer_load_b16(r, at, 0, 0));
    }
#pragma unroll
    for (int u = 0; u < L_EACH; ++u) {
      float y = x[u];
      const uint32_t times = c[u] & ~L_SEEN;
      if (c[u]) {
        y = y > 0.f ? y / rep : y * rep;
        y = y - freq * (float)times - (times ? pres : 0.f);
      }
      if (e[u] != L_NONE) {
        const int j = (int)(e[u] & ~L_MORE), id = v0 + i0 + u * L_THREADS;
        float sum = bias[j];
        if (e[u] & L_MORE)
          for (int k = j + 1; k < p.M; ++k)
            if (ids[k] == id) sum += bias[k];
        y += sum;
      }
      if (off[u]) y = -INFINITY;
      const bool writes = c[u] || e[u] != L_NONE || off[u];
      const int at = writes ? (i0 + u * L_THREADS) * SIZE : DKV_OOB;
      if constexpr (DT == DKV_F32)
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(y), r, at, 0, 0);
      else if constexpr (DT == DKV_F16)
        __builtin_amdgcn_raw_buffer_store_b16((uint16_t)dkv_f32_to_f16_bits(y), r, at, 0, 0);
      else
        __builtin_amdgcn_raw_buffer_store_b16((uint16_t)dkv_f32_to_bf16_bits(y), r, at, 0, 0);
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
  if (!repetition && !(repetition_all > 0.f)) return DKV_E_ARG;
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
  const int words = (p.tokens ? 1 : 0) + (p.bias_ids ? 1 : 0);
  // spans of 2048 tokens to 64 KB of counts and entries (two workgroups a CU), as small as fills the chip
  int span = L_SPAN;
  const int most = words == 2 ? 8192 : 16384;
  while (span < most && (long long)rows * ((V + 2 * span - 1) / (2 * span)) >= 512) span *= 2;
  p.span = span;
  p.slices = (V + span - 1) / span;
  const long long wgs = ((long long)rows + 7) / 8 * 8 * p.slices;
  if (wgs > 0x7fffffffLL) return DKV_E_UNSUPPORTED;
  const size_t lds = (size_t)words * span * 4;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == DKV_F32)
    hipLaunchKernelGGL(adjust_kernel<DKV_F32>, dim3((unsigned)wgs), dim3(L_THREADS), lds, st, p);
  else if (dtype == DKV_F16)
    hipLaunchKernelGGL(adjust_kernel<DKV_F16>, dim3((unsigned)wgs), dim3(L_THREADS), lds, st, p);
  else
    hipLaunchKernelGGL(adjust_kernel<DKV_BF16>, dim3((unsigned)wgs), dim3(L_THREADS), lds, st, p);
  DKV_HIP_CHECK_LAUNCH();
  return DKV_OK;
}
