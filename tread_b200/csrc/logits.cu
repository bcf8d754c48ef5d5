// Adjusting the logits of the next token: penalties for repeated tokens, biases, a grammar's mask (sm_100a).
//
// Per row, with n[v] the count of token v in tokens[prompt_len : len] and seen[v] whether it is in
// tokens[0 : len]:
//   x = logits[v];   seen[v]: x = x > 0 ? x / repetition : x * repetition
//   x -= frequency * n[v] + presence * (n[v] > 0);   x += bias of v;   v not allowed: x = -inf
// in fp32, rounded once to the output's type. Ids outside [0, vocab) count for nothing (padding).
//
// A CTA owns a slice of a row's vocabulary. It counts the row's history into the slice's counters in shared
// memory (whole numbers: the order of the atomics does not matter), then passes over the slice once.
#include "common.cuh"

namespace tread {
namespace {

constexpr int kThreads = 256;
constexpr int kSlice = 8192;
constexpr unsigned kPrompt = 0x80000000u;  // set in a counter: the token is in the prompt

using LogitsArgs = tread_adjust_logits_args;

__device__ __forceinline__ void store(void* out, long long i, int dtype, float x) {
  if (dtype == TREAD_F32)
    static_cast<float*>(out)[i] = x;
  else if (dtype == TREAD_BF16)
    static_cast<__nv_bfloat16*>(out)[i] = __float2bfloat16_rn(x);
  else
    static_cast<__half*>(out)[i] = __float2half_rn(x);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) adjust_logits_kernel(const __grid_constant__ LogitsArgs a, int out_dtype) {
  extern __shared__ unsigned s_mem[];
  unsigned* count = s_mem;                                  // [kSlice]
  float* bias = reinterpret_cast<float*>(s_mem + kSlice);   // [kSlice], where biases are given
  const int b = blockIdx.y, v0 = blockIdx.x * kSlice;
  const int nv = a.V - v0 < kSlice ? a.V - v0 : kSlice;
  for (int i = threadIdx.x; i < nv; i += kThreads) count[i] = 0;
  if (a.num_bias)
    for (int i = threadIdx.x; i < nv; i += kThreads) bias[i] = 0.f;
  __syncthreads();
  if (a.tokens) {
    long long len = a.lens ? a.lens[b] : a.max_tokens;
    len = len < 0 ? 0 : len > a.max_tokens ? a.max_tokens : len;
    const long long prompt = a.prompt_lens ? a.prompt_lens[b] : 0;
    for (long long i = threadIdx.x; i < len; i += kThreads) {
      const long long v = a.tokens[b * a.tokens_ld + i] - v0;
      if (v >= 0 && v < nv) {
        if (i < prompt)
          atomicOr(count + v, kPrompt);
        else
          atomicAdd(count + v, 1u);
      }
    }
  }
  if (a.num_bias) {
    // the same token twice: its first entry adds up all of them, in their order
    const int64_t* ids = a.bias_ids + b * a.bias_ids_ld;
    for (int i = threadIdx.x; i < a.num_bias; i += kThreads) {
      const long long v = ids[i] - v0;
      if (v < 0 || v >= nv) continue;
      bool first = true;
      for (int j = 0; j < i; ++j) first &= ids[j] != ids[i];
      if (!first) continue;
      float sum = 0.f;
      for (int j = i; j < a.num_bias; ++j)
        if (ids[j] == ids[i]) sum += a.bias[b * a.bias_ld + j];
      bias[v] = sum;
    }
  }
  __syncthreads();
  const float rep = a.repetition ? a.repetition[b] : a.repetition_all;
  const float pres = a.presence ? a.presence[b] : a.presence_all;
  const float freq = a.frequency ? a.frequency[b] : a.frequency_all;
  for (int i = threadIdx.x; i < nv; i += kThreads) {
    float x = Num<T>::to_f(static_cast<const T*>(a.logits)[b * a.ld + v0 + i]);
    const unsigned c = count[i];
    if (c) {
      x = x > 0.f ? x / rep : x * rep;
      const unsigned n = c & ~kPrompt;
      if (n) x -= freq * (float)n + pres;
    }
    if (a.num_bias) x += bias[i];
    if (a.allowed && !((a.allowed[b * a.allowed_ld + ((v0 + i) >> 5)] >> ((v0 + i) & 31)) & 1)) x = -INFINITY;
    store(a.out, b * a.ld_out + v0 + i, out_dtype, x);
  }
}

template <typename T>
int launch(const LogitsArgs& a, int B, int out_dtype, cudaStream_t st) {
  const int smem = kSlice * (a.num_bias ? 8 : 4);
  auto kern = adjust_logits_kernel<T>;
  TREAD_CHECK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSlice * 8));
  kern<<<dim3((a.V + kSlice - 1) / kSlice, B), kThreads, smem, st>>>(a, out_dtype);
  TREAD_CHECK_LAUNCH("adjust_logits_kernel");
  return TREAD_OK;
}

}  // namespace
}  // namespace tread

extern "C" int tread_adjust_logits(const tread_adjust_logits_args* args, tread_stream_t stream) {
  using namespace tread;
  TREAD_CHECK_ARG(args, "adjust_logits: null arguments");
  LogitsArgs a = *args;
  TREAD_CHECK_ARG(a.B >= 0 && a.V >= 0, "adjust_logits: B < 0 or V < 0");
  if (a.B == 0 || a.V == 0) return TREAD_OK;
  TREAD_CHECK_ARG(a.logits && a.out, "adjust_logits: null pointer");
  TREAD_CHECK_ARG(a.B <= 65535, "adjust_logits: more than 65535 rows");
  TREAD_CHECK_ARG(dtype_size(a.dtype) != 0 && dtype_size(a.out_dtype) != 0, "adjust_logits: unknown dtype %d or %d",
                  a.dtype, a.out_dtype);
  TREAD_CHECK_ARG(a.B == 1 || (a.ld >= a.V && a.ld_out >= a.V), "adjust_logits: row stride below the vocabulary");
  TREAD_CHECK_ARG(a.max_tokens >= 0 && (!a.tokens || a.B == 1 || a.tokens_ld >= a.max_tokens),
                  "adjust_logits: bad history");
  TREAD_CHECK_ARG(a.num_bias >= 0 && (a.num_bias == 0 || (a.bias_ids && a.bias)), "adjust_logits: bad biases");
  TREAD_CHECK_ARG(a.repetition || a.repetition_all > 0.f, "adjust_logits: repetition must be above 0");
  if (!a.tokens) a.max_tokens = 0;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  switch (a.dtype) {
    case TREAD_BF16: return launch<__nv_bfloat16>(a, a.B, a.out_dtype, st);
    case TREAD_F16: return launch<__half>(a, a.B, a.out_dtype, st);
    default: return launch<float>(a, a.B, a.out_dtype, st);
  }
}
