// Adjusting the logits of the next token: penalties for repeated tokens, biases, a grammar's mask (sm_100a).
//
// Per row, with n[v] the count of token v in tokens[prompt_len : len] and seen[v] whether it is in
// tokens[0 : len]:
//   x = logits[v];   seen[v]: x = x > 0 ? x / repetition : x * repetition
//   x -= frequency * n[v] + presence * (n[v] > 0);   x += bias of v;   v not allowed: x = -inf
// in fp32, rounded once to the output's type. Ids outside [0, vocab) count for nothing (padding).
//
// Bound by reading the logits and writing the result. A CTA owns a slice of a row's vocabulary and issues its
// first loads. While they fly it counts the row's whole history into counters of the slice in shared memory
// (whole numbers: the order of the atomics does not matter), and computes the slice's few biased tokens, each by
// the thread that marked it first. Then one pass reads, penalises, masks and stores every logit, and the biased
// ones are stored again. At 64 rows of 152064 with histories of up to 8768, a mask and 100 biases that takes
// 19.2 us (3.2 TB/s; a casting copy of the same tensors takes 28), the pass alone 13.5. Nearly every warp has one of
// the history's tokens among its 256, so the penalties are selects over a thread's vector rather than branches
// (22.5 us). Finishing those tokens by themselves cost more, in scattered reads and writes of lines that have left
// the caches: 26 us with their values found before the pass, 29 in place after it.
// Reading the history again for every slice costs L2 reads only, and no counters in memory that a caller would
// have to keep or clear.
#include "common.cuh"

namespace tread {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxSlice = 18432;
constexpr int kCtas = 4;         // CTAs of an SM
constexpr int kVec = 8;          // consecutive logits of a thread
constexpr int kAhead = 8;        // ids of the history that a thread has in flight
constexpr int kMaxBias = 2048;   // biases of a row: their values' room in shared memory

using LogitsArgs = tread_adjust_logits_args;

// A token's counter in 16 or 32 bits: how often the output holds it, and two marks.
template <typename W>
struct Counter {
  static constexpr int kBits = sizeof(W) * 8;
  static constexpr unsigned kPrompt = 1u << (kBits - 1);  // the prompt holds it
  static constexpr unsigned kBiased = 1u << (kBits - 2);
  static constexpr unsigned kCount = kBiased - 1;
  // marks or counts token i of the slice; returns its counter as it was
  static __device__ __forceinline__ unsigned mark(W* c, int i, unsigned what) {
    if constexpr (sizeof(W) == 4) return atomicOr(reinterpret_cast<unsigned*>(c) + i, what);
    const int shift = (i & 1) * 16;
    return atomicOr(reinterpret_cast<unsigned*>(c) + (i >> 1), what << shift) >> shift;
  }
  static __device__ __forceinline__ void add(W* c, int i) {
    if constexpr (sizeof(W) == 4)
      atomicAdd(reinterpret_cast<unsigned*>(c) + i, 1u);
    else
      atomicAdd(reinterpret_cast<unsigned*>(c) + (i >> 1), 1u << ((i & 1) * 16));
  }
};

__device__ __forceinline__ void store(void* out, long long i, int dtype, float x) {
  if (dtype == TREAD_F32)
    static_cast<float*>(out)[i] = x;
  else if (dtype == TREAD_BF16)
    static_cast<__nv_bfloat16*>(out)[i] = __float2bfloat16_rn(x);
  else
    static_cast<__half*>(out)[i] = __float2half_rn(x);
}

template <typename T>
__device__ __forceinline__ void store8(void* out, long long i, const float (&x)[kVec]) {
  T* to = static_cast<T*>(out) + i;
  constexpr int E = 16 / sizeof(T);
#pragma unroll
  for (int k = 0; k < kVec; k += E) {
    Vec16<T> v;
#pragma unroll
    for (int e = 0; e < E; ++e) v.e[e] = Num<T>::from_f(x[k + e]);
    st_stream(to + k, v.raw);
  }
}

// VECS: vectors of kVec logits that a thread has in flight
template <typename T, typename W, int VECS>
__global__ void __launch_bounds__(kThreads, kCtas)
    adjust_logits_kernel(const __grid_constant__ LogitsArgs a, int slice) {
  using C = Counter<W>;
  extern __shared__ __align__(16) unsigned char s_mem[];
  __shared__ int s_twice;   // some token of the slice has more than one bias
  __shared__ float s_value[kMaxBias];
  W* count = reinterpret_cast<W*>(s_mem);  // of tokens first - kVec .. first + slice - 1
  const int b = blockIdx.y;
  const T* row = static_cast<const T*>(a.logits) + b * a.ld;
  const long long out_row = b * a.ld_out;
  // vectors start where the row's address is a multiple of 16 bytes: the first slice has the tokens before
  const int head = (int)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / (int)sizeof(T);
  const int first = head + blockIdx.x * slice;  // token of the slice's first vector
  const int begin = blockIdx.x == 0 ? 0 : first;
  const int end = min(a.V, first + slice);
  if (begin >= end) return;
  const int vecs = end > first ? (end - first) / kVec : 0;  // whole ones; the rest of the row token by token
  const int origin = first - kVec;
  const int tid = threadIdx.x;
  const unsigned* allowed = a.allowed ? reinterpret_cast<const unsigned*>(a.allowed) + b * a.allowed_ld : nullptr;
  auto is_allowed = [&](int v) { return !allowed || (allowed[v >> 5] >> (v & 31)) & 1; };
  constexpr int L = kVec * sizeof(T) / 16;  // 16-byte loads of a vector
  int4 x[VECS][L];
  auto load = [&](int i0) {
#pragma unroll
    for (int k = 0; k < VECS; ++k) {
      const int i = i0 + k * kThreads;
      if (i < vecs) {
#pragma unroll
        for (int j = 0; j < L; ++j) x[k][j] = ld_stream(row + first + i * kVec + j * (16 / sizeof(T)));
      }
    }
  };
  load(tid);
  const bool changes = a.tokens || a.num_bias;
  const float rep = a.repetition ? a.repetition[b] : a.repetition_all;
  const float pres = a.presence ? a.presence[b] : a.presence_all;
  const float freq = a.frequency ? a.frequency[b] : a.frequency_all;
  // x / repetition as a product with its reciprocal: a rounding more, a division's dozen instructions fewer;
  // but for reciprocals that overflow or lose digits
  const float inv = 1.f / rep;
  const bool product = rep > 0x1p-100f && rep < 0x1p100f;
  auto repeated = [&](float f) { return f > 0.f ? (product ? f * inv : f / rep) : f * rep; };
  auto counted = [&](float f, unsigned c) { return f - (freq * (float)(c & C::kCount) + pres); };
  auto penalised = [&](float f, unsigned c) {
    if (c) f = repeated(f);
    return c & C::kCount ? counted(f, c) : f;
  };
  unsigned mine = 0;  // biases whose token this thread marked first
  const int64_t* bias_ids = a.bias_ids + b * a.bias_ids_ld;
  const float* bias = a.bias + b * a.bias_ld;
  if (changes) {
    for (int i = tid; i < (int)((slice + kVec) * sizeof(W) / 16); i += kThreads)
      reinterpret_cast<int4*>(s_mem)[i] = make_int4(0, 0, 0, 0);
    if (tid == 0) s_twice = 0;
    __syncthreads();
    for (int i = tid, k = 0; i < a.num_bias; i += kThreads, ++k) {
      const long long v = bias_ids[i];
      if (v < begin || v >= end) continue;
      if (C::mark(count, (int)v - origin, C::kBiased) & C::kBiased)
        s_twice = 1;
      else
        mine |= 1u << k;
    }
    if (a.tokens) {
      long long len = a.lens ? a.lens[b] : a.max_tokens;
      len = len < 0 ? 0 : len > a.max_tokens ? a.max_tokens : len;
      const long long prompt = a.prompt_lens ? a.prompt_lens[b] : 0;
      const long long* ids = reinterpret_cast<const long long*>(a.tokens) + b * a.tokens_ld;
      const unsigned room = end - begin;
      for (int i0 = tid; i0 < (int)len; i0 += kThreads * kAhead) {
        long long v[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
          const int i = i0 + k * kThreads;
          v[k] = i < (int)len ? __ldg(ids + i) : -1;
        }
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
          const unsigned at = (unsigned)v[k] - (unsigned)begin;
          if (at >= room || (v[k] >> 32) != 0) continue;
          const int slot = (int)at + begin - origin;
          if (i0 + k * kThreads < prompt)
            C::mark(count, slot, C::kPrompt);
          else
            C::add(count, slot);
        }
      }
    }
    __syncthreads();
    // the biased tokens, biases added up in the list's order
    for (int k = 0; mine >> k; ++k) {
      if (!((mine >> k) & 1)) continue;
      const int i = k * kThreads + tid, v = (int)bias_ids[i];
      const unsigned c = count[v - origin] & ~C::kBiased;
      float sum = bias[i];
      if (s_twice) {
        sum = 0.f;
        for (int j = 0; j < a.num_bias; ++j)
          if (bias_ids[j] == v) sum += bias[j];
      }
      const float f = Num<T>::to_f(row[v]);
      s_value[i] = is_allowed(v) ? penalised(f, c) + sum : -INFINITY;
    }
    if (a.num_bias) __syncthreads();  // their logits are read before the pass writes them, where out is logits
  }
  // the pass
  const bool aligned =
      (reinterpret_cast<uintptr_t>(a.out) + (out_row + first) * (a.out_dtype == TREAD_F32 ? 4 : 2)) % 16 == 0;
  for (int i0 = tid; i0 < vecs; i0 += VECS * kThreads) {
    if (i0 != tid) load(i0);
#pragma unroll
    for (int k = 0; k < VECS; ++k) {
      const int i = i0 + k * kThreads;
      if (i >= vecs) continue;
      const int v = first + i * kVec;
      float f[kVec];
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        Vec16<T> u;
        u.raw = x[k][e * sizeof(T) / 16];
        f[e] = Num<T>::to_f(u.e[e % (16 / sizeof(T))]);
      }
      if (changes) {
#pragma unroll
        for (int j = 0; j < (int)sizeof(W) / 2; ++j) {
          constexpr int E = 16 / sizeof(W);
          Vec16<W> c;
          c.raw = reinterpret_cast<const int4*>(count + (i + 1) * kVec)[j];
          const unsigned any = c.raw.x | c.raw.y | c.raw.z | c.raw.w;
          if (!any) continue;
          if (product) {  // selects for all: a warp would go through every element's branch for one lane or another
#pragma unroll
            for (int e = 0; e < E; ++e) {
              const float x = f[j * E + e];
              f[j * E + e] = c.e[e] ? x * (x > 0.f ? inv : rep) : x;
            }
          } else {
            for (int e = 0; e < E; ++e)
              if (c.e[e]) f[j * E + e] = repeated(f[j * E + e]);
          }
          constexpr unsigned kCounts = sizeof(W) == 4 ? C::kCount : C::kCount * 0x10001u;
          if (any & kCounts) {  // few are in the output
#pragma unroll
            for (int e = 0; e < E; ++e)
              if (c.e[e] & C::kCount) f[j * E + e] = counted(f[j * E + e], c.e[e]);
          }
        }
      }
      if (allowed) {
        const int shift = v & 31;
        unsigned bits = allowed[v >> 5] >> shift;
        if (shift > 32 - kVec) bits |= allowed[(v >> 5) + 1] << (32 - shift);
#pragma unroll
        for (int e = 0; e < kVec; ++e)
          if (!((bits >> e) & 1)) f[e] = -INFINITY;
      }
      if (!aligned) {
#pragma unroll
        for (int e = 0; e < kVec; ++e) store(a.out, out_row + v + e, a.out_dtype, f[e]);
      } else if (a.out_dtype == TREAD_F32) {
        store8<float>(a.out, out_row + v, f);
      } else if (a.out_dtype == TREAD_BF16) {
        store8<__nv_bfloat16>(a.out, out_row + v, f);
      } else {
        store8<__half>(a.out, out_row + v, f);
      }
    }
  }
  // the first slice's tokens before its vectors (a short row may have no others), and the row's last ones
  auto single = [&](int v) {
    const float f = Num<T>::to_f(row[v]);
    const unsigned c = changes ? count[v - origin] : 0;
    store(a.out, out_row + v, a.out_dtype, is_allowed(v) ? penalised(f, c) : -INFINITY);
  };
  if (tid < min(first, end) - begin) single(begin + tid);
  if (tid < end - first - vecs * kVec) single(first + vecs * kVec + tid);
  if (!a.num_bias) return;
  __syncthreads();
  for (int k = 0; mine >> k; ++k)
    if ((mine >> k) & 1) store(a.out, out_row + bias_ids[k * kThreads + tid], a.out_dtype, s_value[k * kThreads + tid]);
}

template <typename T, typename W, int VECS>
int launch(const LogitsArgs& a, cudaStream_t st) {
  int device = 0, sms = 0;
  TREAD_CHECK_CUDA(cudaGetDevice(&device));
  TREAD_CHECK_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device));
  // equal slices, as many as run at once, down to one vector a thread
  constexpr int kPass = kThreads * kVec;
  int slices = sms * kCtas / a.B;
  const int most = (int)(((long long)a.V + kPass - 1) / kPass), least = (a.V + kMaxSlice - 1) / kMaxSlice;
  slices = slices > most ? most : slices < least ? least : slices;
  const int slice = (((a.V + slices - 1) / slices) + 63) / 64 * 64;  // whole vectors of counters
  const int smem = (slice + kVec) * (int)sizeof(W);
  auto kern = adjust_logits_kernel<T, W, VECS>;
  // the largest slice's, not this call's: another host thread may be between here and its launch
  if (smem > 24 * 1024)
    TREAD_CHECK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                          (kMaxSlice + kVec) * (int)sizeof(W)));
  kern<<<dim3(slices, a.B), kThreads, smem, st>>>(a, slice);
  TREAD_CHECK_LAUNCH("adjust_logits_kernel");
  return TREAD_OK;
}

template <typename T, int VECS>
int dispatch(const LogitsArgs& a, cudaStream_t st) {
  // counters of 16 bits (14 of them the count) halve the shared memory; a longer history needs 32
  return a.max_tokens < (1 << 14) ? launch<T, uint16_t, VECS>(a, st) : launch<T, uint32_t, VECS>(a, st);
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
  TREAD_CHECK_ARG(a.B <= 65535 && a.V <= INT32_MAX - (1 << 20),
                  "adjust_logits: more than 65535 rows or 2^31 - 2^20 tokens");
  TREAD_CHECK_ARG(dtype_size(a.dtype) != 0 && dtype_size(a.out_dtype) != 0, "adjust_logits: unknown dtype %d or %d",
                  a.dtype, a.out_dtype);
  // an input's row stride may be 0: one row for all
  TREAD_CHECK_ARG(a.B == 1 || ((a.ld == 0 || a.ld >= a.V) && a.ld_out >= a.V),
                  "adjust_logits: row stride below the vocabulary");
  // a count fits below a 32-bit counter's two marks
  TREAD_CHECK_ARG(a.max_tokens >= 0 && a.max_tokens < (1 << 30) &&
                      (!a.tokens || a.B == 1 || a.tokens_ld == 0 || a.tokens_ld >= a.max_tokens),
                  "adjust_logits: bad history");
  TREAD_CHECK_ARG(a.num_bias <= kMaxBias, "adjust_logits: more than %d biases", kMaxBias);
  TREAD_CHECK_ARG(a.num_bias >= 0 && (a.num_bias == 0 || (a.bias_ids && a.bias)), "adjust_logits: bad biases");
  TREAD_CHECK_ARG(a.repetition || a.repetition_all > 0.f, "adjust_logits: repetition must be above 0");
  if (!a.tokens) a.max_tokens = 0;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  switch (a.dtype) {
    case TREAD_BF16: return dispatch<__nv_bfloat16, 3>(a, st);
    case TREAD_F16: return dispatch<__half, 3>(a, st);
    default: return dispatch<float, 2>(a, st);
  }
}
