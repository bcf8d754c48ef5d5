// Adjusting the logits of the next token: penalties for repeated tokens, biases, a grammar's mask (sm_100a).
//
// Per row, with n[v] the count of token v in tokens[prompt_len : len] and seen[v] whether it is in
// tokens[0 : len]:
//   x = logits[v];   seen[v]: x = x > 0 ? x / repetition : x * repetition
//   x -= frequency * n[v] + presence * (n[v] > 0);   x += bias of v;   v not allowed: x = -inf
// in fp32, rounded once to the output's type. Ids outside [0, vocab) count for nothing (padding).
//
// Bound by reading the logits and writing the result. A CTA owns a slice of a row's vocabulary: it issues
// the loads of all its logits, counts the row's whole history into counters of its slice in shared memory
// while they fly (whole numbers: the order of the atomics does not matter), then stores every logit, masked,
// in vectors, and goes back to the few that the history or a bias changes: done in the vectors' own code
// they cost a division's instructions for nearly every warp. Reading the history again for every slice costs
// L2 reads only, and no counters in memory that a caller would have to keep or clear. A biased token is
// finished by the thread that marked it first.
#include "common.cuh"

namespace tread {
namespace {

constexpr int kThreads = 256;
constexpr int kCtas = 4;         // CTAs of an SM
constexpr int kVec = 8;          // consecutive logits of a thread
constexpr int kMaxBias = 8192;   // 32 bits of ownership a thread

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

// element e of a vector held in registers
template <typename T>
__device__ __forceinline__ float pick(const int4 (&x)[kVec * sizeof(T) / 16], int e) {
  constexpr int kPer = 4 / sizeof(T);  // elements of a word
  const int w = e / kPer;
  unsigned word = 0;
#pragma unroll
  for (int j = 0; j < (int)(kVec * sizeof(T) / 4); ++j) {
    const int4& q = x[j / 4];
    const unsigned y = j % 4 == 0 ? q.x : j % 4 == 1 ? q.y : j % 4 == 2 ? q.z : q.w;
    if (w == j) word = y;
  }
  if constexpr (kPer == 2) {
    const unsigned short h = (unsigned short)(e & 1 ? word >> 16 : word);
    return Num<T>::to_f(*reinterpret_cast<const T*>(&h));
  } else {
    return __uint_as_float(word);
  }
}

// VECS: vectors of kVec logits that a thread holds; a slice has VECS * kThreads of them at most
template <typename T, typename W, int VECS>
__global__ void __launch_bounds__(kThreads, kCtas)
    adjust_logits_kernel(const __grid_constant__ LogitsArgs a, int slice) {
  using C = Counter<W>;
  extern __shared__ __align__(16) unsigned char s_mem[];
  __shared__ int s_twice;                  // some token of the slice has more than one bias
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
  constexpr int L = kVec * sizeof(T) / 16;                   // 16-byte loads of a vector
  int4 x[VECS][L];
#pragma unroll
  for (int k = 0; k < VECS; ++k) {
    const int i = k * kThreads + threadIdx.x;
    if (i < vecs) {
#pragma unroll
      for (int j = 0; j < L; ++j) x[k][j] = ld_stream(row + first + i * kVec + j * (16 / sizeof(T)));
    }
  }
  const int origin = first - kVec;
  for (int i = threadIdx.x; i < (int)((slice + kVec) * sizeof(W) / 16); i += kThreads)
    reinterpret_cast<int4*>(s_mem)[i] = make_int4(0, 0, 0, 0);
  if (threadIdx.x == 0) s_twice = 0;
  __syncthreads();
  if (a.tokens) {
    long long len = a.lens ? a.lens[b] : a.max_tokens;
    len = len < 0 ? 0 : len > a.max_tokens ? a.max_tokens : len;
    const long long prompt = a.prompt_lens ? a.prompt_lens[b] : 0;
    const long long* ids = reinterpret_cast<const long long*>(a.tokens) + b * a.tokens_ld;
    constexpr int kAhead = 4;
    for (int i0 = threadIdx.x; i0 < (int)len; i0 += kThreads * kAhead) {
      long long v[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) v[k] = i0 + k * kThreads < (int)len ? __ldg(ids + i0 + k * kThreads) : -1;
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        if (v[k] < begin || v[k] >= end) continue;
        if (i0 + k * kThreads < prompt)
          C::mark(count, (int)v[k] - origin, C::kPrompt);
        else
          C::add(count, (int)v[k] - origin);
      }
    }
  }
  unsigned mine = 0;  // biases whose token this thread marked first
  const int64_t* bias_ids = a.bias_ids + b * a.bias_ids_ld;
  const float* bias = a.bias + b * a.bias_ld;
  for (int i = threadIdx.x, k = 0; i < a.num_bias; i += kThreads, ++k) {
    const long long v = bias_ids[i];
    if (v < begin || v >= end) continue;
    if (C::mark(count, (int)v - origin, C::kBiased) & C::kBiased)
      s_twice = 1;
    else
      mine |= 1u << k;
  }
  __syncthreads();
  const float rep = a.repetition ? a.repetition[b] : a.repetition_all;
  const float pres = a.presence ? a.presence[b] : a.presence_all;
  const float freq = a.frequency ? a.frequency[b] : a.frequency_all;
  const unsigned* allowed = a.allowed ? reinterpret_cast<const unsigned*>(a.allowed) + b * a.allowed_ld : nullptr;
  auto is_allowed = [&](int v) { return !allowed || (allowed[v >> 5] >> (v & 31)) & 1; };
  auto penalised = [&](float f, unsigned c) {
    if (c & ~C::kBiased) {
      f = f > 0.f ? f / rep : f * rep;
      if (c & C::kCount) f -= freq * (float)(c & C::kCount) + pres;
    }
    return f;
  };
  const bool aligned =
      (reinterpret_cast<uintptr_t>(a.out) + (out_row + first) * (a.out_dtype == TREAD_F32 ? 4 : 2)) % 16 == 0;
#pragma unroll
  for (int k = 0; k < VECS; ++k) {
    const int i = k * kThreads + threadIdx.x;
    if (i >= vecs) continue;
    const int v = first + i * kVec;
    float f[kVec];
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      Vec16<T> u;
      u.raw = x[k][e * sizeof(T) / 16];
      f[e] = Num<T>::to_f(u.e[e % (16 / sizeof(T))]);
    }
    unsigned bits = 0xff;
    if (allowed) {
      const int shift = v & 31;
      bits = allowed[v >> 5] >> shift;
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
    // which of them the history changes: those again (a biased token is another thread's)
    const W* c = count + (i + 1) * kVec;
    unsigned changed = 0;
#pragma unroll
    for (int j = 0; j < (int)sizeof(W) / 2; ++j) {
      const int4 q = reinterpret_cast<const int4*>(c)[j];
      if (q.x | q.y | q.z | q.w) {
#pragma unroll
        for (int e = 0; e < 16 / (int)sizeof(W); ++e) {
          const unsigned w = e * sizeof(W) / 4 == 0 ? q.x : e * sizeof(W) / 4 == 1 ? q.y : e * sizeof(W) / 4 == 2 ? q.z : q.w;
          const unsigned n = sizeof(W) == 4 ? w : (w >> ((e & 1) * 16)) & 0xffffu;
          if (n && !(n & C::kBiased)) changed |= 1u << (j * (16 / sizeof(W)) + e);
        }
      }
    }
    changed &= bits;
    while (changed) {
      const int e = __ffs(changed) - 1;
      changed &= changed - 1;
      store(a.out, out_row + v + e, a.out_dtype, penalised(pick<T>(x[k], e), c[e]));
    }
  }
  auto single = [&](int v) {
    const unsigned c = count[v - origin];
    if (c & C::kBiased) return;
    const float f = Num<T>::to_f(row[v]);
    store(a.out, out_row + v, a.out_dtype, is_allowed(v) ? penalised(f, c) : -INFINITY);
  };
  // the first slice's tokens before its vectors (a short row may have no others), and the row's last ones
  const int tid = threadIdx.x;
  if (tid < min(first, end) - begin) single(begin + tid);
  if (tid < end - first - vecs * kVec) single(first + vecs * kVec + tid);
  if (a.num_bias) {
    // behind the vectors' stores; where out is logits, an allowed token still has its logit
    __syncthreads();
    for (int k = 0; k < 32 && (mine >> k); ++k) {
      if (!((mine >> k) & 1)) continue;
      const int i = k * kThreads + threadIdx.x;
      const int v = (int)bias_ids[i];
      float sum = bias[i];
      if (s_twice) {
        sum = 0.f;
        for (int j = 0; j < a.num_bias; ++j)
          if (bias_ids[j] == v) sum += bias[j];
      }
      store(a.out, out_row + v, a.out_dtype,
            is_allowed(v) ? penalised(Num<T>::to_f(row[v]), count[v - origin]) + sum : -INFINITY);
    }
  }
}

template <typename T, typename W, int VECS>
int launch(const LogitsArgs& a, cudaStream_t st) {
  int device = 0, sms = 0;
  TREAD_CHECK_CUDA(cudaGetDevice(&device));
  TREAD_CHECK_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device));
  // equal slices, as many as run at once, down to one vector a thread
  constexpr int kPass = kThreads * kVec;
  int slices = sms * kCtas / a.B;
  const int most = (int)(((long long)a.V + kPass - 1) / kPass), least = (most + VECS - 1) / VECS;
  slices = slices > most ? most : slices < least ? least : slices;
  const int slice = (((a.V + slices - 1) / slices) + 63) / 64 * 64;  // whole vectors of counters
  const int smem = (slice + kVec) * (int)sizeof(W);
  auto kern = adjust_logits_kernel<T, W, VECS>;
  if (smem > 48 * 1024) TREAD_CHECK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
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
  TREAD_CHECK_ARG(a.B <= 65535 && a.V <= INT32_MAX - (1 << 20), "adjust_logits: more than 65535 rows or 2^31 - 2^20 tokens");
  TREAD_CHECK_ARG(dtype_size(a.dtype) != 0 && dtype_size(a.out_dtype) != 0, "adjust_logits: unknown dtype %d or %d",
                  a.dtype, a.out_dtype);
  TREAD_CHECK_ARG(a.B == 1 || (a.ld >= a.V && a.ld_out >= a.V), "adjust_logits: row stride below the vocabulary");
  TREAD_CHECK_ARG(a.max_tokens >= 0 && (!a.tokens || a.B == 1 || a.tokens_ld >= a.max_tokens),
                  "adjust_logits: bad history");
  TREAD_CHECK_ARG(a.num_bias <= kMaxBias, "adjust_logits: more than %d biases", kMaxBias);
  TREAD_CHECK_ARG(a.num_bias >= 0 && (a.num_bias == 0 || (a.bias_ids && a.bias)), "adjust_logits: bad biases");
  TREAD_CHECK_ARG(a.repetition || a.repetition_all > 0.f, "adjust_logits: repetition must be above 0");
  if (!a.tokens) a.max_tokens = 0;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  switch (a.dtype) {
    case TREAD_BF16: return dispatch<__nv_bfloat16, 9>(a, st);
    case TREAD_F16: return dispatch<__half, 9>(a, st);
    default: return dispatch<float, 4>(a, st);
  }
}
