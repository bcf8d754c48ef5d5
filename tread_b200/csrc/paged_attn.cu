// Attention of one new token per sequence over a paged key-value cache (sm_100a).
//
//   out[b, h] = sum_t softmax_t(scale * q[b, h] . K[t, g]) V[t, g],   t < lens[b], g = h / (Hq / Hkv)
// where token t's keys and values lie in slot t % page_size of page table[b][t / page_size]. Where no
// key has a score above -inf, or there is none, the softmax has no value and the output is zero.
#include "common.cuh"

namespace tread {
namespace {

constexpr int kTile = 32;

struct DecodeArgs {
  const void* q;
  const void* k_pages;
  const void* v_pages;
  void* out;
  long long q_ld, page_stride, head_stride, num_pages, table_ld;
  const int32_t* table;
  const int64_t* lens;
  int B, Hq, Hkv, max_pages, page_size;
  float scale;
  unsigned* err;
};

// The simplest form: one CTA per (sequence, KV head), one warp per query head of the group, 32 keys at a
// time through shared memory.
template <typename T, int D>
__global__ void paged_attn_kernel(const __grid_constant__ DecodeArgs a) {
  constexpr int DPL = D / 32;
  extern __shared__ float smem[];
  const int G = a.Hq / a.Hkv;
  float* qs = smem;                  // [G][D]
  float* ks = qs + G * D;            // [kTile][D + 1]
  float* vs = ks + kTile * (D + 1);  // [kTile][D]
  __shared__ long long s_row[kTile];
  const int b = blockIdx.x, g = blockIdx.y;
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  long long n = a.lens[b];
  if (n < 0 || n > (long long)a.max_pages * a.page_size) {
    if (threadIdx.x == 0 && a.err) atomicOr(a.err, 2u);
    n = 0;
  }
  for (int i = threadIdx.x; i < G * D; i += blockDim.x)
    qs[i] = Num<T>::to_f(static_cast<const T*>(a.q)[b * a.q_ld + (long long)g * G * D + i]);
  float m = -INFINITY, l = 0.f, o[DPL];
#pragma unroll
  for (int k = 0; k < DPL; ++k) o[k] = 0.f;
  for (long long t0 = 0; t0 < n; t0 += kTile) {
    const int nt = (int)(n - t0 < kTile ? n - t0 : kTile);
    __syncthreads();
    if (threadIdx.x < kTile) {
      long long row = -1;
      if (threadIdx.x < nt) {
        const long long t = t0 + threadIdx.x, pg = t / a.page_size;
        const int id = a.table[b * a.table_ld + pg];
        if (id >= 0 && id < a.num_pages)
          row = id * a.page_stride + g * a.head_stride + (t - pg * a.page_size) * D;
        else if (a.err)
          atomicOr(a.err, 2u);
      }
      s_row[threadIdx.x] = row;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < kTile * D; i += blockDim.x) {
      const int j = i / D, d = i - j * D;
      float kv = 0.f, vv = 0.f;
      if (s_row[j] >= 0) {
        kv = Num<T>::to_f(static_cast<const T*>(a.k_pages)[s_row[j] + d]);
        vv = Num<T>::to_f(static_cast<const T*>(a.v_pages)[s_row[j] + d]);
      }
      ks[j * (D + 1) + d] = kv;
      vs[j * D + d] = vv;
    }
    __syncthreads();
    float s = -INFINITY;
    if (s_row[lane] >= 0) {
      float acc = 0.f;
#pragma unroll 8
      for (int d = 0; d < D; ++d) acc = fmaf(qs[w * D + d], ks[lane * (D + 1) + d], acc);
      s = acc * a.scale;
    }
    float top = s;
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
    const float m_new = fmaxf(m, top);
    if (m_new == -INFINITY) continue;  // no key so far
    const float p = s_row[lane] >= 0 ? expf(s - m_new) : 0.f;
    const float alpha = expf(m - m_new);
    float sum = p;
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    l = l * alpha + sum;
#pragma unroll
    for (int k = 0; k < DPL; ++k) o[k] *= alpha;
    for (int j = 0; j < kTile; ++j) {
      const float pj = __shfl_sync(0xffffffffu, p, j);
#pragma unroll
      for (int k = 0; k < DPL; ++k) o[k] = fmaf(pj, vs[j * D + lane + 32 * k], o[k]);
    }
    m = m_new;
  }
  T* row = static_cast<T*>(a.out) + ((long long)b * a.Hq + g * G + w) * D;
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int k = 0; k < DPL; ++k) row[lane + 32 * k] = Num<T>::from_f(o[k] * inv);
}

template <typename T, int D>
int launch(const DecodeArgs& a, cudaStream_t st) {
  const int G = a.Hq / a.Hkv;
  const int smem = (int)sizeof(float) * (G * D + kTile * (D + 1) + kTile * D);
  auto kern = paged_attn_kernel<T, D>;
  if (smem > 48 * 1024 - 512)
    TREAD_CHECK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  kern<<<dim3(a.B, a.Hkv), 32 * G, smem, st>>>(a);
  TREAD_CHECK_LAUNCH("paged_attn_kernel");
  return TREAD_OK;
}

template <typename T>
int dispatch(int D, const DecodeArgs& a, cudaStream_t st) {
  switch (D) {
    case 64: return launch<T, 64>(a, st);
    case 128: return launch<T, 128>(a, st);
    default: return launch<T, 256>(a, st);
  }
}

}  // namespace
}  // namespace tread

extern "C" size_t tread_paged_attn_workspace_bytes(int Hq, int Hkv, int D) { return 0; }

extern "C" int tread_paged_attn(const void* q, int64_t q_ld, const void* k_pages, const void* v_pages,
                                int64_t page_stride, int64_t head_stride, int64_t num_pages, int page_size,
                                const int32_t* table, int64_t table_ld, int max_pages, const int64_t* lens, int B,
                                int Hq, int Hkv, int D, float sm_scale, void* out, int dtype, void* err_flag,
                                void* workspace, size_t workspace_bytes, tread_stream_t stream) {
  using namespace tread;
  TREAD_CHECK_ARG(B >= 0, "paged_attn: B < 0");
  if (B == 0) return TREAD_OK;
  TREAD_CHECK_ARG(q && k_pages && v_pages && lens && out, "paged_attn: null pointer");
  TREAD_CHECK_ARG(Hq > 0 && Hkv > 0 && Hkv <= 65535 && Hq % Hkv == 0 && Hq / Hkv <= 16,
                  "paged_attn: bad heads Hq=%d Hkv=%d", Hq, Hkv);
  TREAD_CHECK_ARG(D == 64 || D == 128 || D == 256, "paged_attn: head_dim %d not in {64,128,256}", D);
  TREAD_CHECK_ARG(dtype_size(dtype) != 0, "paged_attn: unknown dtype %d", dtype);
  TREAD_CHECK_ARG(page_size > 0 && num_pages >= 0 && num_pages <= INT32_MAX &&
                      (num_pages <= 1 || page_stride >= (int64_t)page_size * D) &&
                      (Hkv == 1 || head_stride >= (int64_t)page_size * D),
                  "paged_attn: bad page geometry");
  TREAD_CHECK_ARG(max_pages >= 0 && (table || max_pages == 0) && (B <= 1 || table_ld >= max_pages),
                  "paged_attn: bad page table");
  DecodeArgs a;
  a.q = q, a.k_pages = k_pages, a.v_pages = v_pages, a.out = out, a.q_ld = q_ld, a.page_stride = page_stride;
  a.head_stride = head_stride, a.num_pages = num_pages, a.table_ld = table_ld, a.table = table, a.lens = lens;
  a.B = B, a.Hq = Hq, a.Hkv = Hkv, a.max_pages = max_pages, a.page_size = page_size, a.scale = sm_scale;
  a.err = static_cast<unsigned*>(err_flag);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  switch (dtype) {
    case TREAD_BF16: return dispatch<__nv_bfloat16>(D, a, st);
    case TREAD_F16: return dispatch<__half>(D, a, st);
    default: return dispatch<float>(D, a, st);
  }
}
