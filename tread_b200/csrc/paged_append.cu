// Appending keys and values to a paged cache, with the position rotation applied on the way (sm_100a).
//
// Row r of the new keys / values belongs to token pos[r] of sequence seq[r]. Its place is
//   page = table[seq[r]][pos[r] / page_size],  slot = pos[r] % page_size
// in pools of pages [page][Hkv][page_size][D]. Keys (and the rows' query heads, if given) are rotated by
//   angle_i = rope_pos[r] * inv_freq[i];  c = cos(angle_i) * s,  w = sin(angle_i) * s
//   x'[i] = x[i] * c - x[i + D/2] * w,  x'[i + D/2] = x[i + D/2] * c + x[i] * w      (i < D/2)
// in fp32, rounded once. The angle's product is formed in 64 bits, in units of half turns, and its whole
// turns are dropped before it is rounded to 32: a far position keeps every digit (in 32 bits, position
// 16384 would already lose 1e-3 rad).
//
// The work is reading (Hq + 2 Hkv) D elements a row and writing as many: bound by memory for a prompt,
// by latency for a few tokens. One CTA takes a tile of rows and computes their places and cosines once in
// shared memory; a group of D/2/VEC threads moves one head of one row, 16 bytes of each half a thread.
#include "common.cuh"

namespace tread {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxHalf = 128;
constexpr int kMaxTile = 16;  // rows per CTA
constexpr int kUnroll = 4;    // pieces (one head of one row) in flight per thread

using AppendArgs = tread_paged_append_args;

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T e[VEC];
};

template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) paged_append_kernel(const __grid_constant__ AppendArgs a, int tile_log2) {
  using P = Pack<T, VEC>;
  __shared__ long long s_dst[kMaxTile];  // element offset of the row's slot in the pools, -1: skip
  __shared__ float2 s_cs[kMaxTile * kMaxHalf];
  const int tile = 1 << tile_log2;
  const long long r0 = (long long)blockIdx.x << tile_log2;
  const int half = a.D >> 1;
  if (threadIdx.x < tile) {
    const long long r = r0 + threadIdx.x;
    long long dst = -1;
    if (r < a.R) {
      const long long p = a.pos[r];
      if (p >= 0) {  // a negative position marks a padding row
        const int s = a.seq ? a.seq[r] : (int)r;
        const long long pg = p / a.page_size;
        bool ok = s >= 0 && s < a.num_seqs && pg < a.max_pages;
        if (ok) {
          const int id = a.table[s * a.table_ld + pg];
          ok = id >= 0 && id < a.num_pages;
          if (ok) dst = id * a.page_stride + (p - pg * a.page_size) * a.D;
        }
        if (!ok && a.err_flag) atomicOr(static_cast<unsigned*>(a.err_flag), 1u);
      }
    }
    s_dst[threadIdx.x] = dst;
  }
  if (a.inv_freq) {
    for (int w = threadIdx.x; w < tile * half; w += kThreads) {
      const int t = w / half, i = w - t * half;
      const long long r = r0 + t;
      if (r < a.R) {
        const double half_turns = (double)a.rope_pos[r] * (double)a.inv_freq[i] * 0.31830988618379067154;
        float sn, cs;
        sincospif((float)(half_turns - 2.0 * rint(0.5 * half_turns)), &sn, &cs);
        s_cs[w] = make_float2(cs * a.attn_scaling, sn * a.attn_scaling);
      }
    }
  }
  __syncthreads();
  const int hv = half / VEC;                   // threads of one piece
  const int per_pass = kThreads / hv;          // pieces of one pass over the CTA
  const int piece0 = threadIdx.x / hv, i0 = (threadIdx.x - piece0 * hv) * VEC;
  if (piece0 >= per_pass) return;
  const int heads = a.Hq + 2 * a.Hkv;
  const int n = heads << tile_log2;
  const int stride = per_pass * gridDim.y;
  for (int p0 = piece0 + blockIdx.y * per_pass; p0 < n; p0 += stride * kUnroll) {
    P x1[kUnroll], x2[kUnroll];
    T* to[kUnroll];
    int cs[kUnroll];  // offset of the row's cosines, -1: copy, -2: write zeros
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int p = p0 + u * stride;
      to[u] = nullptr;
      if (p >= n) continue;
      const int t = p & (tile - 1), h = p >> tile_log2;
      const long long r = r0 + t, dst = s_dst[t];
      if (r >= a.R) continue;
      const T* from;
      cs[u] = a.inv_freq ? t * half : -1;
      if (h < a.Hq) {
        from = static_cast<const T*>(a.q) + r * a.q_ld + h * a.q_sh;
        to[u] = static_cast<T*>(a.q_out) + (r * a.Hq + h) * a.D;
        if (dst < 0) cs[u] = -2;
      } else if (dst < 0) {
        continue;
      } else if (h < a.Hq + a.Hkv) {
        from = static_cast<const T*>(a.k) + r * a.k_ld + (h - a.Hq) * a.k_sh;
        to[u] = static_cast<T*>(a.k_pages) + dst + (h - a.Hq) * a.head_stride;
      } else {
        const int g = h - a.Hq - a.Hkv;
        from = static_cast<const T*>(a.v) + r * a.v_ld + g * a.v_sh;
        to[u] = static_cast<T*>(a.v_pages) + dst + g * a.head_stride;
        cs[u] = -1;
      }
      x1[u] = *reinterpret_cast<const P*>(from + i0);
      x2[u] = *reinterpret_cast<const P*>(from + i0 + half);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      if (!to[u]) continue;
      if (cs[u] >= 0) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float2 c = s_cs[cs[u] + i0 + e];
          const float y1 = Num<T>::to_f(x1[u].e[e]), y2 = Num<T>::to_f(x2[u].e[e]);
          x1[u].e[e] = Num<T>::from_f(y1 * c.x - y2 * c.y);
          x2[u].e[e] = Num<T>::from_f(y2 * c.x + y1 * c.y);
        }
      } else if (cs[u] == -2) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) x1[u].e[e] = x2[u].e[e] = Num<T>::from_f(0.f);
      }
      *reinterpret_cast<P*>(to[u] + i0) = x1[u];
      *reinterpret_cast<P*>(to[u] + i0 + half) = x2[u];
    }
  }
}

template <typename T>
int launch(const AppendArgs& a, bool vec, cudaStream_t st) {
  int tile_log2 = 0;
  while ((1 << tile_log2) < kMaxTile && ((long long)a.R >> tile_log2) > 512) ++tile_log2;
  constexpr int VEC = 16 / sizeof(T);
  const long long tiles = ((long long)a.R + (1 << tile_log2) - 1) >> tile_log2;
  const int hv = (a.D / 2) / (vec ? VEC : 1), per_pass = kThreads / hv;
  const long long passes = (((long long)(a.Hq + 2 * a.Hkv) << tile_log2) + per_pass - 1) / per_pass;
  long long split = (592 + tiles - 1) / tiles;  // head splits until every SM has a few CTAs
  const long long most = (passes + kUnroll - 1) / kUnroll;
  if (split > most) split = most;
  if (split < 1) split = 1;
  dim3 grid((unsigned)tiles, (unsigned)split);
  if (vec)
    paged_append_kernel<T, VEC><<<grid, kThreads, 0, st>>>(a, tile_log2);
  else
    paged_append_kernel<T, 1><<<grid, kThreads, 0, st>>>(a, tile_log2);
  TREAD_CHECK_LAUNCH("paged_append_kernel");
  return TREAD_OK;
}

}  // namespace
}  // namespace tread

extern "C" int tread_paged_append(const tread_paged_append_args* args, tread_stream_t stream) {
  using namespace tread;
  TREAD_CHECK_ARG(args, "paged_append: null arguments");
  AppendArgs a = *args;
  TREAD_CHECK_ARG(a.R >= 0, "paged_append: R < 0");
  if (a.R == 0) return TREAD_OK;
  TREAD_CHECK_ARG(a.k && a.v && a.k_pages && a.v_pages && a.pos, "paged_append: null pointer");
  TREAD_CHECK_ARG(a.Hkv > 0 && a.Hkv <= 65535 && a.Hq >= 0 && a.Hq <= 65535, "paged_append: bad heads Hq=%d Hkv=%d",
                  a.Hq, a.Hkv);
  TREAD_CHECK_ARG(a.D >= 2 && a.D % 2 == 0 && a.D / 2 <= kMaxHalf, "paged_append: bad head_dim %d", a.D);
  TREAD_CHECK_ARG(a.Hq == 0 || (a.q && a.q_out && a.inv_freq), "paged_append: query heads need q, q_out and inv_freq");
  TREAD_CHECK_ARG(dtype_size(a.dtype) != 0, "paged_append: unknown dtype %d", a.dtype);
  TREAD_CHECK_ARG(a.page_size > 0 && a.num_pages >= 0 && a.num_pages <= INT32_MAX &&
                      (a.num_pages <= 1 || a.page_stride >= (int64_t)a.page_size * a.D) &&
                      (a.Hkv == 1 || a.head_stride >= (int64_t)a.page_size * a.D),
                  "paged_append: bad page geometry");
  TREAD_CHECK_ARG(a.num_seqs >= 0 && a.max_pages >= 0 && (a.table || a.num_seqs == 0 || a.max_pages == 0) &&
                      (a.num_seqs <= 1 || a.table_ld >= a.max_pages),
                  "paged_append: bad page table");
  TREAD_CHECK_ARG(a.seq || a.R <= a.num_seqs, "paged_append: %d rows without seq, but %d sequences", a.R, a.num_seqs);
  if (!a.rope_pos) a.rope_pos = a.pos;
  // 16-byte vectors where every head of every row starts on a 16-byte boundary, else single elements
  const int64_t ve = 16 / (int64_t)dtype_size(a.dtype);
  const bool vec = (a.D / 2) % ve == 0 && (a.k_ld | a.k_sh | a.v_ld | a.v_sh | a.page_stride | a.head_stride) % ve == 0 &&
                   (a.Hq == 0 || (a.q_ld | a.q_sh) % ve == 0) && aligned16(a.k) && aligned16(a.v) &&
                   aligned16(a.k_pages) && aligned16(a.v_pages) && (a.Hq == 0 || (aligned16(a.q) && aligned16(a.q_out)));
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  switch (a.dtype) {
    case TREAD_BF16: return launch<__nv_bfloat16>(a, vec, st);
    case TREAD_F16: return launch<__half>(a, vec, st);
    default: return launch<float>(a, vec, st);
  }
}
