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
// The work is reading (Hq + 2 Hkv) D elements a row and writing as many: bound by memory for a prompt, by
// latency for a few tokens. A thread owns VEC columns of either half (16 bytes each) of one row and walks over
// heads, so it reads its cosines once, from a table that the CTA computes together, and keeps them in
// registers; two heads' loads are in flight together (four: 20 % slower, 80 registers leave fewer warps). A
// tile of rows times a part of the heads is a CTA. Loads and stores pass the caches as streams, which is what
// carries it: without the hints 104 us instead of 79 at 16640 rows of 56 heads of 128 (6.0 TB/s, 0.92 of the
// copy rate), and 173 instead of 150 us at 8256 rows of 224 heads (6.3 TB/s, 0.97).
#include "common.cuh"

namespace tread {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxHalf = 128;
constexpr int kMaxTile = 64;  // rows per CTA
constexpr int kUnroll = 2;    // heads in flight per thread

using AppendArgs = tread_paged_append_args;

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T e[VEC];
};

template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> load(const T* p) {
  Pack<T, VEC> x;
  if constexpr (sizeof(x) == 16)
    *reinterpret_cast<int4*>(&x) = ld_stream(p);
  else
    x = *reinterpret_cast<const Pack<T, VEC>*>(p);
  return x;
}
template <typename T, int VEC>
__device__ __forceinline__ void store(T* p, const Pack<T, VEC>& x) {
  if constexpr (sizeof(x) == 16)
    st_stream(p, *reinterpret_cast<const int4*>(&x));
  else
    *reinterpret_cast<Pack<T, VEC>*>(p) = x;
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads, 4) paged_append_kernel(const __grid_constant__ AppendArgs a, int tile_log2) {
  using P = Pack<T, VEC>;
  __shared__ long long s_dst[kMaxTile];  // element offset of the row's slot in the pools, -1: skip
  __shared__ float2 s_cs[kThreads * VEC];  // [row of the tile][column]: a tile has kThreads / (half / VEC) rows at most
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
    const int rows = kThreads / half, i = (int)threadIdx.x % half;  // a thread stays in its column
    const double turn = (double)a.inv_freq[i] * 0.31830988618379067154;  // half turns a position
    for (int w = (int)threadIdx.x < rows * half ? (int)threadIdx.x / half : tile; w < tile && r0 + w < a.R; w += rows) {
      const double half_turns = (double)a.rope_pos[r0 + w] * turn;
      float sn, cs;
      sincospif((float)(half_turns - 2.0 * rint(0.5 * half_turns)), &sn, &cs);
      s_cs[w * half + i] = make_float2(cs * a.attn_scaling, sn * a.attn_scaling);
    }
  }
  __syncthreads();
  const int hv = half / VEC;  // threads of one head of one row
  const int place = threadIdx.x / hv, i0 = ((int)threadIdx.x - place * hv) * VEC;
  const int lanes = kThreads / hv >> tile_log2;  // heads side by side
  const int t = place & (tile - 1), lane = place >> tile_log2;
  const long long r = r0 + t;
  if (lane >= lanes || r >= a.R) return;
  const long long dst = s_dst[t];
  float cs[VEC], sn[VEC];
  if (a.inv_freq) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const float2 c = s_cs[t * half + i0 + e];
      cs[e] = c.x, sn[e] = c.y;
    }
  }
  const T* q = static_cast<const T*>(a.q) + r * a.q_ld + i0;
  const T* k = static_cast<const T*>(a.k) + r * a.k_ld + i0;
  const T* v = static_cast<const T*>(a.v) + r * a.v_ld + i0;
  T* q_out = static_cast<T*>(a.q_out) + r * a.Hq * a.D + i0;
  T* k_to = static_cast<T*>(a.k_pages) + dst + i0;
  T* v_to = static_cast<T*>(a.v_pages) + dst + i0;
  const int heads = dst < 0 ? a.Hq : a.Hq + 2 * a.Hkv;  // a row without a place: its queries only
  const int step = lanes * gridDim.y;
  for (int h0 = lane + lanes * (int)blockIdx.y; h0 < heads; h0 += step * kUnroll) {
    P x1[kUnroll], x2[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int h = h0 + u * step, g = h - a.Hq;
      if (h >= heads) break;
      const T* from = g < 0 ? q + h * a.q_sh : g < a.Hkv ? k + g * a.k_sh : v + (g - a.Hkv) * a.v_sh;
      x1[u] = load<T, VEC>(from);
      x2[u] = load<T, VEC>(from + half);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int h = h0 + u * step, g = h - a.Hq;
      if (h >= heads) break;
      T* to = g < 0        ? q_out + (long long)h * a.D
              : g < a.Hkv ? k_to + g * a.head_stride
                          : v_to + (g - a.Hkv) * a.head_stride;
      if (dst < 0) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) x1[u].e[e] = x2[u].e[e] = Num<T>::from_f(0.f);
      } else if (g < a.Hkv && a.inv_freq) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float y1 = Num<T>::to_f(x1[u].e[e]), y2 = Num<T>::to_f(x2[u].e[e]);
          x1[u].e[e] = Num<T>::from_f(y1 * cs[e] - y2 * sn[e]);
          x2[u].e[e] = Num<T>::from_f(y2 * cs[e] + y1 * sn[e]);
        }
      }
      store<T, VEC>(to, x1[u]);
      store<T, VEC>(to + half, x2[u]);
    }
  }
}

template <typename T>
int launch(const AppendArgs& a, bool vec, cudaStream_t st) {
  constexpr int VEC = 16 / sizeof(T);
  const int hv = (a.D / 2) / (vec ? VEC : 1), places = kThreads / hv;
  int device = 0, sms = 0;
  TREAD_CHECK_CUDA(cudaGetDevice(&device));
  TREAD_CHECK_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device));
  // a CTA's places are rows first (each row's cosines are then found once), as far as there are rows for eight
  // CTAs an SM, then heads. Rows for two an SM take 81 us instead of 79 at 16640 rows of 56 heads of 128, and
  // heads split until an SM has eight CTAs instead of four, 86.
  int tile_log2 = 0;
  while ((2 << tile_log2) <= places && (2 << tile_log2) <= kMaxTile && (a.R >> (tile_log2 + 1)) >= 8 * sms) ++tile_log2;
  const long long tiles = ((long long)a.R + (1 << tile_log2) - 1) >> tile_log2;
  const int lanes = places >> tile_log2;
  const long long passes = (a.Hq + 2LL * a.Hkv + lanes * kUnroll - 1) / (lanes * kUnroll);
  long long split = (4 * sms + tiles - 1) / tiles;
  if (split > passes) split = passes;
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
                      (a.num_seqs <= 1 || a.table_ld == 0 || a.table_ld >= a.max_pages),
                  "paged_append: bad page table");
  TREAD_CHECK_ARG(a.seq || a.R <= a.num_seqs, "paged_append: %d rows without seq, but %d sequences", a.R, a.num_seqs);
  if (!a.rope_pos) a.rope_pos = a.pos;
  // the stride of a dimension of one is any number
  if (a.R == 1) a.k_ld = a.v_ld = a.q_ld = 0;
  if (a.Hq == 1) a.q_sh = 0;
  if (a.Hkv == 1) a.k_sh = a.v_sh = a.head_stride = 0;
  if (a.num_pages <= 1) a.page_stride = 0;
  // 16-byte vectors where every head of every row starts on a 16-byte boundary, else single elements
  const int64_t ve = 16 / (int64_t)dtype_size(a.dtype);
  const int64_t strides = a.k_ld | a.k_sh | a.v_ld | a.v_sh | a.page_stride | a.head_stride;
  const bool vec = (a.D / 2) % ve == 0 && strides % ve == 0 && aligned16(a.k) && aligned16(a.v) &&
                   aligned16(a.k_pages) && aligned16(a.v_pages) &&
                   (a.Hq == 0 || ((a.q_ld | a.q_sh) % ve == 0 && aligned16(a.q) && aligned16(a.q_out)));
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  switch (a.dtype) {
    case TREAD_BF16: return launch<__nv_bfloat16>(a, vec, st);
    case TREAD_F16: return launch<__half>(a, vec, st);
    default: return launch<float>(a, vec, st);
  }
}
