// Attention of one new token per sequence over a paged key-value cache (sm_100a).
//
//   out[b, h] = sum_t softmax_t(scale * q[b, h] . K[t, g]) V[t, g],   t < lens[b], g = h / (Hq / Hkv)
// where token t's keys and values lie in slot t % page_size of page table[b][t / page_size]. Where no
// key has a score above -inf, or there is none, the softmax has no value and the output is zero.
//
// Every key and value is read once: 4 D bytes a token and KV head in 16 bits, against 4 D G operations
// (G = Hq / Hkv query heads share them). At G = 7 that is 7 operations a byte, far below what the tensor
// cores need to be busy: the bound is HBM, and for few keys the latency of a launch.
//
// Split. The lengths are on the device, so the kernel itself deals out the work: all sequences' keys, per
// KV head in units of 16, form one line that is cut into equal shares, one per CTA, whatever the lengths.
// An item costs more than its units (its queries, the joining of the warps, the output): about kItemCost of
// them, which are counted in. A CTA's share covers parts of one or more items (sequence, KV head). Its warps
// take the units of the share in turn, each with a ring of units in flight in shared memory (cp.async, 16
// bytes a lane, rows swizzled so that eight rows' same chunk lie in eight banks), its own running maximum
// and sum, and its own accumulators. At an item's end the warps' states are joined in shared memory; an item
// that several CTAs share leaves its states in the workspace, where a second kernel joins them in the order of
// the shares (no atomics: the result does not depend on timing).
//
// 16-bit types run on mma.sync with keys as rows and the group's query heads as the 8 columns, so that a
// group of 7 fills 7 of 8 columns (heads as rows would fill 7 of 16): S^T = K Q^T, O^T = V^T P^T, and the
// heads of S^T's, P^T's and O^T's columns stay in the same lanes. P meets V as the sum of two numbers of the
// type, its rounding and what that left out: the weights keep 16 bits or more (in fp16 down to 2^-22 of the
// largest weight, see kRaise), and the output's own rounding is nearly all that is lost (rounded once, the weights
// add as much error again); 1 % of the time.
// fp32 runs on FMAs.
//
// Measured, of 6.54 TB/s: 64 sequences of 2400-16640 tokens (28 / 4 heads of 128, bf16) 155 us, 6.2 TB/s; 18 of up
// to 16640 (40 / 8 heads, fp16, pages of 16) 62 us, 5.9 TB/s; one of 8257 8.9 us, of which the two launches
// take 3.3; 256 of 1-700 (14 / 2 heads of 64) 12.5 us. For small shares what counts is how little code runs: the
// fetch is in one place, and the line is summed in 32 bits.
#include <type_traits>

#include "common.cuh"

namespace tread {
namespace {

constexpr int kUnit = 16;      // keys of one unit
constexpr int kMaxCtas = 384;  // shares at most
constexpr int kItemCost = 8;   // units that an item's fixed cost amounts to
constexpr int kMinShare = 4;   // a unit for every warp: more parts cost more to join
constexpr float kLog2e = 1.4426950408889634f;

// The running maximum may lag behind the scores by kSlack (a weight is at most 2^kSlack), and 16-bit weights are
// formed 2^kRaise times too large: sums and accumulators carry the same factor, the quotient drops it. bf16 reaches
// as far down as fp32. fp16 ends at 2^-24 and 2^16: raised as far as it goes, a weight's second part is off by at
// most 2^-25-13 = 2^-38 of the largest weight, so that keys 2^-27 below one key (an attention sink whose value is
// near zero) keep the 11 bits of the output; unraised, they were lost from 2^-14 on.
template <typename T>
constexpr float kSlack = std::is_same<T, __half>::value ? 2.f : 8.f;
template <typename T>
constexpr float kRaise = std::is_same<T, __half>::value ? 8192.f : 1.f;

struct DecodeArgs : tread_paged_attn_args {
  int G;
  float scale_log2;
  unsigned* err;
  // {parts, state of the first, b, g} of the items that the join has to look at: by item (b Hkv + g) where
  // there are no more of them than CTAs, else by the CTA in which an item starts that ends in another
  int4* desc;  // [kMaxCtas]
  float2* ml;   // [kMaxCtas][2][G] {maximum, sum} of the partial states
  float* part;  // [kMaxCtas][2][G][D]
};

__host__ __device__ __forceinline__ bool by_items(const DecodeArgs& a, int ctas) {
  return (long long)a.B * a.Hkv <= ctas;
}

__device__ __forceinline__ unsigned smem_addr(const void* p) {
  return static_cast<unsigned>(__cvta_generic_to_shared(p));
}

// 16 bytes, zeros where `read` is false
__device__ __forceinline__ void cp_async16(unsigned dst, const void* src, bool read) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(read ? 16 : 0) : "memory");
}

template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void ldmatrix_x4(unsigned (&r)[4], unsigned addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

__device__ __forceinline__ void ldmatrix_x4_trans(unsigned (&r)[4], unsigned addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

__device__ __forceinline__ unsigned transpose8x8(unsigned x) {
  unsigned y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const unsigned (&a)[4], const unsigned (&b)[2]) {
  if constexpr (sizeof(T) == 2 && std::is_same<T, __half>::value)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}

template <typename T>
__device__ __forceinline__ unsigned pack2(float lo, float hi) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const unsigned*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const unsigned*>(&h);
  }
}

// exp2(x - m) where m may still be -inf (no finite score so far): then x is -inf too, or a NaN to pass on
__device__ __forceinline__ float weight(float x, float m) { return exp2f(x - (m == -INFINITY ? 0.f : m)); }

// Place of element d of head h in a warp's accumulators: the four head pairs of a fragment's lanes lie in
// four groups of banks.
template <int D>
__device__ __forceinline__ int place_of(int h, int d) {
  return h * D + (d ^ (((h >> 1) & 3) << 3));
}

// Shared memory and launch shape of one instance. Two CTAs per SM where their rings fit beside each other, so that
// one joins while the other streams; 130 to 190 KB of units in flight per SM. For 16 heads of 128 on one KV head
// (16-bit) 60 sequences of up to 4000 tokens take 19.3 us, 23.1 with one CTA and three times the stages, 200 of
// 5-20 10.9 and 12.9; one of 8000 10.1 and 9.3. Longer keys fit twice with half the warps only. That pays where a
// unit is little work, with one head (fp32, 8/8 heads of 128, 200 of 5-20: 30 -> 19 us, long ones alike), and is
// slower at most lengths elsewhere (16/2 heads of 256, bf16, 150 of 20-500: 23.7 -> 27.0 us).
template <typename T, int D, int GP>
struct Shape {
  static constexpr int kRow = D * sizeof(T);               // bytes of one key
  static constexpr int kUnitBytes = 2 * kUnit * kRow;      // keys, then values
  static constexpr int kWarps = kUnitBytes > (GP == 1 ? 8192 : 16384) ? 2 : 4;
  static constexpr int kJoin = kWarps * GP * D * 4;        // the warps' accumulators at an item's end
  static constexpr int kQ = sizeof(T) == 4 ? GP * D * 4 + kWarps * kUnit * GP * 4 : 0;  // fp32: queries and weights
  static constexpr int kCtas = kWarps * kUnitBytes <= 32768 ? 2 : 1;
  static constexpr int kRoom = (kCtas == 2 ? 112 : 224) * 1024 - kJoin - kQ;
  static constexpr int kFit = kRoom / (kWarps * kUnitBytes);
  static constexpr int kStages = kFit > 6 ? 6 : kFit;
  static constexpr int kSmem = kStages * kWarps * kUnitBytes + kJoin + kQ;
  static_assert(kStages >= 2, "ring");
};

// One warp's state over 16-bit keys.
template <typename T, int D, int GP>
struct MmaState {
  static constexpr int NT = GP / 8;
  unsigned qf[NT][D / 16][2];
  float o[NT][D / 16][4];
  float m[NT][2], l[NT][2];  // of heads 8 nt + 2 (lane % 4) + {0, 1}; l: this lane's keys only

  __device__ void start(const DecodeArgs& a, int b, int g, void*, int, int lane) {
    const T* q = static_cast<const T*>(a.q) + b * a.q_ld + (long long)g * a.G * D;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int h = nt * 8 + (lane >> 2);
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        const unsigned* p = reinterpret_cast<const unsigned*>(q + h * D + ks * 16 + (lane & 3) * 2);
        qf[nt][ks][0] = h < a.G ? p[0] : 0u;
        qf[nt][ks][1] = h < a.G ? p[4] : 0u;
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) m[nt][i] = -INFINITY, l[nt][i] = 0.f;
#pragma unroll
      for (int mt = 0; mt < D / 16; ++mt)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[nt][mt][i] = 0.f;
    }
  }

  __device__ __forceinline__ void unit(const DecodeArgs& a, unsigned keys, unsigned values, unsigned live, void*,
                                       int, int lane) {
    constexpr int kRow = D * sizeof(T);
    float s[NT][2][4];  // two chains each, so that a product does not wait for the last one's sum
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[nt][0][i] = s[nt][1][i] = 0.f;
    {
      const int row = lane & 15;
      const unsigned base = keys + row * kRow;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        unsigned f[4];
        ldmatrix_x4(f, base + (((2 * ks + (lane >> 4)) ^ (row & 7)) << 4));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma16816<T>(s[nt][ks & 1], f, qf[nt][ks]);
      }
    }
    const bool live0 = (live >> (lane >> 2)) & 1, live1 = (live >> ((lane >> 2) + 8)) & 1;
    unsigned p[NT][2], rest[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = (s[nt][0][i] + s[nt][1][i]) * a.scale_log2;
      if (live != 0xffffu) {
        if (!live0) x[0] = x[1] = -INFINITY;
        if (!live1) x[2] = x[3] = -INFINITY;
      }
      float top[2] = {fmaxf(x[0], x[2]), fmaxf(x[1], x[3])};
      // the maximum moves only when a score leaves it behind by more than kSlack: rarely. The difference, since a
      // sum with a large maximum would be rounded; -inf and NaN compare false.
      if (__any_sync(0xffffffffu, top[0] - m[nt][0] > kSlack<T> || top[1] - m[nt][1] > kSlack<T>)) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
          for (int off = 4; off <= 16; off <<= 1) top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], off));
          const float next = fmaxf(m[nt][i], top[i]);
          const float alpha = weight(m[nt][i], next);
          m[nt][i] = next;
          l[nt][i] *= alpha;
#pragma unroll
          for (int mt = 0; mt < D / 16; ++mt) o[nt][mt][i] *= alpha, o[nt][mt][i + 2] *= alpha;
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = weight(x[i], m[nt][i & 1]) * kRaise<T>;
      l[nt][0] += x[0] + x[2];
      l[nt][1] += x[1] + x[3];
      p[nt][0] = transpose8x8(pack2<T>(x[0], x[1]));
      p[nt][1] = transpose8x8(pack2<T>(x[2], x[3]));
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] -= Num<T>::to_f(Num<T>::from_f(x[i]));
      rest[nt][0] = transpose8x8(pack2<T>(x[0], x[1]));
      rest[nt][1] = transpose8x8(pack2<T>(x[2], x[3]));
    }
    {
      const int row = (lane & 7) + ((lane >> 4) << 3);
      const unsigned base = values + row * kRow;
#pragma unroll
      for (int mt = 0; mt < D / 16; ++mt) {
        unsigned f[4];
        ldmatrix_x4_trans(f, base + (((2 * mt + ((lane >> 3) & 1)) ^ (row & 7)) << 4));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          mma16816<T>(o[nt][mt], f, p[nt]);
          mma16816<T>(o[nt][mt], f, rest[nt]);
        }
      }
    }
  }

  // the state into shared memory: accumulators [GP][D] (place_of), maxima and sums [GP]
  __device__ void leave(float* so, float2* sml, int lane) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float sum = l[nt][i];
#pragma unroll
        for (int off = 4; off <= 16; off <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        const int h = nt * 8 + (lane & 3) * 2 + i;
        if (lane < 4) sml[h] = make_float2(m[nt][i], sum);
#pragma unroll
        for (int mt = 0; mt < D / 16; ++mt) {
          so[place_of<D>(h, mt * 16 + (lane >> 2))] = o[nt][mt][i];
          so[place_of<D>(h, mt * 16 + (lane >> 2) + 8)] = o[nt][mt][i + 2];
        }
      }
    }
  }
};

// One warp's state over fp32 keys: scores with a half warp per half of D and a lane per key, then values
// with D / 32 elements a lane.
template <int D, int GP>
struct FmaState {
  static constexpr int kPer = D / 32;
  float o[GP][kPer], m[GP], l[GP];  // l: this lane's key only

  __device__ void start(const DecodeArgs& a, int b, int g, void* extra, int warp, int lane) {
    float* sq = static_cast<float*>(extra);
    const float* q = static_cast<const float*>(a.q) + b * a.q_ld + (long long)g * a.G * D;
    for (int i = threadIdx.x; i < GP * D; i += blockDim.x) sq[i] = i < a.G * D ? q[i] : 0.f;
#pragma unroll
    for (int h = 0; h < GP; ++h) {
      m[h] = -INFINITY, l[h] = 0.f;
#pragma unroll
      for (int e = 0; e < kPer; ++e) o[h][e] = 0.f;
    }
    __syncthreads();
  }

  __device__ __forceinline__ void unit(const DecodeArgs& a, unsigned keys, unsigned values, unsigned live, void* extra,
                                       int warp, int lane) {
    constexpr int kRow = D * 4;
    const float* sq = static_cast<const float*>(extra);
    float* sp = static_cast<float*>(extra) + GP * D + warp * kUnit * GP;  // [kUnit][GP]
    const int key = lane & 15, half = lane >> 4;
    float s[GP];
#pragma unroll
    for (int h = 0; h < GP; ++h) s[h] = 0.f;
#pragma unroll (GP < 8 ? 8 : 4)
    for (int i = 0; i < D / 8; ++i) {
      const int c = half * (D / 8) + i;
      float4 k;
      asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                   : "=f"(k.x), "=f"(k.y), "=f"(k.z), "=f"(k.w)
                   : "r"(keys + key * kRow + ((c ^ (key & 7)) << 4))
                   : "memory");
#pragma unroll
      for (int h = 0; h < GP; ++h) {
        const float4 q = *reinterpret_cast<const float4*>(sq + h * D + c * 4);
        s[h] = fmaf(k.x, q.x, s[h]);
        s[h] = fmaf(k.y, q.y, s[h]);
        s[h] = fmaf(k.z, q.z, s[h]);
        s[h] = fmaf(k.w, q.w, s[h]);
      }
    }
    const bool on = (live >> key) & 1;
    bool moved = false;
#pragma unroll
    for (int h = 0; h < GP; ++h) {
      s[h] = (s[h] + __shfl_xor_sync(0xffffffffu, s[h], 16)) * a.scale_log2;
      if (!on) s[h] = -INFINITY;
      moved |= s[h] - m[h] > kSlack<float>;
    }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int h = 0; h < GP; ++h) {
        float top = s[h];
#pragma unroll
        for (int off = 1; off <= 8; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
        const float next = fmaxf(m[h], top);
        const float alpha = weight(m[h], next);
        m[h] = next;
        l[h] *= alpha;
#pragma unroll
        for (int e = 0; e < kPer; ++e) o[h][e] *= alpha;
      }
    }
#pragma unroll
    for (int h = 0; h < GP; ++h) {
      s[h] = weight(s[h], m[h]);
      if (half == 0) {
        l[h] += s[h];
        sp[key * GP + h] = s[h];
      }
    }
    __syncwarp();
#pragma unroll (GP < 8 ? 8 : 4)
    for (int t = 0; t < kUnit; ++t) {
      float v[kPer];
      if constexpr (kPer == 2) {
        asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];"
                     : "=f"(v[0]), "=f"(v[1])
                     : "r"(values + t * kRow + (((lane >> 1) ^ (t & 7)) << 4) + (lane & 1) * 8)
                     : "memory");
      } else {
#pragma unroll
        for (int e = 0; e < kPer; e += 4)
          asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                       : "=f"(v[e]), "=f"(v[e + 1]), "=f"(v[e + 2]), "=f"(v[e + 3])
                       : "r"(values + t * kRow + (((lane + e * 8) ^ (t & 7)) << 4))
                       : "memory");
      }
#pragma unroll
      for (int h = 0; h < GP; ++h) {
        const float w = sp[t * GP + h];
#pragma unroll
        for (int e = 0; e < kPer; ++e) o[h][e] = fmaf(w, v[e], o[h][e]);
      }
    }
    __syncwarp();  // the weights are written again by the next unit
  }

  __device__ void leave(float* so, float2* sml, int lane) {
#pragma unroll
    for (int h = 0; h < GP; ++h) {
      float sum = l[h];
#pragma unroll
      for (int off = 16; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
      if (lane == 0) sml[h] = make_float2(m[h], sum);
#pragma unroll
      for (int e = 0; e < kPer; ++e)
        so[place_of<D>(h, kPer == 2 ? lane * 2 + e : (e / 4) * 128 + lane * 4 + e % 4)] = o[h][e];
    }
  }
};

template <typename T, int D, int GP>
struct StateOf {
  using type = MmaState<T, D, GP>;
};
template <int D, int GP>
struct StateOf<float, D, GP> {
  using type = FmaState<D, GP>;
};

// A sequence's length, 0 where it is out of range.
__device__ __forceinline__ int length_of(const DecodeArgs& a, int b) {
  const long long n = __ldg(reinterpret_cast<const long long*>(a.lens) + b);
  return n < 0 || n > (long long)a.max_pages * a.page_size ? 0 : (int)n;
}
__device__ __forceinline__ int units_of(int len) { return (len + kUnit - 1) / kUnit; }

// A place on the line of units: unit j of item (b, g), the item having n units of len tokens.
struct Place {
  int b, g, j, n, len;

  __device__ __forceinline__ void settle(const DecodeArgs& a) {  // j may lie behind the item's end
    while (j >= n) {
      j -= n;
      if (++g < a.Hkv) continue;
      g = 0;
      do {
        if (++b >= a.B) {
          n = 1 << 30, j = 0, b = a.B - 1, len = 0;  // the line's end: never loaded
          return;
        }
        len = length_of(a, b);
        n = units_of(len);
      } while (n == 0);
    }
  }
};

// The CTAs of an SM stand in the bounds even where they are one: without them the compiler saves registers for
// more, and fp32 takes up to twice as long (16/1 heads of 128, 60 sequences of up to 4000: 118 us, 59 with).
template <typename T, int D, int GP, bool WHOLE>  // WHOLE: a unit never crosses a page (page_size % 16 == 0)
__global__ void __launch_bounds__(Shape<T, D, GP>::kWarps * 32, Shape<T, D, GP>::kCtas)
    paged_attn_kernel(const __grid_constant__ DecodeArgs a) {
  using S = Shape<T, D, GP>;
  constexpr int W = S::kWarps, kThreads = W * 32, kStages = S::kStages;
  static_assert((W & (W - 1)) == 0, "the warps' turns");
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ unsigned s_live[W][kStages];
  __shared__ float2 s_ml[W][GP];
  __shared__ int2 s_scan[W];
  __shared__ int s_ends[2];
  __shared__ Place s_place;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float* s_o = reinterpret_cast<float*>(smem + kStages * W * S::kUnitBytes);
  void* extra = smem + kStages * W * S::kUnitBytes + S::kJoin;
  const unsigned ring = smem_addr(smem) + warp * (kStages * S::kUnitBytes);

  // the line: every thread adds up a run of sequences, a scan places the runs. An item's weight is its units and
  // kItemCost; units and weights are summed side by side (the caller has made sure that they fit).
  const int run = (a.B + kThreads - 1) / kThreads;
  const int b0 = min(a.B, (int)threadIdx.x * run), b1 = min(a.B, b0 + run);
  int units = 0, items = 0;
  for (int b = b0; b < b1; ++b) {
    const int len = length_of(a, b);
    units += units_of(len);
    items += len > 0;
    if (len == 0 && b % gridDim.x == blockIdx.x) {
      const long long n = __ldg(reinterpret_cast<const long long*>(a.lens) + b);
      if (n != 0 && a.err) atomicOr(a.err, 2u);
    }
  }
  int upto = units, upto_items = items;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, upto, off), y = __shfl_up_sync(0xffffffffu, upto_items, off);
    if (lane >= off) upto += x, upto_items += y;
  }
  if (lane == 31) s_scan[warp] = make_int2(upto, upto_items);
  __syncthreads();
  int before = upto - units, total = 0, before_items = upto_items - items, total_items = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    if (w < warp) before += s_scan[w].x, before_items += s_scan[w].y;
    total += s_scan[w].x, total_items += s_scan[w].y;
  }
  const int line = (total + kItemCost * total_items) * a.Hkv;
  const int share = max(kMinShare, (line + (int)gridDim.x - 1) / (int)gridDim.x);
  // the share's ends on the line of units alone, and the place of its first unit
  const int c0 = min(line, (int)blockIdx.x * share), c1 = min(line, c0 + share);
  const int run0 = (before + kItemCost * before_items) * a.Hkv, run1 = run0 + (units + kItemCost * items) * a.Hkv;
#pragma unroll 1
  for (int i = 0; i < 2; ++i) {
    const int cut = i == 0 ? c0 : c1;
    if (cut >= line) {
      if (threadIdx.x == 0) s_ends[i] = total * a.Hkv;
      continue;
    }
    if (cut < run0 || cut >= run1) continue;  // in another thread's run
    int at = run0, at_units = before * a.Hkv;
    for (int b = b0;; ++b) {
      const int len = length_of(a, b), n = units_of(len), weight = len > 0 ? n + kItemCost : 0;
      if (cut < at + weight * a.Hkv) {
        const int g = (cut - at) / weight, j = max(0, cut - at - g * weight - kItemCost);
        s_ends[i] = at_units + g * n + j;
        if (i == 0) s_place = Place{b, g, j, n, len};
        break;
      }
      at += weight * a.Hkv;
      at_units += n * a.Hkv;
    }
  }
  // sequences without a key: zeros
  const bool by_item = by_items(a, gridDim.x);
  for (int b = blockIdx.x; b < a.B; b += gridDim.x)
    if (length_of(a, b) == 0) {
      for (int i = threadIdx.x; i < a.Hq * D; i += kThreads)
        static_cast<T*>(a.out)[(long long)b * a.Hq * D + i] = Num<T>::from_f(0.f);
      if (by_item)
        for (int g = threadIdx.x; g < a.Hkv; g += kThreads) a.desc[b * a.Hkv + g] = make_int4(0, 0, 0, 0);
    }
  __syncthreads();
  const int u0 = s_ends[0], u1 = s_ends[1];
  if (u0 >= u1) {
    if (threadIdx.x == 0 && !by_item) a.desc[blockIdx.x] = make_int4(0, 0, 0, 0);
    return;
  }

  typename StateOf<T, D, GP>::type st;
  st.start(a, s_place.b, s_place.g, extra, warp, lane);  // the first item's queries are on their way

  // the warp's own walk along the share, kStages units ahead of what it computes; the pages' numbers are
  // read a unit further ahead
  Place load = s_place, next = load;
  load.j += warp;
  load.settle(a);
  next = load;
  next.j += W;
  next.settle(a);
  int load_at = u0 + warp;
  auto page_of = [&](const Place& p, int at) -> int {  // of the unit's first key, or of the lane's key
    const unsigned t = p.j * kUnit + (WHOLE ? 0 : lane & 15);
    return at < u1 && t < (unsigned)p.len ? __ldg(a.table + p.b * a.table_ld + t / (unsigned)a.page_size) : -1;
  };
  int id = page_of(load, load_at), next_id = page_of(next, load_at + W);
  auto fetch = [&](int stage) {
    if (load_at < u1) {
      constexpr int kChunks = S::kRow / 16, kIter = kUnit * kChunks / 32;
      const unsigned dst = ring + stage * S::kUnitBytes;
      const unsigned t0 = load.j * kUnit, t = t0 + (WHOLE ? 0 : lane & 15);
      const bool known = id >= 0 && id < a.num_pages;
      const unsigned slot = t - t / (unsigned)a.page_size * a.page_size;
      const long long off = known ? id * a.page_stride + load.g * a.head_stride + (long long)slot * D : 0;
      const int rows = min(kUnit, load.len - (int)t0);
      const char* kp = static_cast<const char*>(a.k_pages);
      const char* vp = static_cast<const char*>(a.v_pages);
      unsigned live = (1u << rows) - 1;
      if (WHOLE && known && rows == kUnit) {  // the common unit: 16 rows that follow each other
        kp += off * (int)sizeof(T) + lane * 16;
        vp += off * (int)sizeof(T) + lane * 16;
        constexpr int kRows = kChunks < 32 ? 32 / kChunks : 1;  // rows of one step of 512 bytes
        const unsigned to =
            dst + (kChunks < 32 ? lane / kChunks * S::kRow + (((lane % kChunks) ^ (lane / kChunks)) << 4) : lane << 4);
#pragma unroll
        for (int it = 0; it < kIter; ++it) {
          const int row = kChunks <= 32 ? it * kRows : it * 32 / kChunks;  // the step's first row
          const unsigned at = (to ^ ((row & 7) << 4)) + (kChunks <= 32 ? row * S::kRow : it * 512);
          cp_async16(at, kp + it * 512, true);
          cp_async16(at + kUnit * S::kRow, vp + it * 512, true);
        }
      } else {
        if (WHOLE) {
          if (!known) live = 0;
        } else {
          live &= __ballot_sync(0xffffffffu, known);  // lanes 16..31 repeat lanes 0..15
        }
        if (live != (1u << rows) - 1 && lane == 0 && a.err) atomicOr(a.err, 2u);
#pragma unroll 1
        for (int it = 0; it < kIter; ++it) {
          const int row = (it * 32 + lane) / kChunks, c = (it * 32 + lane) % kChunks;
          const long long start = WHOLE ? off + row * D : __shfl_sync(0xffffffffu, off, row);
          const long long from = start * (int)sizeof(T) + c * 16;
          const bool read = (live >> row) & 1;
          const unsigned to = dst + row * S::kRow + ((c ^ (row & 7)) << 4);
          cp_async16(to, kp + (read ? from : 0), read);  // rows that are not read are zero
          cp_async16(to + kUnit * S::kRow, vp + (read ? from : 0), read);
        }
      }
      if (lane == 0) s_live[warp][stage] = live;
      load_at += W;
      load = next;
      id = next_id;
      next.j += W;
      next.settle(a);
      next_id = page_of(next, load_at + W);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  Place at = s_place;
  int pos = u0;
  int step = 0;              // the warp's units so far, modulo the ring
  int slot = 0, owed = kStages;  // the ring's next slot to fill, and how many are free
  int4 open = make_int4(0, 0, 0, 0);
  while (pos < u1) {
    const int seg = min(at.n - at.j, u1 - pos);
    if (pos != u0) st.start(a, at.b, at.g, extra, warp, lane);
    // one more turn than there are units, for the slots that the last one (or nothing yet) has left free: the
    // code of a fetch is in one place, since a short share's time is mostly that of reading instructions
    for (int i = (warp - (pos - u0)) & (W - 1);; i += W) {
#pragma unroll 1
      for (; owed > 0; --owed) {
        fetch(slot);
        slot = slot + 1 == kStages ? 0 : slot + 1;
      }
      if (i >= seg) break;
      cp_async_wait<kStages - 1>();
      __syncwarp();
      const unsigned stage = ring + step * S::kUnitBytes;
      st.unit(a, stage, stage + kUnit * S::kRow, s_live[warp][step], extra, warp, lane);
      step = step + 1 == kStages ? 0 : step + 1;
      owed = 1;
      __syncwarp();  // every lane has read the unit before its place is filled again
    }
    // the item's end, or the share's: join the warps
    st.leave(s_o + warp * GP * D, s_ml[warp], lane);
    __syncthreads();
    const bool whole = seg == at.n;
    const long long p = (long long)blockIdx.x * 2 + (pos == u0 ? 0 : 1);
    for (int i = threadIdx.x; i < a.G * (D / 8); i += kThreads) {  // eight elements of a head
      const int h = i / (D / 8), d = i % (D / 8) * 8;
      float top = -INFINITY, sum = 0.f, x[8] = {};
#pragma unroll
      for (int w = 0; w < W; ++w) top = fmaxf(top, s_ml[w][h].x);
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float f = weight(s_ml[w][h].x, top);
        const float4* o = reinterpret_cast<const float4*>(s_o + w * GP * D + place_of<D>(h, d));
        const float4 y = o[0], z = o[1];
        sum += f * s_ml[w][h].y;
        x[0] += f * y.x, x[1] += f * y.y, x[2] += f * y.z, x[3] += f * y.w;
        x[4] += f * z.x, x[5] += f * z.y, x[6] += f * z.z, x[7] += f * z.w;
      }
      if (whole) {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        T* to = static_cast<T*>(a.out) + ((long long)at.b * a.Hq + at.g * a.G + h) * D + d;
        constexpr int E = 16 / sizeof(T);
#pragma unroll
        for (int k = 0; k < 8; k += E) {
          Vec16<T> v;
#pragma unroll
          for (int e = 0; e < E; ++e) v.e[e] = Num<T>::from_f(x[k + e] * inv);
          *reinterpret_cast<int4*>(to + k) = v.raw;
        }
      } else {
        float4* to = reinterpret_cast<float4*>(a.part + (p * a.G + h) * D + d);
        to[0] = make_float4(x[0], x[1], x[2], x[3]);
        to[1] = make_float4(x[4], x[5], x[6], x[7]);
        if (d == 0) a.ml[p * a.G + h] = make_float2(top, sum);
      }
    }
    if (!whole && at.j == 0)  // starts here, ends in the CTA of its last unit
      open = make_int4((c1 + at.n - seg - 1) / share - (int)blockIdx.x + 1, (int)p, at.b, at.g);
    if (by_item && at.j == 0 && threadIdx.x == 0)
      a.desc[at.b * a.Hkv + at.g] = whole ? make_int4(0, 0, 0, 0) : open;
    pos += seg;
    at.j += seg;
    if (pos < u1) at.settle(a);
    __syncthreads();
  }
  cp_async_wait<0>();
  if (threadIdx.x == 0 && !by_item) a.desc[blockIdx.x] = open;
}

// Items whose keys several CTAs share: CTA (i, h) joins head h of the item that desc[i] names. All parts' maxima and sums are read at once and turned into weights; the warps then take
// the accumulators in turn, kAhead loads in flight each.
constexpr int kJoinWarps = 8;

template <typename T, int D>
__global__ void __launch_bounds__(kJoinWarps * 32) paged_attn_join_kernel(const __grid_constant__ DecodeArgs a) {
  constexpr int kPer = D / 32, kAhead = 8, kThreads = kJoinWarps * 32;
  __shared__ float s_o[kJoinWarps][D], s_m[kJoinWarps], s_l[kJoinWarps], s_f[kMaxCtas];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 open = a.desc[blockIdx.x];
  if (open.x == 0) return;
  const int h = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // the first part is in either of its CTA's slots, the others in their CTAs' first
  auto state = [&](int i) { return (long long)(i == 0 ? open.y : (open.y / 2 + i) * 2) * a.G + h; };
  float o[kPer] = {};
  float2 ml[(kMaxCtas + kThreads - 1) / kThreads];
  float top = -INFINITY, sum = 0.f;
#pragma unroll
  for (int k = 0; k < (kMaxCtas + kThreads - 1) / kThreads; ++k) {
    const int i = threadIdx.x + k * kThreads;
    ml[k] = i < open.x ? a.ml[state(i)] : make_float2(-INFINITY, 0.f);
    top = fmaxf(top, ml[k].x);
  }
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
  if (lane == 0) s_m[warp] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kJoinWarps; ++w) top = fmaxf(top, s_m[w]);
#pragma unroll
  for (int k = 0; k < (kMaxCtas + kThreads - 1) / kThreads; ++k) {
    const int i = threadIdx.x + k * kThreads;
    if (i >= open.x) continue;
    s_f[i] = weight(ml[k].x, top);
    sum += s_f[i] * ml[k].y;
  }
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
  if (lane == 0) s_l[warp] = sum;
  __syncthreads();
  for (int i0 = warp; i0 < open.x; i0 += kJoinWarps * kAhead) {
    float x[kAhead][kPer];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int i = i0 + k * kJoinWarps;
      if (i >= open.x) break;
      const float* from = a.part + state(i) * D + lane * kPer;
      if constexpr (kPer == 2) {
        *reinterpret_cast<float2*>(x[k]) = *reinterpret_cast<const float2*>(from);
      } else {
#pragma unroll
        for (int e = 0; e < kPer; e += 4)
          *reinterpret_cast<float4*>(x[k] + e) = *reinterpret_cast<const float4*>(from + e);
      }
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int i = i0 + k * kJoinWarps;
      if (i >= open.x) break;
#pragma unroll
      for (int e = 0; e < kPer; ++e) o[e] = fmaf(s_f[i], x[k][e], o[e]);
    }
  }
#pragma unroll
  for (int e = 0; e < kPer; ++e) s_o[warp][lane * kPer + e] = o[e];
  __syncthreads();
  float all = 0.f;
#pragma unroll
  for (int w = 0; w < kJoinWarps; ++w) all += s_l[w];
  const float inv = all == 0.f ? 0.f : 1.f / all;
  T* to = static_cast<T*>(a.out) + ((long long)open.z * a.Hq + open.w * a.G + h) * D;
  for (int d = threadIdx.x; d < D; d += kThreads) {
    float x = 0.f;
#pragma unroll
    for (int w = 0; w < kJoinWarps; ++w) x += s_o[w][d];
    to[d] = Num<T>::from_f(x * inv);
  }
}

template <typename T, int D, int GP>
int launch(const DecodeArgs& a, int sms, cudaStream_t st) {
  using S = Shape<T, D, GP>;
  auto kern = a.page_size % kUnit == 0 ? paged_attn_kernel<T, D, GP, true> : paged_attn_kernel<T, D, GP, false>;
  TREAD_CHECK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem));
  int ctas = sms * S::kCtas;
  if (ctas > kMaxCtas) ctas = kMaxCtas;
  kern<<<ctas, S::kWarps * 32, S::kSmem, st>>>(a);
  TREAD_CHECK_LAUNCH("paged_attn_kernel");
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(by_items(a, ctas) ? a.B * a.Hkv : ctas, a.G);
  cfg.blockDim = dim3(kJoinWarps * 32);
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  TREAD_CHECK_CUDA(cudaLaunchKernelEx(&cfg, paged_attn_join_kernel<T, D>, a));
  return TREAD_OK;
}

template <typename T, int GP>
int launch_width(int D, const DecodeArgs& a, int sms, cudaStream_t st) {
  switch (D) {
    case 64: return launch<T, 64, GP>(a, sms, st);
    case 128: return launch<T, 128, GP>(a, sms, st);
    default: return launch<T, 256, GP>(a, sms, st);
  }
}

template <typename T>
int dispatch(int D, const DecodeArgs& a, int sms, cudaStream_t st) {
  // On FMAs a head that is not there costs as much as others, so fp32 has narrower instances too. 32 sequences of
  // 2000 tokens, D = 128, when these were made: 16/8 heads 145 us with eight wide, 107 us with four; 8/8 heads 145
  // and 87 us with one.
  // (A column of the tensor cores' tiles costs nothing; eight is their width.)
  if constexpr (sizeof(T) == 4) {
    if (a.G == 1) return launch_width<T, 1>(D, a, sms, st);
    if (a.G <= 4) return launch_width<T, 4>(D, a, sms, st);
  }
  return a.G <= 8 ? launch_width<T, 8>(D, a, sms, st) : launch_width<T, 16>(D, a, sms, st);
}

size_t align256(size_t n) { return (n + 255) & ~size_t(255); }

}  // namespace
}  // namespace tread

extern "C" size_t tread_paged_attn_workspace_bytes(int Hq, int Hkv, int D) {
  using namespace tread;
  if (Hq <= 0 || Hkv <= 0 || D <= 0 || Hq / Hkv > 16 || D > 256) return 0;
  const size_t states = (size_t)kMaxCtas * 2 * (Hq / Hkv);
  return align256(kMaxCtas * sizeof(int4)) + align256(states * sizeof(float2)) + states * D * sizeof(float);
}

extern "C" int tread_paged_attn(const tread_paged_attn_args* args, tread_stream_t stream) {
  using namespace tread;
  TREAD_CHECK_ARG(args, "paged_attn: null arguments");
  DecodeArgs a;
  static_cast<tread_paged_attn_args&>(a) = *args;
  TREAD_CHECK_ARG(a.B >= 0, "paged_attn: B < 0");
  if (a.B == 0) return TREAD_OK;
  TREAD_CHECK_ARG(a.q && a.k_pages && a.v_pages && a.lens && a.out, "paged_attn: null pointer");
  TREAD_CHECK_ARG(a.Hq > 0 && a.Hkv > 0 && a.Hkv <= 65535 && a.Hq % a.Hkv == 0 && a.Hq / a.Hkv <= 16,
                  "paged_attn: bad heads Hq=%d Hkv=%d", a.Hq, a.Hkv);
  TREAD_CHECK_ARG(a.D == 64 || a.D == 128 || a.D == 256, "paged_attn: head_dim %d not in {64,128,256}", a.D);
  const int64_t es = (int64_t)dtype_size(a.dtype);
  TREAD_CHECK_ARG(es != 0, "paged_attn: unknown dtype %d", a.dtype);
  TREAD_CHECK_ARG(a.page_size > 0 && a.num_pages >= 0 && a.num_pages <= INT32_MAX &&
                      (a.num_pages <= 1 || a.page_stride >= (int64_t)a.page_size * a.D) &&
                      (a.Hkv == 1 || a.head_stride >= (int64_t)a.page_size * a.D),
                  "paged_attn: bad page geometry");
  TREAD_CHECK_ARG(a.max_pages >= 0 && (a.table || a.max_pages == 0) && (a.B <= 1 || a.table_ld == 0 || a.table_ld >= a.max_pages),
                  "paged_attn: bad page table");
  TREAD_CHECK_ARG((int64_t)a.max_pages * a.page_size <= INT32_MAX - kUnit,
                  "paged_attn: a sequence of 2^31 tokens or more");
  TREAD_CHECK_ARG(((int64_t)a.max_pages * a.page_size / kUnit + 1 + kItemCost) * a.Hkv <= (1 << 30) / a.B,
                  "paged_attn: a table of more than 2^34 tokens, counted by KV head");
  // the stride of a dimension of one is any number
  if (a.B == 1) a.q_ld = 0;
  if (a.num_pages <= 1) a.page_stride = 0;
  if (a.Hkv == 1) a.head_stride = 0;
  TREAD_CHECK_ARG(aligned16(a.q) && aligned16(a.k_pages) && aligned16(a.v_pages) && aligned16(a.out) &&
                      ((a.q_ld | a.page_stride | a.head_stride) * es) % 16 == 0,
                  "paged_attn: q, out and pages must lie on 16-byte boundaries");
  TREAD_CHECK_ARG(a.workspace && (reinterpret_cast<uintptr_t>(a.workspace) & 255u) == 0 &&
                      a.workspace_bytes >= (int64_t)tread_paged_attn_workspace_bytes(a.Hq, a.Hkv, a.D),
                  "paged_attn: workspace too small or not 256-byte aligned");
  int device = 0, sms = 0;
  TREAD_CHECK_CUDA(cudaGetDevice(&device));
  TREAD_CHECK_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device));
  a.G = a.Hq / a.Hkv;
  a.scale_log2 = a.sm_scale * kLog2e;
  a.err = static_cast<unsigned*>(a.err_flag);
  char* ws = static_cast<char*>(a.workspace);
  a.desc = reinterpret_cast<int4*>(ws);
  ws += align256(kMaxCtas * sizeof(int4));
  a.ml = reinterpret_cast<float2*>(ws);
  ws += align256((size_t)kMaxCtas * 2 * a.G * sizeof(float2));
  a.part = reinterpret_cast<float*>(ws);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  switch (a.dtype) {
    case TREAD_BF16: return dispatch<__nv_bfloat16>(a.D, a, sms, st);
    case TREAD_F16: return dispatch<__half>(a.D, a, sms, st);
    default: return dispatch<float>(a.D, a, sms, st);
  }
}
