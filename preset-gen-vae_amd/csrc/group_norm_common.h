// Shared by the GroupNorm + activation kernels (group_norm.hip, group_norm_f8.hip, group_norm_bwd.hip).
//
// GroupNorm + activation over x[N][P][C] (P pixels of an item, channels last), forward, backward and forward into 8-bit blocks:
//   mean, var over the P x C/G values of (item, group); xh = (x - mean) / sqrt(var + eps); u = gamma xh + beta; y = act(u)
//   du = gy act'(u); gbeta = sum du; ggamma = sum du xh; h = gamma du; gx = rstd (h - mean(h) - xh mean(h xh))
//
// Bound by memory.  A thread owns 8 neighbouring channels for the whole kernel (their gamma, beta, mean and rstd stay in
// registers) and walks over pixels: a row of C channels is C / 8 threads and 16 or 32 bytes each.  Two schemes:
//   fused     the pixels of one item and of a few whole groups fit in the registers of a workgroup: every value is read once,
//             mean and variance are two passes over registers (the variance of x - mean: nothing cancels), one launch.
//   two-pass  everything else: partial sums per slice of pixels, a second pass that reads the slices from their ends (what the
//             first pass read last is still in the last-level cache).  The slices' sums of x and x^2 are 64-bit ones: their
//             difference is the variance, and it may be far smaller than either.
#pragma once
#include "f8_common.h"

struct gn_args {
  int N, P, C, G, cg;
  int64_t total;        // values of x
  const void* x;
  const float* gamma;   // nullable
  const float* beta;    // nullable
  float eps, slope;
  int act;
  float* mean;          // [N][G]
  float* rstd;
  void* y;              // forward
  uint8_t* q;           // forward into 8-bit blocks: [N * P][Kp], scales [Kp / 128][N * P]
  float* scale;
  int Kp;
  const void* gy;       // backward
  void* gx;
  float* part;          // partial sums (see each kernel)
  int parts;            // two-pass forward: partial sums per (item, group) that the second pass adds up itself (0: finalised)
  int W, tpr, slices, colblocks;   // channels per workgroup, threads per row, pixel slices of an item, column blocks of a row
  uint32_t m_tpr, m_cg, m_per;   // fused kernels: magic numbers of tpr, cg and the pieces (or channels) of a group in a row
  int lg;                        // log2 of the lanes that add up one group
};

struct gn_plan {
  bool fused;
  int W, tpr, colblocks, lg;
  int nt, kv;      // fused: threads, pieces per thread
  int slices;      // two-pass
};

// the launches, one translation unit each (the kernels are many: type x alignment x group width x slab size)
int pgv_gn_forward(const gn_args& p, const gn_plan& pl, int dtype, bool vec, hipStream_t st);
int pgv_gn_forward_f8(const gn_args& p, const gn_plan& pl, int dtype, bool vec, int fmt, hipStream_t st);
int pgv_gn_backward(const gn_args& p, const gn_plan& pl, int dtype, bool vec, float* ggamma, float* gbeta, hipStream_t st);

namespace {

// first pixel of a slice
__device__ __forceinline__ int slice_at(const gn_args& p, int k) {
  const int each = p.P / p.slices, more = p.P - each * p.slices;
  return k * each + min(k, more);
}

// x / d for x d < 2^32: the workgroup's own indices
__device__ __forceinline__ int div_small(int x, int d, uint32_t magic) { return d == 1 ? x : (int)__umulhi((uint32_t)x, magic); }
static inline uint32_t magic_of(int64_t d) { return d <= 1 ? 0u : (uint32_t)(((1ull << 32) + d - 1) / d); }

// 1 / sqrt(v) within an ulp: the hardware's estimate and one Newton step
__device__ __forceinline__ float rsqrt_(float v) {
  if (v < 0x1p-100f) return 1.f / sqrtf(v);   // (the estimate takes a denormal for zero)
  const float y = __builtin_amdgcn_rsqf(v);
  return fmaf(y * 0.5f, fmaf(-v * y, y, 1.f), y);
}

__device__ __forceinline__ float sigmoid_(float u) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(u * -1.4426950408889634f));
}
__device__ __forceinline__ void act8(float (&u)[8], int act, float slope) {
  if (act == PGV_ACT_SILU) {
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] = u[i] * sigmoid_(u[i]);
  } else if (act == PGV_ACT_LEAKY_RELU) {
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] = u[i] > 0.f ? u[i] : slope * u[i];
  } else if (act == PGV_ACT_HARDTANH) {
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] = u[i] != u[i] ? u[i] : fminf(1.f, fmaxf(-1.f, u[i]));
  }
}
// g[i] *= act'(u[i])
__device__ __forceinline__ void act_grad8(float (&g)[8], const float (&u)[8], int act, float slope) {
  if (act == PGV_ACT_SILU) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float s = sigmoid_(u[i]);
      g[i] *= s * fmaf(u[i], 1.f - s, 1.f);
    }
  } else if (act == PGV_ACT_LEAKY_RELU) {
#pragma unroll
    for (int i = 0; i < 8; ++i) g[i] = u[i] > 0.f ? g[i] : slope * g[i];
  } else if (act == PGV_ACT_HARDTANH) {
#pragma unroll
    for (int i = 0; i < 8; ++i) g[i] = (u[i] > -1.f && u[i] < 1.f) ? g[i] : (u[i] != u[i] ? u[i] : 0.f);
  }
}

// 8 neighbouring values as they lie in memory: 16-bit types stay two to a register until they are used
template <typename T>
struct raw8 {
  static constexpr int WORDS = 2 * sizeof(T);
  uint32_t w[WORDS];
  __device__ __forceinline__ float operator[](int i) const {
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(w[i]);
    } else if constexpr (__is_same(T, __bf16)) {
      return __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
    } else {
      return (float)__builtin_bit_cast(_Float16, (uint16_t)(i & 1 ? w[i >> 1] >> 16 : w[i >> 1]));
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) w[i] = 0;
  }
  // the compiler forgets what it derived from the words: the widened values of one pass are not kept for the next
  __device__ __forceinline__ void forget() {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) asm volatile("" : "+v"(w[i]));
  }
};
// VEC: 16-byte pieces of a 16-byte aligned row.  Otherwise the row starts anywhere: whole pieces are the same loads at the
// alignment of a value (32 x 1000 x 1020 bfloat16 forward: 114 us value by value), and a piece that ends behind its row is read
// with the neighbours that follow it and cut, except at the end of the tensor.
template <bool VEC, typename T>
__device__ __forceinline__ raw8<T> load_raw(const T* __restrict__ p, int n, const T* end) {
  raw8<T> r;
  if constexpr (VEC) {
#pragma unroll
    for (int h = 0; h < r.WORDS / 4; ++h) {
      const i32x4 a = reinterpret_cast<const i32x4*>(p)[h];
#pragma unroll
      for (int i = 0; i < 4; ++i) r.w[4 * h + i] = (uint32_t)a[i];
    }
  } else if (p + 8 <= end) {
#pragma unroll
    for (int h = 0; h < r.WORDS / 4; ++h) {
      const i32x4 a = reinterpret_cast<const at_align<i32x4, (int)sizeof(T)>*>(p)[h].v;
#pragma unroll
      for (int i = 0; i < 4; ++i) r.w[4 * h + i] = (uint32_t)a[i];
    }
#pragma unroll
    for (int i = 0; i < r.WORDS; ++i) {
      if constexpr (sizeof(T) == 4)
        r.w[i] = i < n ? r.w[i] : 0u;
      else
        r.w[i] &= (2 * i < n ? 0xffffu : 0u) | (2 * i + 1 < n ? 0xffff0000u : 0u);
    }
  } else {
    r.clear();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i >= n) continue;
      if constexpr (sizeof(T) == 4)
        r.w[i] = __float_as_uint((float)p[i]);
      else
        r.w[i >> 1] |= (uint32_t)__builtin_bit_cast(uint16_t, p[i]) << (i & 1 ? 16 : 0);
    }
  }
  return r;
}
template <bool VEC, typename T>
__device__ __forceinline__ void store8(T* __restrict__ p, int n, const float (&v)[8]) {
  constexpr int AL = VEC ? 16 : sizeof(T);
  if (VEC || n == 8) {
    if constexpr (sizeof(T) == 4) {
      f32x4 a, b;
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = v[i], b[i] = v[4 + i];
      reinterpret_cast<at_align<f32x4, AL>*>(p)[0].v = a;
      reinterpret_cast<at_align<f32x4, AL>*>(p)[1].v = b;
    } else {
      typedef T t8 __attribute__((ext_vector_type(8)));
      t8 a;
#pragma unroll
      for (int i = 0; i < 8; ++i) a[i] = (T)v[i];
      reinterpret_cast<at_align<t8, AL>*>(p)->v = a;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = (T)v[i];
  }
}

// One thread's place: 8 channels from c, valid ones n (0: a pad column of the 8-bit rows or an idle thread), pixel phase r of rpp.
// SAME (C/G a multiple of 8): the 8 channels are of one group g[0], and mean, rstd and the like are one register each.
template <bool SAME>
struct place {
  static constexpr int A = SAME ? 1 : 8;
  int c, n, r, rpp;
  int g[A];   // groups of the channels within the item
};
// LOCAL: c0 is a whole number of groups, and g counts from the workgroup's first one
template <bool SAME, bool LOCAL = false>
__device__ __forceinline__ place<SAME> my_place(const gn_args& p, int c0, int nt) {
  place<SAME> q;
  const int row = div_small(threadIdx.x, p.tpr, p.m_tpr), j = threadIdx.x - row * p.tpr;
  q.rpp = div_small(nt, p.tpr, p.m_tpr);
  q.r = row;
  q.c = c0 + 8 * j;
  const int end = min(c0 + p.W, p.C);
  q.n = q.r < q.rpp ? max(0, min(8, end - q.c)) : 0;
#pragma unroll
  for (int i = 0; i < q.A; ++i) q.g[i] = i >= q.n ? 0 : LOCAL ? div_small(8 * j + i, p.cg, p.m_cg) : (q.c + i) / p.cg;
  return q;
}
// the per-channel vectors of a place; channels beyond the valid ones normalise to 0.  ar = gamma rstd: u = (x - mean) ar + beta
// is two operations, and subtracting the mean first loses nothing when it is far from zero.
template <bool SAME>
struct chan {
  float ga[8], be[8], mu[SAME ? 1 : 8], rs[SAME ? 1 : 8], ar[8];
};
template <bool VEC>
__device__ __forceinline__ void load8f(const float* __restrict__ v, int c, int n, float fill, float (&o)[8]) {
  if (v == nullptr) {   // (uniform)
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = i < n ? fill : 0.f;
  } else if constexpr (VEC) {
    f32x4 a = {0.f, 0.f, 0.f, 0.f}, b = a;
    if (n > 0) a = reinterpret_cast<const f32x4*>(v + c)[0], b = reinterpret_cast<const f32x4*>(v + c)[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = a[i], o[4 + i] = b[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = i < n ? v[c + i] : 0.f;
  }
}
template <bool VEC, bool SAME>
__device__ __forceinline__ void load_affine(const gn_args& p, const place<SAME>& q, chan<SAME>& k) {
  load8f<VEC>(p.gamma, q.c, q.n, 1.f, k.ga);
  load8f<VEC>(p.beta, q.c, q.n, 0.f, k.be);
#pragma unroll
  for (int i = 0; i < 8; ++i) k.ar[i] = k.ga[i] * k.rs[SAME ? 0 : i];
}
template <bool SAME>
__device__ __forceinline__ void load_stats(const gn_args& p, const place<SAME>& q, int item, int gfirst, chan<SAME>& k) {
#pragma unroll
  for (int i = 0; i < q.A; ++i) {
    const int64_t g = (int64_t)item * p.G + gfirst + q.g[i];
    k.mu[i] = i < q.n ? p.mean[g] : 0.f;
    k.rs[i] = i < q.n ? p.rstd[g] : 0.f;
  }
}

// Sums over the entries of every group: L neighbouring lanes per group (a power of two, at most 64), each over every L-th entry.
// at(g, e): entry e < cnt(g) of local group g; done(g, sum): called by one lane.
template <int NT, typename V, typename At, typename Cnt, typename Done>
__device__ __forceinline__ void sum_groups(int groups, int lg, At at, Cnt cnt, Done done) {
  const int L = 1 << lg, s = threadIdx.x & (L - 1), step = NT >> lg;
  for (int g0 = 0; g0 < groups; g0 += step) {
    const int g = g0 + (threadIdx.x >> lg);
    V v{};
    const int n = g < groups ? cnt(g) : 0;
    for (int e = s; e < n; e += L) v.add(at(g, e));
    for (int o = L >> 1; o > 0; o >>= 1) v.add(v.from(o));
    if (s == 0 && g < groups) done(g, v);
  }
}
static inline int lanes_log2(int64_t nt, int64_t groups) {
  int lg = 0;
  while (lg < 6 && (nt >> (lg + 1)) >= groups) ++lg;
  return lg;
}
struct sum1 {
  float a;
  __device__ __forceinline__ void add(const sum1& o) { a += o.a; }
  __device__ __forceinline__ sum1 from(int o) const {
    sum1 r;
    r.a = __shfl_xor(a, o, 64);
    return r;
  }
};
template <typename F>
struct sum2 {
  F a, b;
  __device__ __forceinline__ void add(const sum2& o) { a += o.a, b += o.b; }
  __device__ __forceinline__ sum2 from(int o) const {
    sum2 r;
    r.a = __shfl_xor(a, o, 64);
    r.b = __shfl_xor(b, o, 64);
    return r;
  }
};

constexpr int MAXG = 256;    // groups of a workgroup of the fused kernels
constexpr int MAXW = 2048;   // channels of a workgroup of the two-pass kernels: 8 for each of 256 threads

// levels of gn_param_grads_kernel: rows that one workgroup adds up
constexpr int ROWS = 1024;

inline void set_plan(gn_args& p, const gn_plan& pl, bool same) {
  p.W = pl.W;
  p.tpr = pl.tpr;
  p.slices = pl.slices;
  p.colblocks = pl.colblocks;
  p.lg = pl.lg;
  p.m_tpr = magic_of(pl.tpr);
  p.m_cg = magic_of(p.cg);
  p.m_per = magic_of(same ? p.cg / 8 : p.cg);
}

}  // namespace
