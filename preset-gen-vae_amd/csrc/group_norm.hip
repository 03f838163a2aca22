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
#include "f8_common.h"

namespace {

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

// y (or its 8-bit block) of one pixel
template <bool VEC, bool Q, int FMT, bool SAME, typename T>
__device__ __forceinline__ void put(const gn_args& p, const place<SAME>& q, const chan<SAME>& k, int64_t pix, const raw8<T>& x) {
  float u[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) u[i] = fmaf(x[i] - k.mu[SAME ? 0 : i], k.ar[i], k.be[i]);
  act8(u, p.act, p.slope);
  if constexpr (!Q) {
    store8<VEC>((T*)p.y + pix * p.C + q.c, q.n, u);
  } else {   // 16 lanes side by side hold a block of 128 channels (tpr is a multiple of 16)
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, f8_abs_bits(u[i]));
    m = f8_max16(m);
    float s, inv;
    f8_scale<FMT>(m, s, inv);
    i32x2 o;
    o.x = f8_pack4<FMT>(u[0] * inv, u[1] * inv, u[2] * inv, u[3] * inv);
    o.y = f8_pack4<FMT>(u[4] * inv, u[5] * inv, u[6] * inv, u[7] * inv);
    *reinterpret_cast<i32x2*>(p.q + pix * p.Kp + q.c) = o;
    if ((threadIdx.x & 15) == 0) p.scale[(int64_t)(q.c / F8B) * p.N * p.P + pix] = s;
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

// ---- forward, fused: a workgroup per item and column block of W channels -----------------------------------------------------------
// A thread holds KV pieces in registers and KL more in LDS (16 bytes each: 16-bit types only).
template <typename T, int NT, int KV, int KL, bool VEC, bool Q, int FMT, bool SAME>
__global__ __launch_bounds__(NT) void gn_fwd_fused_kernel(gn_args p) {
  constexpr int A = SAME ? 1 : 8;
  extern __shared__ __attribute__((aligned(16))) i32x4 held[];   // [KL][NT]
  __shared__ __attribute__((aligned(16))) float val[NT * A];
  __shared__ float gs[2][MAXG];
  const int tid = threadIdx.x, item = blockIdx.x / p.colblocks, cb = blockIdx.x - item * p.colblocks, c0 = cb * p.W;
  const place<SAME> q = my_place<SAME, true>(p, c0, NT);
  const int gfirst = cb * (p.W / p.cg), groups = min(p.W / p.cg, p.G - gfirst);
  const T* xend = (const T*)p.x + p.total;
  const T* x = (const T*)p.x + (int64_t)item * p.P * p.C;   // (the item's bytes are addressed with 32 bits: make_gn_plan)
  const uint32_t at0 = (uint32_t)(q.r * p.C + q.c), step = (uint32_t)(q.rpp * p.C);
  auto get = [&](int k) {
    raw8<T> d;
    if (q.r + k * q.rpp < p.P && q.n > 0)
      d = load_raw<VEC>(x + (at0 + k * step), q.n, xend);
    else
      d.clear();
    return d;
  };
  if constexpr (KL > 0) {
#pragma unroll
    for (int h = 0; h < KL; h += 4) {
      raw8<T> e[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) e[k] = get(KV + h + k);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        held[(h + k) * NT + tid] = i32x4{(int)e[k].w[0], (int)e[k].w[1], (int)e[k].w[2], (int)e[k].w[3]};
    }
  }
  raw8<T> d[KV];
#pragma unroll
  for (int k = 0; k < KV; ++k) d[k] = get(k);
  auto from_lds = [&](int k) {   // (a thread reads what it wrote: no barrier)
    const i32x4 v = held[k * NT + tid];
    raw8<T> e;
#pragma unroll
    for (int i = 0; i < 4; ++i) e.w[i] = (uint32_t)v[i];
    return e;
  };
  chan<SAME> ch;
  const float inv_n = 1.f / ((float)p.P * (float)p.cg);
  const int per = SAME ? p.cg >> 3 : p.cg, pitch = SAME ? p.tpr : p.tpr * 8;
  // pass 0: mean; pass 1: variance
#pragma unroll
  for (int i = 0; i < A; ++i) ch.mu[i] = 0.f;
#pragma unroll
  for (int pass = 0; pass < 2; ++pass) {
#pragma unroll
    for (int k = 0; k < KV; ++k) d[k].forget();
    float s[A];
#pragma unroll
    for (int i = 0; i < A; ++i) s[i] = 0.f;
    auto take = [&](const raw8<T>& e) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float v = e[i] - ch.mu[SAME ? 0 : i];
        if (pass)
          s[SAME ? 0 : i] = fmaf(v, v, s[SAME ? 0 : i]);
        else
          s[SAME ? 0 : i] += v;
      }
    };
#pragma unroll
    for (int k = 0; k < KV; ++k)
      if (q.r + k * q.rpp < p.P) take(d[k]);
    if constexpr (KL > 0)
#pragma unroll 2
      for (int k = 0; k < KL; ++k)
        if (q.r + (KV + k) * q.rpp < p.P) take(from_lds(k));
    if (pass) __syncthreads();   // the readers of val of pass 0 are done
#pragma unroll
    for (int i = 0; i < A; ++i) val[tid * A + i] = i < q.n ? s[i] : 0.f;
    __syncthreads();
    sum_groups<NT, sum1>(groups, p.lg,
        [&](int g, int e) {
          const int r = div_small(e, per, p.m_per);
          sum1 v;
          v.a = val[r * pitch + g * per + (e - r * per)];
          return v;
        },
        [&](int) { return q.rpp * per; },
        [&](int g, const sum1& v) {
          const float m = pass ? rsqrt_(v.a * inv_n + p.eps) : v.a * inv_n;
          gs[pass][g] = m;
          if (p.mean) (pass ? p.rstd : p.mean)[(int64_t)item * p.G + gfirst + g] = m;
        });
    __syncthreads();
#pragma unroll
    for (int i = 0; i < A; ++i) (pass ? ch.rs : ch.mu)[i] = i < q.n ? gs[pass][q.g[i]] : 0.f;
  }
  if (q.r >= q.rpp) return;
  load_affine<VEC>(p, q, ch);
#pragma unroll
  for (int k = 0; k < KV; ++k) {
    const int r = q.r + k * q.rpp;
    d[k].forget();
    if (r < p.P && (Q || q.n > 0)) put<VEC, Q, FMT>(p, q, ch, (int64_t)item * p.P + r, d[k]);
  }
  if constexpr (KL > 0)
#pragma unroll 1
    for (int k = 0; k < KL; ++k) {
      const int r = q.r + (KV + k) * q.rpp;
      if (r < p.P && (Q || q.n > 0)) put<VEC, Q, FMT>(p, q, ch, (int64_t)item * p.P + r, from_lds(k));
    }
}

// ---- forward, two-pass --------------------------------------------------------------------------------------------------
// partial sums: part (as sum2<double>) [N][column blocks * slices][G] of (sum, sum of squares), zero for groups outside the block
template <typename T, bool VEC, bool SAME>
__global__ __launch_bounds__(256) void gn_stats_kernel(gn_args p) {
  constexpr int A = SAME ? 1 : 8;
  __shared__ sum2<double> val[256 * A];
  const int tid = threadIdx.x, item = blockIdx.x / p.slices, slice = blockIdx.x - item * p.slices, c0 = blockIdx.y * p.W;
  const place<SAME> q = my_place<SAME>(p, c0, 256);
  const int r0 = slice_at(p, slice), r1 = slice_at(p, slice + 1);
  const T* xend = (const T*)p.x + p.total;
  const T* x = (const T*)p.x + (int64_t)item * p.P * p.C + q.c;
  sum2<double> s[A]{};
  auto take = [&](const raw8<T>& d) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const double v = (double)d[i];
      s[SAME ? 0 : i].a += v;
      s[SAME ? 0 : i].b = fma(v, v, s[SAME ? 0 : i].b);
    }
  };
  if (q.n > 0) {
    int r = r0 + q.r;
    for (; r + 3 * q.rpp < r1; r += 4 * q.rpp) {
      raw8<T> d[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) d[k] = load_raw<VEC>(x + (int64_t)(r + k * q.rpp) * p.C, q.n, xend);
#pragma unroll
      for (int k = 0; k < 4; ++k) take(d[k]);
    }
    for (; r < r1; r += q.rpp) take(load_raw<VEC>(x + (int64_t)r * p.C, q.n, xend));
  }
#pragma unroll
  for (int i = 0; i < A; ++i) val[tid * A + i] = s[i];
  __syncthreads();
  sum2<double>* out = (sum2<double>*)p.part + ((int64_t)item * (p.slices * gridDim.y) + (int64_t)blockIdx.y * p.slices + slice) * p.G;
  const int cend = min(c0 + p.W, p.C), pitch = SAME ? p.tpr : p.tpr * 8;
  sum_groups<256, sum2<double>>(p.G, p.lg,
      [&](int g, int e) {
        const int lo = max(g * p.cg, c0), w = (min((g + 1) * p.cg, cend) - lo) / (SAME ? 8 : 1), r = e / w;
        return val[r * pitch + (lo - c0) / (SAME ? 8 : 1) + (e - r * w)];
      },
      [&](int g) { return q.rpp * (max(0, min((g + 1) * p.cg, cend) - max(g * p.cg, c0)) / (SAME ? 8 : 1)); },
      [&](int g, const sum2<double>& v) { out[g] = v; });
}

__device__ __forceinline__ void finalize(const gn_args& p, const sum2<double>& v, float& mean, float& rstd) {
  const double n = (double)p.P * (double)p.cg, m = v.a / n, var = v.b / n - m * m;
  mean = (float)m;
  rstd = (float)(1.0 / sqrt((var > 0.0 || var != var ? var : 0.0) + (double)p.eps));
}
__global__ __launch_bounds__(64) void gn_finalize_kernel(gn_args p, int parts) {
  const int item = blockIdx.x / p.G, g = blockIdx.x - item * p.G, lane = threadIdx.x;
  const sum2<double>* in = (const sum2<double>*)p.part + (int64_t)item * parts * p.G + g;
  sum2<double> v{};
  for (int e = lane; e < parts; e += 64) v.add(in[(int64_t)e * p.G]);
  v.a = pgv_wave_sum_d(v.a);
  v.b = pgv_wave_sum_d(v.b);
  const int64_t o = (int64_t)item * p.G + g;
  if (lane == 0) finalize(p, v, p.mean[o], p.rstd[o]);
}

template <typename T, bool VEC, bool Q, int FMT, bool SAME>
__global__ __launch_bounds__(256) void gn_apply_kernel(gn_args p) {
  __shared__ float gs[2][MAXW + 2];
  const int item = blockIdx.x / p.slices, slice = blockIdx.x - item * p.slices, c0 = blockIdx.y * p.W;
  const place<SAME> q = my_place<SAME>(p, c0, 256);
  const int gfirst = c0 / p.cg;
  if (p.parts) {   // (uniform) few partial sums: every workgroup adds up those of its groups
    const int groups = (min(c0 + p.W, p.C) - 1) / p.cg - gfirst + 1;
    const sum2<double>* in = (const sum2<double>*)p.part + (int64_t)item * p.parts * p.G + gfirst;
    sum_groups<256, sum2<double>>(groups, p.lg, [&](int g, int e) { return in[(int64_t)e * p.G + g]; }, [&](int) { return p.parts; },
        [&](int g, const sum2<double>& v) {
          finalize(p, v, gs[0][g], gs[1][g]);
          if (slice == 0) {   // (two blocks that share a group write the same values)
            p.mean[(int64_t)item * p.G + gfirst + g] = gs[0][g];
            p.rstd[(int64_t)item * p.G + gfirst + g] = gs[1][g];
          }
        });
    __syncthreads();
  }
  if (q.r >= q.rpp || (!Q && q.n == 0)) return;
  const int r0 = slice_at(p, slice), r1 = slice_at(p, slice + 1);
  const T* xend = (const T*)p.x + p.total;
  const T* x = (const T*)p.x + (int64_t)item * p.P * p.C + q.c;
  chan<SAME> ch;
  if (p.parts) {
#pragma unroll
    for (int i = 0; i < q.A; ++i) {
      ch.mu[i] = i < q.n ? gs[0][q.g[i] - gfirst] : 0.f;
      ch.rs[i] = i < q.n ? gs[1][q.g[i] - gfirst] : 0.f;
    }
  } else {
    load_stats(p, q, item, 0, ch);
  }
  load_affine<VEC>(p, q, ch);
  // (downwards: the end of a slice, which the pass before read last, is still in the last-level cache)
  const int top = r0 + r1 - 1;
  auto get = [&](int r) {
    raw8<T> d;
    if (!Q || q.n > 0)
      d = load_raw<VEC>(x + (int64_t)(top - r) * p.C, q.n, xend);
    else
      d.clear();
    return d;
  };
  int r = r0 + q.r;
  for (; r + 3 * q.rpp < r1; r += 4 * q.rpp) {
    raw8<T> d[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) d[k] = get(r + k * q.rpp);
#pragma unroll
    for (int k = 0; k < 4; ++k) put<VEC, Q, FMT>(p, q, ch, (int64_t)item * p.P + top - r - k * q.rpp, d[k]);
  }
  for (; r < r1; r += q.rpp) put<VEC, Q, FMT>(p, q, ch, (int64_t)item * p.P + top - r, get(r));
}

// ---- backward -----------------------------------------------------------------------------------------------------------
// xh and du of 8 values
template <bool SAME, typename T>
__device__ __forceinline__ void grads8(const gn_args& p, const chan<SAME>& k, const raw8<T>& x, const raw8<T>& gy, float (&xh)[8],
                                       float (&du)[8]) {
  float u[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float v = x[i] - k.mu[SAME ? 0 : i];
    xh[i] = v * k.rs[SAME ? 0 : i];
    u[i] = fmaf(v, k.ar[i], k.be[i]);
    du[i] = gy[i];
  }
  act_grad8(du, u, p.act, p.slope);
}
template <bool VEC, bool SAME, typename T>
__device__ __forceinline__ void put_gx(const gn_args& p, const place<SAME>& q, const chan<SAME>& k, const float (&c1)[SAME ? 1 : 8],
                                       const float (&c2)[SAME ? 1 : 8], int64_t pix, const raw8<T>& x, const raw8<T>& gy) {
  float xh[8], du[8], o[8];
  grads8(p, k, x, gy, xh, du);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int h = SAME ? 0 : i;
    o[i] = k.rs[h] * (fmaf(k.ga[i], du[i], -c1[h]) - xh[i] * c2[h]);
  }
  store8<VEC>((T*)p.gx + pix * p.C + q.c, q.n, o);
}

// Per-channel sums over the pixel phases of a workgroup, a = sum du and b = sum du xh, into tot[2][width]: the threads' values
// go to val[2][NT * 8], every thread adds a share of the rows of one channel, the shares (in place) are added last.
template <int NT>
__device__ __forceinline__ void channel_sums(const gn_args& p, int n, int rpp, const float (&a)[8], const float (&b)[8], float* val,
                                             float* tot, int width) {
  f32x4* v = reinterpret_cast<f32x4*>(val + threadIdx.x * 8);
  f32x4* w = reinterpret_cast<f32x4*>(val + NT * 8 + threadIdx.x * 8);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    f32x4 ta, tb;
#pragma unroll
    for (int i = 0; i < 4; ++i) ta[i] = 4 * h + i < n ? a[4 * h + i] : 0.f, tb[i] = 4 * h + i < n ? b[4 * h + i] : 0.f;
    v[h] = ta;
    w[h] = tb;
  }
  __syncthreads();
  const int shares = max(1, NT / width), pitch = p.tpr * 8;
  if (shares == 1) {
    for (int c = threadIdx.x; c < width; c += NT) {
      float s = 0.f, t = 0.f;
      for (int r = 0; r < rpp; ++r) s += val[r * pitch + c], t += val[NT * 8 + r * pitch + c];
      tot[c] = s;
      tot[width + c] = t;
    }
  } else {
    const int sh = threadIdx.x / width, c = threadIdx.x - sh * width;
    float s = 0.f, t = 0.f;
    if (sh < shares)
      for (int r = sh; r < rpp; r += shares) s += val[r * pitch + c], t += val[NT * 8 + r * pitch + c];
    __syncthreads();
    if (sh < shares) val[sh * width + c] = s, val[NT * 8 + sh * width + c] = t;
    __syncthreads();
    if (threadIdx.x < 2 * width && 2 * width <= NT) {   // both sums at once where the threads suffice
      const int k = threadIdx.x / width, cc = threadIdx.x - k * width;
      float u = 0.f;
      for (int i = 0; i < shares; ++i) u += val[k * NT * 8 + i * width + cc];
      tot[threadIdx.x] = u;
    } else if (2 * width > NT && threadIdx.x < width) {
      float u = 0.f, y = 0.f;
      for (int i = 0; i < shares; ++i) u += val[i * width + threadIdx.x], y += val[NT * 8 + i * width + threadIdx.x];
      tot[threadIdx.x] = u;
      tot[width + threadIdx.x] = y;
    }
  }
  __syncthreads();
}

// fused: part [N][2][C] = the item's channel sums
template <typename T, int NT, int KV, bool VEC, bool SAME>
__global__ __launch_bounds__(NT) void gn_bwd_fused_kernel(gn_args p) {
  extern __shared__ __attribute__((aligned(16))) float sm[];
  float* val = sm;                 // [2][NT * 8]
  float* tot = sm + NT * 16;       // [2][width]
  __shared__ float gs[2][MAXG];
  const int item = blockIdx.x / p.colblocks, cb = blockIdx.x - item * p.colblocks, c0 = cb * p.W, width = min(p.W, p.C - c0);
  const place<SAME> q = my_place<SAME, true>(p, c0, NT);
  const int gfirst = cb * (p.W / p.cg);
  const T* xend = (const T*)p.x + p.total;
  const T* x = (const T*)p.x + (int64_t)item * p.P * p.C;
  const T* gend = (const T*)p.gy + p.total;
  const T* gy = (const T*)p.gy + (int64_t)item * p.P * p.C;
  const uint32_t at0 = (uint32_t)(q.r * p.C + q.c), step = (uint32_t)(q.rpp * p.C);
  raw8<T> d[KV], e[KV];
#pragma unroll
  for (int k = 0; k < KV; ++k) {
    if (q.r + k * q.rpp < p.P && q.n > 0) {
      d[k] = load_raw<VEC>(x + (at0 + k * step), q.n, xend);
      e[k] = load_raw<VEC>(gy + (at0 + k * step), q.n, gend);
    } else {
      d[k].clear();
      e[k].clear();
    }
  }
  chan<SAME> ch;
  load_stats(p, q, item, gfirst, ch);
  load_affine<VEC>(p, q, ch);
  float a[8], b[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) a[i] = 0.f, b[i] = 0.f;
#pragma unroll
  for (int k = 0; k < KV; ++k)
    if (q.r + k * q.rpp < p.P) {
      float xh[8], du[8];
      grads8(p, ch, d[k], e[k], xh, du);
#pragma unroll
      for (int i = 0; i < 8; ++i) a[i] += du[i], b[i] = fmaf(du[i], xh[i], b[i]);
    }
#pragma unroll
  for (int k = 0; k < KV; ++k) d[k].forget(), e[k].forget();
  channel_sums<NT>(p, q.n, q.rpp, a, b, val, tot, width);
  const float inv_n = 1.f / ((float)p.P * (float)p.cg);
  sum_groups<NT, sum2<float>>(min(p.W / p.cg, p.G - gfirst), p.lg,
      [&](int g, int i) {
        const int c = g * p.cg + i;
        const float ga = p.gamma ? p.gamma[c0 + c] : 1.f;
        sum2<float> v;
        v.a = ga * tot[c];
        v.b = ga * tot[width + c];
        return v;
      },
      [&](int) { return p.cg; }, [&](int g, const sum2<float>& v) { gs[0][g] = v.a * inv_n, gs[1][g] = v.b * inv_n; });
  if (p.part)
    for (int c = threadIdx.x; c < width; c += NT) {
      p.part[((int64_t)item * 2) * p.C + c0 + c] = tot[c];
      p.part[((int64_t)item * 2 + 1) * p.C + c0 + c] = tot[width + c];
    }
  __syncthreads();
  if (q.n == 0) return;
  float c1[q.A], c2[q.A];
#pragma unroll
  for (int i = 0; i < q.A; ++i) {
    c1[i] = gs[0][q.g[i]];
    c2[i] = gs[1][q.g[i]];
  }
#pragma unroll
  for (int k = 0; k < KV; ++k) {
    const int r = q.r + k * q.rpp;
    if (r < p.P) put_gx<VEC>(p, q, ch, c1, c2, (int64_t)item * p.P + r, d[k], e[k]);
  }
}

// two-pass, first: part [N][slices][2][C]
template <typename T, bool VEC, bool SAME>
__global__ __launch_bounds__(256) void gn_bwd_sums_kernel(gn_args p) {
  __shared__ __attribute__((aligned(16))) float val[4096];
  __shared__ float tot[4096];
  const int item = blockIdx.x / p.slices, slice = blockIdx.x - item * p.slices, c0 = blockIdx.y * p.W, width = min(p.W, p.C - c0);
  const place<SAME> q = my_place<SAME>(p, c0, 256);
  const int r0 = slice_at(p, slice), r1 = slice_at(p, slice + 1);
  const int64_t base = (int64_t)item * p.P * p.C + q.c;
  const T* xend = (const T*)p.x + p.total;
  const T* x = (const T*)p.x + base;
  const T* gend = (const T*)p.gy + p.total;
  const T* gy = (const T*)p.gy + base;
  chan<SAME> ch;
  load_stats(p, q, item, 0, ch);
  load_affine<VEC>(p, q, ch);
  float a[8], b[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) a[i] = 0.f, b[i] = 0.f;
  auto take = [&](const raw8<T>& d, const raw8<T>& e) {
    float xh[8], du[8];
    grads8(p, ch, d, e, xh, du);
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] += du[i], b[i] = fmaf(du[i], xh[i], b[i]);
  };
  if (q.n > 0) {
    int r = r0 + q.r;
    for (; r + 3 * q.rpp < r1; r += 4 * q.rpp) {
      raw8<T> d[4], e[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        d[k] = load_raw<VEC>(x + (int64_t)(r + k * q.rpp) * p.C, q.n, xend);
        e[k] = load_raw<VEC>(gy + (int64_t)(r + k * q.rpp) * p.C, q.n, gend);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) take(d[k], e[k]);
    }
    for (; r < r1; r += q.rpp) take(load_raw<VEC>(x + (int64_t)r * p.C, q.n, xend), load_raw<VEC>(gy + (int64_t)r * p.C, q.n, gend));
  }
  channel_sums<256>(p, q.n, q.rpp, a, b, val, tot, width);
  float* out = p.part + ((int64_t)item * p.slices + slice) * 2 * p.C + c0;
  for (int c = threadIdx.x; c < width; c += 256) {
    out[c] = tot[c];
    out[p.C + c] = tot[width + c];
  }
}

// slices -> channel sums of the item, item_tot [N][2][C]: 32 channels x 8 interleaved chains of slices per workgroup
__global__ __launch_bounds__(256) void gn_bwd_item_kernel(gn_args p, float* __restrict__ item_tot) {
  __shared__ float red[8][64];
  const int l = threadIdx.x & 31, ph = threadIdx.x >> 5, c = blockIdx.y * 32 + l, item = blockIdx.x;
  const float* in = p.part + (int64_t)item * p.slices * 2 * p.C + c;
  float a = 0.f, b = 0.f;
  if (c < p.C)
#pragma unroll 4
    for (int r = ph; r < p.slices; r += 8) {
      a += in[(int64_t)r * 2 * p.C];
      b += in[((int64_t)r * 2 + 1) * p.C];
    }
  red[ph][l] = a;
  red[ph][32 + l] = b;
  __syncthreads();
  if (threadIdx.x < 64 && c < p.C) {
    float s = 0.f;
    for (int i = 0; i < 8; ++i) s += red[i][threadIdx.x];
    item_tot[((int64_t)item * 2 + (threadIdx.x >> 5)) * p.C + c] = s;
  }
}
template <typename T, bool VEC, bool SAME>
__global__ __launch_bounds__(256) void gn_bwd_apply_kernel(gn_args p, const float* __restrict__ item_tot) {
  __shared__ float gs[2][MAXW + 2];
  const int item = blockIdx.x / p.slices, slice = blockIdx.x - item * p.slices, c0 = blockIdx.y * p.W;
  const place<SAME> q = my_place<SAME>(p, c0, 256);
  // the means of h and h xh of this block's groups, from the item's channel sums (a group may reach beyond the block)
  const int gfirst = c0 / p.cg, groups = (min(c0 + p.W, p.C) - 1) / p.cg - gfirst + 1;
  const float* tot = item_tot + (int64_t)item * 2 * p.C;
  const float inv_n = 1.f / ((float)p.P * (float)p.cg);
  sum_groups<256, sum2<float>>(groups, p.lg,
      [&](int g, int i) {
        const int c = (gfirst + g) * p.cg + i;
        const float ga = p.gamma ? p.gamma[c] : 1.f;
        sum2<float> v;
        v.a = ga * tot[c];
        v.b = ga * tot[p.C + c];
        return v;
      },
      [&](int) { return p.cg; }, [&](int g, const sum2<float>& v) { gs[0][g] = v.a * inv_n, gs[1][g] = v.b * inv_n; });
  __syncthreads();
  if (q.n == 0) return;
  const int r0 = slice_at(p, slice), r1 = slice_at(p, slice + 1);
  const int64_t base = (int64_t)item * p.P * p.C + q.c;
  const T* xend = (const T*)p.x + p.total;
  const T* x = (const T*)p.x + base;
  const T* gend = (const T*)p.gy + p.total;
  const T* gy = (const T*)p.gy + base;
  chan<SAME> ch;
  load_stats(p, q, item, 0, ch);
  load_affine<VEC>(p, q, ch);
  float c1[q.A], c2[q.A];
#pragma unroll
  for (int i = 0; i < q.A; ++i) {
    c1[i] = gs[0][i < q.n ? q.g[i] - gfirst : 0];
    c2[i] = gs[1][i < q.n ? q.g[i] - gfirst : 0];
  }
#pragma unroll 2
  for (int r = r1 - 1 - q.r; r >= r0; r -= q.rpp) {   // (downwards, as in gn_apply_kernel)
    const raw8<T> d = load_raw<VEC>(x + (int64_t)r * p.C, q.n, xend), e = load_raw<VEC>(gy + (int64_t)r * p.C, q.n, gend);
    put_gx<VEC>(p, q, ch, c1, c2, (int64_t)item * p.P + r, d, e);
  }
}

// gbeta / ggamma: rows [rows][2][C] of channel sums, added in a fixed order (32 interleaved chains, then their sum).  With more
// than ROWS rows the workgroups along y take ROWS each and leave rows of the same layout in `next` for a second launch.
constexpr int ROWS = 1024;
__global__ __launch_bounds__(1024) void gn_param_grads_kernel(const float* __restrict__ part, int rows, int C,
                                                              float* __restrict__ ggamma, float* __restrict__ gbeta,
                                                              float* __restrict__ next) {
  __shared__ double red[32][65];
  const int l = threadIdx.x & 31, ph = threadIdx.x >> 5, c = blockIdx.x * 32 + l, r0 = blockIdx.y * ROWS;
  const int r1 = min(rows, r0 + ROWS);
  double a = 0.0, b = 0.0;
  if (c < C)
#pragma unroll 4
    for (int r = r0 + ph; r < r1; r += 32) {
      a += (double)part[(int64_t)r * 2 * C + c];
      b += (double)part[((int64_t)r * 2 + 1) * C + c];
    }
  red[ph][l] = a;
  red[ph][32 + l] = b;
  __syncthreads();
  if (threadIdx.x < 64) {
    double s = 0.0;
#pragma unroll 8
    for (int i = 0; i < 32; ++i) s += red[i][threadIdx.x];
    float* out = threadIdx.x < 32 ? gbeta : ggamma;
    if (next) out = next + ((int64_t)blockIdx.y * 2 + (threadIdx.x >> 5)) * C;
    if (out && c < C) out[c] = (float)s;
  }
}

// ---- which scheme: a function of the sizes and the element size -----------------------------------------------------------
struct gn_plan {
  bool fused;
  int W, tpr, colblocks, lg;
  int nt, kv;      // fused: threads, pieces per thread
  int slices;      // two-pass
};

int64_t gcd_(int64_t a, int64_t b) {
  while (b) {
    const int64_t t = a % b;
    a = b;
    b = t;
  }
  return a;
}

// kind 0 forward, 1 forward into 8-bit blocks, 2 backward
gn_plan make_gn_plan(int64_t N, int64_t P, int64_t C, int64_t G, int esize, int kind) {
  gn_plan r = {};
  const int64_t cg = C / G;
  // fused: whole groups, rows of at least 128 bytes where the channels allow, 8-bit blocks whole
  int64_t W = cg;
  const int64_t unit = kind == 1 ? F8B : 1;
  W = cg / gcd_(cg, unit) * unit;
  if (W < C && W * esize < 128) W = W * pgv_cdiv(128, W * esize);
  if (W % 8 && W < C) W = W * (8 / gcd_(W, 8));
  while (P * pgv_cdiv(W, 8) < 64 && W < C) W *= 2;   // few pixels: enough channels for a wave
  if (W > C) W = C;
  int64_t tpr = pgv_cdiv(W, 8);
  if (kind == 1) tpr = pgv_cdiv(W, F8B) * 16;
  const int64_t groups = pgv_cdiv(W, cg);
  // {threads, pieces of 8 values a thread holds, bytes per value at most}: the pieces take 8 or 4 registers each, twice that for
  // the backward pass, out of 128 with 1024 threads, 256 with 512 and 512 with fewer; pieces 17 to 24 are held in LDS.  One wave
  // per workgroup saves the barriers and most of what a thread does besides its values, where there are workgroups enough to
  // fill the device without more (160 x 16 blocks of 12 pixels: 8 us against 26 us with 256 threads).
  static const int fwd[][3] = {{64, 1, 4},  {64, 4, 4},   {64, 8, 4},   {256, 1, 4},   {256, 4, 4},
                               {256, 8, 4}, {1024, 4, 4}, {1024, 8, 4}, {1024, 16, 2}, {1024, 24, 2}};
  static const int bwd[][3] = {{64, 1, 4}, {64, 4, 4}, {64, 8, 4}, {256, 1, 4}, {256, 4, 4}, {256, 8, 4}, {512, 8, 4}, {512, 16, 2}};
  const bool many = N * pgv_cdiv(C, W) >= 1024;
  if (groups <= MAXG && P * C * esize < (1ll << 31))
    for (int i = many ? 0 : 3; i < (kind == 2 ? 8 : 10); ++i) {
      const int* c = kind == 2 ? bwd[i] : fwd[i];
      if (esize > c[2] || (c[1] == 24 && cg % 8)) continue;   // (groups of other widths need the LDS for their reductions)
      const int64_t rpp = c[0] / tpr;
      if (rpp >= 1 && P <= rpp * c[1]) {
        r.fused = true;
        r.W = (int)W;
        r.tpr = (int)tpr;
        r.nt = c[0];
        r.kv = c[1];
        r.colblocks = (int)pgv_cdiv(C, W);
        r.lg = lanes_log2(r.nt, groups);
        return r;
      }
    }
  r.W = (int)(C < MAXW ? C : MAXW);
  r.tpr = (int)(kind == 1 ? pgv_cdiv(r.W, F8B) * 16 : pgv_cdiv(r.W, 8));
  r.colblocks = (int)pgv_cdiv(C, r.W);
  r.lg = lanes_log2(256, G);
  const int64_t rpp = 256 / r.tpr;
  int64_t s = pgv_cdiv(2048, N * r.colblocks);
  const int64_t most = pgv_cdiv(P, rpp * 4);
  s = s < most ? s : most;
  r.slices = (int)(s < 1 ? 1 : s);
  return r;
}

int gn_check(const char* who, int64_t N, int64_t P, int64_t C, int64_t G, int dtype, int act) {
  PGV_CHECK_ARG(f8_dt_ok(dtype), "%s: unknown element type %d", who, dtype);
  PGV_CHECK_ARG(act >= PGV_ACT_NONE && act <= PGV_ACT_SILU, "%s: unknown activation %d", who, act);
  PGV_CHECK_ARG(N >= 0 && P >= 0 && C >= 0 && G > 0 && C % G == 0, "%s: bad sizes N=%lld P=%lld C=%lld groups=%lld", who,
                (long long)N, (long long)P, (long long)C, (long long)G);
  PGV_CHECK_ARG(N <= (1ll << 24) && P <= (1ll << 28) && C <= (1ll << 20) && N * G < (1ll << 31), "%s: too large (items %lld, pixels %lld, channels %lld)", who,
                (long long)N, (long long)P, (long long)C);
  return PGV_OK;
}

void set_plan(gn_args& p, const gn_plan& pl, bool same) {
  p.W = pl.W;
  p.tpr = pl.tpr;
  p.slices = pl.slices;
  p.colblocks = pl.colblocks;
  p.lg = pl.lg;
  p.m_tpr = magic_of(pl.tpr);
  p.m_cg = magic_of(p.cg);
  p.m_per = magic_of(same ? p.cg / 8 : p.cg);
}

template <typename T, bool VEC, bool Q, int FMT, bool SAME>
int gn_forward(gn_args p, const gn_plan& pl, hipStream_t st) {
  set_plan(p, pl, SAME);
  if (pl.fused) {
    const dim3 grid((unsigned)((int64_t)p.N * pl.colblocks));
#define PGV_F(NT, KV) gn_fwd_fused_kernel<T, NT, KV, 0, VEC, Q, FMT, SAME><<<grid, NT, 0, st>>>(p)
    if (pl.nt == 64)
      pl.kv == 1 ? PGV_F(64, 1) : pl.kv == 4 ? PGV_F(64, 4) : PGV_F(64, 8);
    else if (pl.nt == 256)
      pl.kv == 1 ? PGV_F(256, 1) : pl.kv == 4 ? PGV_F(256, 4) : PGV_F(256, 8);
    else if (pl.kv <= 8)
      pl.kv == 4 ? PGV_F(1024, 4) : PGV_F(1024, 8);
    else if constexpr (sizeof(T) == 2) {
      if (pl.kv == 16) {
        PGV_F(1024, 16);
      } else if constexpr (SAME) {
        auto k = gn_fwd_fused_kernel<T, 1024, 16, 8, VEC, Q, FMT, SAME>;
        constexpr int lds = 8 * 1024 * 16;
        static std::atomic<uint64_t> done{0};
        const int rc = f8_allow_lds((const void*)k, lds, done, "pgv_group_norm_act");
        if (rc != PGV_OK) return rc;
        k<<<grid, 1024, lds, st>>>(p);
      }
    }
#undef PGV_F
    return PGV_OK;
  }
  const dim3 grid((unsigned)((int64_t)p.N * pl.slices), (unsigned)pl.colblocks);
  gn_stats_kernel<T, VEC, SAME><<<grid, 256, 0, st>>>(p);
  // (a launch costs 5 us; 32 sums of 32 groups read by every workgroup cost 1, 128 of them more than the launch)
  const int parts = pl.slices * pl.colblocks;
  p.parts = parts <= 32 ? parts : 0;
  if (!p.parts) gn_finalize_kernel<<<dim3((unsigned)((int64_t)p.G * p.N)), 64, 0, st>>>(p, parts);
  gn_apply_kernel<T, VEC, Q, FMT, SAME><<<grid, 256, 0, st>>>(p);
  return PGV_OK;
}

template <typename T, int NT, int KV, bool VEC, bool SAME>
int launch_bwd_fused(const gn_args& p, dim3 grid, hipStream_t st) {
  auto k = gn_bwd_fused_kernel<T, NT, KV, VEC, SAME>;
  constexpr int most = NT * 16 * (int)sizeof(float) + 2 * 8 * NT * (int)sizeof(float);   // W is at most 8 NT channels
  static std::atomic<uint64_t> done{0};
  const int rc = f8_allow_lds((const void*)k, most, done, "pgv_group_norm_act_bwd");
  if (rc != PGV_OK) return rc;
  k<<<grid, NT, sizeof(float) * ((size_t)NT * 16 + 2 * (size_t)p.W), st>>>(p);
  return PGV_OK;
}

template <typename T, bool VEC, bool SAME>
int gn_backward(gn_args p, const gn_plan& pl, float* ggamma, float* gbeta, hipStream_t st) {
  set_plan(p, pl, SAME);
  const float* item_tot = p.part;
  if (pl.fused) {
    const dim3 grid((unsigned)((int64_t)p.N * pl.colblocks));
    int rc = PGV_OK;
    if (pl.nt == 64)
      rc = pl.kv == 1   ? launch_bwd_fused<T, 64, 1, VEC, SAME>(p, grid, st)
           : pl.kv == 4 ? launch_bwd_fused<T, 64, 4, VEC, SAME>(p, grid, st)
                        : launch_bwd_fused<T, 64, 8, VEC, SAME>(p, grid, st);
    else if (pl.nt == 256)
      rc = pl.kv == 1   ? launch_bwd_fused<T, 256, 1, VEC, SAME>(p, grid, st)
           : pl.kv == 4 ? launch_bwd_fused<T, 256, 4, VEC, SAME>(p, grid, st)
                        : launch_bwd_fused<T, 256, 8, VEC, SAME>(p, grid, st);
    else if (pl.kv == 8)
      rc = launch_bwd_fused<T, 512, 8, VEC, SAME>(p, grid, st);
    else if constexpr (sizeof(T) == 2)
      rc = launch_bwd_fused<T, 512, 16, VEC, SAME>(p, grid, st);
    if (rc != PGV_OK) return rc;
  } else {
    const dim3 grid((unsigned)((int64_t)p.N * pl.slices), (unsigned)pl.colblocks);
    float* tot = p.part + (int64_t)p.N * pl.slices * 2 * p.C;
    gn_bwd_sums_kernel<T, VEC, SAME><<<grid, 256, 0, st>>>(p);
    gn_bwd_item_kernel<<<dim3((unsigned)p.N, (unsigned)pgv_cdiv(p.C, 32)), 256, 0, st>>>(p, tot);
    gn_bwd_apply_kernel<T, VEC, SAME><<<grid, 256, 0, st>>>(p, tot);
    item_tot = tot;
  }
  if (ggamma || gbeta) {
    const unsigned cols = (unsigned)pgv_cdiv(p.C, 32);
    int rows = p.N;
    float* next = p.part + (int64_t)p.N * (pl.fused ? 1 : pl.slices + 1) * 2 * p.C;
    while (rows > ROWS) {
      const int n = (int)pgv_cdiv(rows, ROWS);
      gn_param_grads_kernel<<<dim3(cols, (unsigned)n), 1024, 0, st>>>(item_tot, rows, p.C, nullptr, nullptr, next);
      item_tot = next;
      next += (int64_t)n * 2 * p.C;
      rows = n;
    }
    gn_param_grads_kernel<<<dim3(cols), 1024, 0, st>>>(item_tot, rows, p.C, ggamma, gbeta, nullptr);
  }
  return PGV_OK;
}

}  // namespace

extern "C" int64_t pgv_group_norm_workspace(int64_t N, int64_t P, int64_t C, int64_t G, int dtype, int kind) {
  if (N <= 0 || P <= 0 || C <= 0 || G <= 0 || C % G || !f8_dt_ok(dtype) || kind < 0 || kind > 2) return 0;
  const gn_plan pl = make_gn_plan(N, P, C, G, f8_dt_size(dtype), kind);
  if (kind == 2) {
    int64_t rows = N * (pl.fused ? 1 : pl.slices + 1);
    for (int64_t n = N; n > ROWS;) n = pgv_cdiv(n, ROWS), rows += n;   // (gn_param_grads_kernel's levels)
    return 4 * rows * 2 * C;
  }
  const int64_t stats = kind == 1 && !pl.fused ? 8 * N * G : 0;   // mean and rstd live here when the caller has no use for them
  return stats + (pl.fused ? 0 : 16 * N * G * pl.slices * pl.colblocks);
}

static int gn_fwd_any(const char* who, const void* x, int dtype, int64_t N, int64_t P, int64_t C, int64_t G, const float* gamma,
                      const float* beta, float eps, int act, float slope, void* y, float* mean, float* rstd, void* q, float* scale,
                      int fmt, void* workspace, int64_t workspace_bytes, void* stream) {
  const int rc = gn_check(who, N, P, C, G, dtype, act);
  if (rc != PGV_OK) return rc;
  if (N == 0 || P == 0 || C == 0) return PGV_OK;
  const int kind = q ? 1 : 0;
  PGV_CHECK_ARG(x && (q ? scale != nullptr : (y && mean && rstd)), "%s: null tensor", who);
  PGV_CHECK_ARG(!q || (uintptr_t)q % 16 == 0, "%s: the 8-bit output must be 16-byte aligned", who);
  const int64_t need = pgv_group_norm_workspace(N, P, C, G, dtype, kind);
  if (need > 0 && (!workspace || workspace_bytes < need)) {
    pgv_set_error("%s: workspace of %lld bytes needed", who, (long long)need);
    return PGV_E_WORKSPACE;
  }
  const gn_plan pl = make_gn_plan(N, P, C, G, f8_dt_size(dtype), kind);
  gn_args p = {};
  p.N = (int)N, p.P = (int)P, p.C = (int)C, p.G = (int)G, p.cg = (int)(C / G), p.total = N * P * C;
  p.x = x, p.gamma = gamma, p.beta = beta, p.eps = eps, p.slope = slope, p.act = act;
  p.y = y, p.q = (uint8_t*)q, p.scale = scale, p.Kp = (int)(pgv_cdiv(C, F8B) * F8B);
  p.mean = mean, p.rstd = rstd;
  p.part = (float*)workspace;
  if (kind == 1 && !pl.fused) {
    float* tail = (float*)((char*)workspace + need - 8 * N * G);
    p.mean = tail, p.rstd = tail + N * G;
  }
  const bool vec = C % 8 == 0 && (uintptr_t)x % 16 == 0 && (uintptr_t)gamma % 16 == 0 && (uintptr_t)beta % 16 == 0 && (q || (uintptr_t)y % 16 == 0);
  hipStream_t st = pgv_stream(stream);
  int r;
  const bool same = p.cg % 8 == 0;
#define PGV_V(T, VEC, Q, FMT) (same ? gn_forward<T, VEC, Q, FMT, true>(p, pl, st) : gn_forward<T, VEC, Q, FMT, false>(p, pl, st))
#define PGV_T(T, Q, FMT) (vec ? PGV_V(T, true, Q, FMT) : PGV_V(T, false, Q, FMT))
#define PGV_D(Q, FMT) (dtype == PGV_DT_F32 ? PGV_T(float, Q, FMT) : dtype == PGV_DT_BF16 ? PGV_T(__bf16, Q, FMT) : PGV_T(_Float16, Q, FMT))
  if (!q)
    r = PGV_D(false, PGV_F8_E4M3);
  else
    r = fmt == PGV_F8_E4M3 ? PGV_D(true, PGV_F8_E4M3) : PGV_D(true, PGV_F8_E5M2);
#undef PGV_D
#undef PGV_T
#undef PGV_V
  if (r != PGV_OK) return r;
  PGV_CHECK_LAUNCH(who);
  return PGV_OK;
}

extern "C" int pgv_group_norm_act_fwd(const void* x, int dtype, int64_t N, int64_t P, int64_t C, int64_t G, const float* gamma,
                                      const float* beta, float eps, int act, float slope, void* y, float* mean, float* rstd,
                                      void* workspace, int64_t workspace_bytes, void* stream) {
  return gn_fwd_any("pgv_group_norm_act_fwd", x, dtype, N, P, C, G, gamma, beta, eps, act, slope, y, mean, rstd, nullptr, nullptr, 0,
                    workspace, workspace_bytes, stream);
}

extern "C" int pgv_group_norm_act_f8(const void* x, int dtype, int64_t N, int64_t P, int64_t C, int64_t G, const float* gamma,
                                     const float* beta, float eps, int act, float slope, int fmt, void* q, float* scale,
                                     void* workspace, int64_t workspace_bytes, void* stream) {
  PGV_CHECK_ARG(fmt == PGV_F8_E4M3 || fmt == PGV_F8_E5M2, "pgv_group_norm_act_f8: unknown 8-bit format %d", fmt);
  PGV_CHECK_ARG(q || N == 0 || P == 0 || C == 0, "pgv_group_norm_act_f8: null tensor");
  return gn_fwd_any("pgv_group_norm_act_f8", x, dtype, N, P, C, G, gamma, beta, eps, act, slope, nullptr, nullptr, nullptr, q, scale,
                    fmt, workspace, workspace_bytes, stream);
}

extern "C" int pgv_group_norm_act_bwd(const void* gy, const void* x, int dtype, int64_t N, int64_t P, int64_t C, int64_t G,
                                      const float* gamma, const float* beta, const float* mean, const float* rstd, int act,
                                      float slope, void* gx, float* ggamma, float* gbeta, void* workspace, int64_t workspace_bytes,
                                      void* stream) {
  const int rc = gn_check("pgv_group_norm_act_bwd", N, P, C, G, dtype, act);
  if (rc != PGV_OK) return rc;
  PGV_CHECK_ARG((N > 0 && P > 0 && C > 0) || (!ggamma && !gbeta), "pgv_group_norm_act_bwd: parameter gradients of an empty tensor");
  if (N == 0 || P == 0 || C == 0) return PGV_OK;
  PGV_CHECK_ARG(gy && x && mean && rstd && gx, "pgv_group_norm_act_bwd: null tensor");
  const int64_t need = pgv_group_norm_workspace(N, P, C, G, dtype, 2);
  if (!workspace || workspace_bytes < need) {
    pgv_set_error("pgv_group_norm_act_bwd: workspace of %lld bytes needed", (long long)need);
    return PGV_E_WORKSPACE;
  }
  const gn_plan pl = make_gn_plan(N, P, C, G, f8_dt_size(dtype), 2);
  gn_args p = {};
  p.N = (int)N, p.P = (int)P, p.C = (int)C, p.G = (int)G, p.cg = (int)(C / G), p.total = N * P * C;
  p.x = x, p.gy = gy, p.gx = gx, p.gamma = gamma, p.beta = beta, p.slope = slope, p.act = act;
  p.mean = const_cast<float*>(mean), p.rstd = const_cast<float*>(rstd);
  p.part = (float*)workspace;
  const bool vec = C % 8 == 0 && (uintptr_t)gamma % 16 == 0 && (uintptr_t)beta % 16 == 0 && (uintptr_t)x % 16 == 0 && (uintptr_t)gy % 16 == 0 && (uintptr_t)gx % 16 == 0;
  hipStream_t st = pgv_stream(stream);
  const bool same = p.cg % 8 == 0;
#define PGV_T(T)                                                                                                  \
  (vec ? (same ? gn_backward<T, true, true>(p, pl, ggamma, gbeta, st) : gn_backward<T, true, false>(p, pl, ggamma, gbeta, st)) \
       : gn_backward<T, false, false>(p, pl, ggamma, gbeta, st))
  const int r = dtype == PGV_DT_F32 ? PGV_T(float) : dtype == PGV_DT_BF16 ? PGV_T(__bf16) : PGV_T(_Float16);
#undef PGV_T
  if (r != PGV_OK) return r;
  PGV_CHECK_LAUNCH("pgv_group_norm_act_bwd");
  return PGV_OK;
}
