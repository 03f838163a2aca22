// GroupNorm + activation over x[N][P][C] (P pixels of an item, channels last), forward, backward and forward into 8-bit blocks:
//   mean, var over the P x C/G values of (item, group); xh = (x - mean) / sqrt(var + eps); u = gamma xh + beta; y = act(u)
//   du = gy act'(u); gbeta = sum du; ggamma = sum du xh; h = gamma du; gx = rstd (h - mean(h) - xh mean(h xh))
//
// Bound by memory.  A thread owns 8 neighbouring channels for the whole kernel (their gamma, beta, mean and rstd stay in
// registers) and walks over pixels: a row of C channels is C / 8 threads and 16 or 32 bytes each.  Two schemes:
//   fused     the pixels of one item and of a few whole groups fit in the registers of a workgroup: every value is read once,
//             mean and variance are two passes over registers (the variance of x - mean: nothing cancels), one launch.
//   two-pass  everything else: partial sums per slice of pixels, a finalising kernel, a second pass.  The slices' sums of x and
//             x^2 are 64-bit ones: their difference is the variance, and it may be far smaller than either.
#include "f8_common.h"

namespace {

struct gn_args {
  int N, P, C, G, cg;
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
  float* coef;          // backward: [N][G][2] = mean(h), mean(h xh)
  int W, tpr, slices;   // channels per workgroup, threads per row, pixel slices
};

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

// 8 neighbouring values as they lie in memory
template <typename T>
struct raw8 {
  T v[8];
};
template <bool VEC, typename T>
__device__ __forceinline__ raw8<T> load_raw(const T* __restrict__ p, int n) {
  raw8<T> r;
  if constexpr (VEC) {
    typedef T t8 __attribute__((ext_vector_type(8)));
    typedef T t4 __attribute__((ext_vector_type(4)));
    if constexpr (sizeof(T) == 4) {
      const t4 a = reinterpret_cast<const t4*>(p)[0], b = reinterpret_cast<const t4*>(p)[1];
#pragma unroll
      for (int i = 0; i < 4; ++i) r.v[i] = a[i], r.v[4 + i] = b[i];
    } else {
      const t8 a = *reinterpret_cast<const t8*>(p);
#pragma unroll
      for (int i = 0; i < 8; ++i) r.v[i] = a[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) r.v[i] = i < n ? p[i] : (T)0.f;
  }
  return r;
}
template <bool VEC, typename T>
__device__ __forceinline__ void store8(T* __restrict__ p, int n, const float (&v)[8]) {
  if constexpr (VEC) {
    if constexpr (sizeof(T) == 4) {
      f32x4 a, b;
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = v[i], b[i] = v[4 + i];
      reinterpret_cast<f32x4*>(p)[0] = a;
      reinterpret_cast<f32x4*>(p)[1] = b;
    } else {
      typedef T t8 __attribute__((ext_vector_type(8)));
      t8 a;
#pragma unroll
      for (int i = 0; i < 8; ++i) a[i] = (T)v[i];
      *reinterpret_cast<t8*>(p) = a;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = (T)v[i];
  }
}

// One thread's place: 8 channels from c, valid ones n (0: a pad column of the 8-bit rows or an idle thread), pixel phase r.
struct place {
  int c, n, r, rpp;
};
__device__ __forceinline__ place my_place(const gn_args& p, int c0, int nt) {
  place q;
  const int j = threadIdx.x % p.tpr;
  q.rpp = nt / p.tpr;
  q.r = threadIdx.x / p.tpr;
  q.c = c0 + 8 * j;
  const int end = min(c0 + p.W, p.C);
  q.n = q.r < q.rpp ? max(0, min(8, end - q.c)) : 0;
  return q;
}
// the per-channel vectors of a place; channels beyond the valid ones normalise to 0
struct chan {
  float ga[8], be[8], mu[8], rs[8];
};
__device__ __forceinline__ void load_affine(const gn_args& p, const place& q, chan& k) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    k.ga[i] = i < q.n && p.gamma ? p.gamma[q.c + i] : (i < q.n ? 1.f : 0.f);
    k.be[i] = i < q.n && p.beta ? p.beta[q.c + i] : 0.f;
  }
}
__device__ __forceinline__ void load_stats(const gn_args& p, const place& q, int item, chan& k) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t g = (int64_t)item * p.G + (i < q.n ? (q.c + i) / p.cg : 0);
    k.mu[i] = i < q.n ? p.mean[g] : 0.f;
    k.rs[i] = i < q.n ? p.rstd[g] : 0.f;
  }
}

// y (or its 8-bit block) of one pixel
template <bool VEC, bool Q, int FMT, typename T>
__device__ __forceinline__ void put(const gn_args& p, const place& q, const chan& k, int64_t pix, const raw8<T>& x) {
  float u[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) u[i] = fmaf(((float)x.v[i] - k.mu[i]) * k.rs[i], k.ga[i], k.be[i]);
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

// sums over (pixel phases x channels) of each local group: val[tid][8] in LDS -> out[group]
__device__ __forceinline__ void group_sums(const gn_args& p, const float* val, int tpr, int rpp, int groups, float* out) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, nw = blockDim.x >> 6;
  for (int g = wave; g < groups; g += nw) {
    float s = 0.f;
    for (int e = lane; e < rpp * p.cg; e += 64) {
      const int r = e / p.cg, c = g * p.cg + e % p.cg;
      s += val[r * tpr * 8 + c];
    }
    s = pgv_wave_sum(s);
    if (lane == 0) out[g] = s;
  }
}
// the same for groups of whole 8-channel pieces: val[tid] is the sum of a thread's channels
__device__ __forceinline__ void group_sums8(const gn_args& p, const float* val, int tpr, int rpp, int groups, float* out) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, nw = blockDim.x >> 6, per = p.cg >> 3;
  for (int g = wave; g < groups; g += nw) {
    float s = 0.f;
    for (int e = lane; e < rpp * per; e += 64) s += val[(e / per) * tpr + g * per + e % per];
    s = pgv_wave_sum(s);
    if (lane == 0) out[g] = s;
  }
}

constexpr int MAXG = 256;   // groups of a workgroup of the fused kernels

// ---- forward, fused: grid (column blocks of W channels, items) -----------------------------------------------------------
template <typename T, int NT, int KV, bool VEC, bool Q, int FMT, bool SAME>
__global__ __launch_bounds__(NT) void gn_fwd_fused_kernel(gn_args p) {
  __shared__ float val[SAME ? NT : NT * 8];
  __shared__ float gs[2][MAXG];
  const int tid = threadIdx.x, item = blockIdx.y, c0 = blockIdx.x * p.W;
  const place q = my_place(p, c0, NT);
  const bool idle = q.r >= q.rpp;
  const int groups = min(p.W, p.C - c0) / p.cg;
  const T* x = (const T*)p.x + (int64_t)item * p.P * p.C;
  raw8<T> d[KV];
#pragma unroll
  for (int k = 0; k < KV; ++k) {
    const int r = q.r + k * q.rpp;
    if (r < p.P && q.n > 0)
      d[k] = load_raw<VEC>(x + (int64_t)r * p.C + q.c, q.n);
    else
#pragma unroll
      for (int i = 0; i < 8; ++i) d[k].v[i] = (T)0.f;
  }
  chan ch;
  load_affine(p, q, ch);
  const float inv_n = 1.f / ((float)p.P * (float)p.cg);
  // pass 0: mean; pass 1: variance
#pragma unroll
  for (int i = 0; i < 8; ++i) ch.mu[i] = 0.f;
#pragma unroll
  for (int pass = 0; pass < 2; ++pass) {
    float s[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] = 0.f;
#pragma unroll
    for (int k = 0; k < KV; ++k)
      if (q.r + k * q.rpp < p.P)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float v = (float)d[k].v[i] - ch.mu[i];
          s[i] += pass ? v * v : v;
        }
    if (pass) __syncthreads();   // the readers of val and gs of pass 0 are done
    if constexpr (SAME) {
      val[tid] = q.n > 0 ? ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7])) : 0.f;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) val[tid * 8 + i] = i < q.n ? s[i] : 0.f;
    }
    __syncthreads();
    if constexpr (SAME)
      group_sums8(p, val, p.tpr, q.rpp, groups, gs[pass]);
    else
      group_sums(p, val, p.tpr, q.rpp, groups, gs[pass]);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int g = i < q.n ? (q.c + i - c0) / p.cg : 0;
      if (pass == 0)
        ch.mu[i] = i < q.n ? gs[0][g] * inv_n : 0.f;
      else
        ch.rs[i] = i < q.n ? 1.f / sqrtf(gs[1][g] * inv_n + p.eps) : 0.f;
    }
  }
  if (p.mean)
    for (int g = tid; g < groups; g += NT) {
      const int64_t o = (int64_t)item * p.G + c0 / p.cg + g;
      p.mean[o] = gs[0][g] * inv_n;
      p.rstd[o] = 1.f / sqrtf(gs[1][g] * inv_n + p.eps);
    }
  if (idle) return;
#pragma unroll
  for (int k = 0; k < KV; ++k) {
    const int r = q.r + k * q.rpp;
    if (r < p.P && (Q || q.n > 0)) put<VEC, Q, FMT>(p, q, ch, (int64_t)item * p.P + r, d[k]);
  }
}

// ---- forward, two-pass --------------------------------------------------------------------------------------------------
// partial sums: part (as double2) [N][slices * column blocks][G] of (sum, sum of squares), zero for groups outside the block
template <typename T, bool VEC, bool SAME>
__global__ __launch_bounds__(256) void gn_stats_kernel(gn_args p) {
  __shared__ double2 val[SAME ? 256 : 2048];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, item = blockIdx.z, slice = blockIdx.x, c0 = blockIdx.y * p.W;
  const place q = my_place(p, c0, 256);
  const int r0 = (int)((int64_t)p.P * slice / p.slices), r1 = (int)((int64_t)p.P * (slice + 1) / p.slices);
  const T* x = (const T*)p.x + (int64_t)item * p.P * p.C + q.c;
  constexpr int A = SAME ? 1 : 8;
  double s[A], ss[A];
#pragma unroll
  for (int i = 0; i < A; ++i) s[i] = 0.0, ss[i] = 0.0;
  if (q.n > 0) {
    int r = r0 + q.r;
    for (; r + 3 * q.rpp < r1; r += 4 * q.rpp) {
      raw8<T> d[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) d[k] = load_raw<VEC>(x + (int64_t)(r + k * q.rpp) * p.C, q.n);
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const double v = (double)(float)d[k].v[i];
          s[SAME ? 0 : i] += v;
          ss[SAME ? 0 : i] = fma(v, v, ss[SAME ? 0 : i]);
        }
    }
    for (; r < r1; r += q.rpp) {
      const raw8<T> d = load_raw<VEC>(x + (int64_t)r * p.C, q.n);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const double v = (double)(float)d.v[i];
        s[SAME ? 0 : i] += v;
        ss[SAME ? 0 : i] = fma(v, v, ss[SAME ? 0 : i]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < A; ++i) val[tid * A + i] = make_double2(s[i], ss[i]);
  __syncthreads();
  double2* out = (double2*)p.part + ((int64_t)item * (p.slices * gridDim.y) + (int64_t)blockIdx.y * p.slices + slice) * p.G;
  const int cend = min(c0 + p.W, p.C);
  for (int g = wave; g < p.G; g += 4) {
    const int lo = max(g * p.cg, c0), hi = min((g + 1) * p.cg, cend);   // (lo >= hi: outside this block)
    double a = 0.0, b = 0.0;
    if (lo < hi) {
      const int w = SAME ? (hi - lo) >> 3 : hi - lo, base = SAME ? (lo - c0) >> 3 : lo - c0, pitch = SAME ? p.tpr : p.tpr * 8;
      for (int e = lane; e < q.rpp * w; e += 64) {
        const double2 v = val[(e / w) * pitch + base + e % w];
        a += v.x;
        b += v.y;
      }
      a = pgv_wave_sum_d(a);
      b = pgv_wave_sum_d(b);
    }
    if (lane == 0) out[g] = make_double2(a, b);
  }
}

__global__ __launch_bounds__(64) void gn_finalize_kernel(gn_args p, int parts) {
  const int g = blockIdx.x, item = blockIdx.y, lane = threadIdx.x;
  const double2* in = (const double2*)p.part + (int64_t)item * parts * p.G + g;
  double a = 0.0, b = 0.0;
  for (int e = lane; e < parts; e += 64) {
    const double2 v = in[(int64_t)e * p.G];
    a += v.x;
    b += v.y;
  }
  a = pgv_wave_sum_d(a);
  b = pgv_wave_sum_d(b);
  if (lane == 0) {
    const double n = (double)p.P * (double)p.cg, m = a / n, var = b / n - m * m;
    p.mean[(int64_t)item * p.G + g] = (float)m;
    p.rstd[(int64_t)item * p.G + g] = (float)(1.0 / sqrt((var > 0.0 || var != var ? var : 0.0) + (double)p.eps));
  }
}

template <typename T, bool VEC, bool Q, int FMT>
__global__ __launch_bounds__(256) void gn_apply_kernel(gn_args p) {
  const int item = blockIdx.z, slice = blockIdx.x, c0 = blockIdx.y * p.W;
  const place q = my_place(p, c0, 256);
  if (q.r >= q.rpp || (!Q && q.n == 0)) return;
  const int r0 = (int)((int64_t)p.P * slice / p.slices), r1 = (int)((int64_t)p.P * (slice + 1) / p.slices);
  const T* x = (const T*)p.x + (int64_t)item * p.P * p.C + q.c;
  chan ch;
  load_affine(p, q, ch);
  load_stats(p, q, item, ch);
  int r = r0 + q.r;
  for (; r + 3 * q.rpp < r1; r += 4 * q.rpp) {
    raw8<T> d[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (!Q || q.n > 0)
        d[k] = load_raw<VEC>(x + (int64_t)(r + k * q.rpp) * p.C, q.n);
      else
#pragma unroll
        for (int i = 0; i < 8; ++i) d[k].v[i] = (T)0.f;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) put<VEC, Q, FMT>(p, q, ch, (int64_t)item * p.P + r + k * q.rpp, d[k]);
  }
  for (; r < r1; r += q.rpp) {
    raw8<T> d;
    if (!Q || q.n > 0)
      d = load_raw<VEC>(x + (int64_t)r * p.C, q.n);
    else
#pragma unroll
      for (int i = 0; i < 8; ++i) d.v[i] = (T)0.f;
    put<VEC, Q, FMT>(p, q, ch, (int64_t)item * p.P + r, d);
  }
}

// ---- backward -----------------------------------------------------------------------------------------------------------
// xh and du of 8 values
template <typename T>
__device__ __forceinline__ void grads8(const gn_args& p, const chan& k, const raw8<T>& x, const raw8<T>& gy, float (&xh)[8],
                                       float (&du)[8]) {
  float u[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    xh[i] = ((float)x.v[i] - k.mu[i]) * k.rs[i];
    u[i] = fmaf(xh[i], k.ga[i], k.be[i]);
    du[i] = (float)gy.v[i];
  }
  act_grad8(du, u, p.act, p.slope);
}
template <bool VEC, typename T>
__device__ __forceinline__ void put_gx(const gn_args& p, const place& q, const chan& k, const float (&c1)[8], const float (&c2)[8],
                                       int64_t pix, const raw8<T>& x, const raw8<T>& gy) {
  float xh[8], du[8], o[8];
  grads8(p, k, x, gy, xh, du);
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = k.rs[i] * (fmaf(k.ga[i], du[i], -c1[i]) - xh[i] * c2[i]);
  store8<VEC>((T*)p.gx + pix * p.C + q.c, q.n, o);
}
// per-channel sums over the pixel phases of a workgroup: a = sum du, b = sum du xh -> tot[2][W]
template <int NT>
__device__ __forceinline__ void channel_sums(const gn_args& p, const place& q, const float (&a)[8], const float (&b)[8],
                                             float* val /* [NT * 8] */, float* tot /* [2][NT * 8 at most] */, int width) {
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    if (t) __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) val[threadIdx.x * 8 + i] = i < q.n ? (t ? b[i] : a[i]) : 0.f;
    __syncthreads();
    for (int c = threadIdx.x; c < width; c += NT) {
      float s = 0.f;
      for (int r = 0; r < q.rpp; ++r) s += val[r * p.tpr * 8 + c];
      tot[t * width + c] = s;
    }
  }
  __syncthreads();
}

// fused: part [N][2][C] = the item's channel sums
template <typename T, int NT, int KV, bool VEC>
__global__ __launch_bounds__(NT) void gn_bwd_fused_kernel(gn_args p) {
  extern __shared__ float sm[];
  float* val = sm;                 // [NT * 8]
  float* tot = sm + NT * 8;        // [2][width]
  __shared__ float gs[2][MAXG];
  const int item = blockIdx.y, c0 = blockIdx.x * p.W, width = min(p.W, p.C - c0);
  const place q = my_place(p, c0, NT);
  const T* x = (const T*)p.x + (int64_t)item * p.P * p.C;
  const T* gy = (const T*)p.gy + (int64_t)item * p.P * p.C;
  raw8<T> d[KV], e[KV];
#pragma unroll
  for (int k = 0; k < KV; ++k) {
    const int r = q.r + k * q.rpp;
    if (r < p.P && q.n > 0) {
      d[k] = load_raw<VEC>(x + (int64_t)r * p.C + q.c, q.n);
      e[k] = load_raw<VEC>(gy + (int64_t)r * p.C + q.c, q.n);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) d[k].v[i] = (T)0.f, e[k].v[i] = (T)0.f;
    }
  }
  chan ch;
  load_affine(p, q, ch);
  load_stats(p, q, item, ch);
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
  channel_sums<NT>(p, q, a, b, val, tot, width);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int g = wave; g < width / p.cg; g += NT / 64) {
    float s1 = 0.f, s2 = 0.f;
    for (int i = lane; i < p.cg; i += 64) {
      const int c = g * p.cg + i;
      const float ga = p.gamma ? p.gamma[c0 + c] : 1.f;
      s1 = fmaf(ga, tot[c], s1);
      s2 = fmaf(ga, tot[width + c], s2);
    }
    s1 = pgv_wave_sum(s1);
    s2 = pgv_wave_sum(s2);
    const float n = (float)p.P * (float)p.cg;
    if (lane == 0) gs[0][g] = s1 / n, gs[1][g] = s2 / n;
  }
  if (p.part)
    for (int c = threadIdx.x; c < width; c += NT) {
      p.part[((int64_t)item * 2) * p.C + c0 + c] = tot[c];
      p.part[((int64_t)item * 2 + 1) * p.C + c0 + c] = tot[width + c];
    }
  __syncthreads();
  if (q.n == 0) return;
  float c1[8], c2[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int g = i < q.n ? (q.c + i - c0) / p.cg : 0;
    c1[i] = gs[0][g];
    c2[i] = gs[1][g];
  }
#pragma unroll
  for (int k = 0; k < KV; ++k) {
    const int r = q.r + k * q.rpp;
    if (r < p.P) put_gx<VEC>(p, q, ch, c1, c2, (int64_t)item * p.P + r, d[k], e[k]);
  }
}

// two-pass, first: part [N][slices][2][C]
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void gn_bwd_sums_kernel(gn_args p) {
  __shared__ float val[2048], tot[4096];
  const int item = blockIdx.z, slice = blockIdx.x, c0 = blockIdx.y * p.W, width = min(p.W, p.C - c0);
  const place q = my_place(p, c0, 256);
  const int r0 = (int)((int64_t)p.P * slice / p.slices), r1 = (int)((int64_t)p.P * (slice + 1) / p.slices);
  const int64_t base = (int64_t)item * p.P * p.C + q.c;
  const T* x = (const T*)p.x + base;
  const T* gy = (const T*)p.gy + base;
  chan ch;
  load_affine(p, q, ch);
  load_stats(p, q, item, ch);
  float a[8], b[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) a[i] = 0.f, b[i] = 0.f;
  if (q.n > 0)
#pragma unroll 2
    for (int r = r0 + q.r; r < r1; r += q.rpp) {
      const raw8<T> d = load_raw<VEC>(x + (int64_t)r * p.C, q.n), e = load_raw<VEC>(gy + (int64_t)r * p.C, q.n);
      float xh[8], du[8];
      grads8(p, ch, d, e, xh, du);
#pragma unroll
      for (int i = 0; i < 8; ++i) a[i] += du[i], b[i] = fmaf(du[i], xh[i], b[i]);
    }
  channel_sums<256>(p, q, a, b, val, tot, width);
  float* out = p.part + ((int64_t)item * p.slices + slice) * 2 * p.C + c0;
  for (int c = threadIdx.x; c < width; c += 256) {
    out[c] = tot[c];
    out[p.C + c] = tot[width + c];
  }
}

// slices -> the group means of h and h xh
__global__ __launch_bounds__(64) void gn_bwd_finalize_kernel(gn_args p) {
  const int g = blockIdx.x, item = blockIdx.y, lane = threadIdx.x;
  const float* in = p.part + (int64_t)item * p.slices * 2 * p.C + g * p.cg;
  double s1 = 0.0, s2 = 0.0;
  for (int64_t e = lane; e < (int64_t)p.slices * p.cg; e += 64) {
    const int sl = (int)(e / p.cg), c = (int)(e % p.cg);
    const double ga = p.gamma ? (double)p.gamma[g * p.cg + c] : 1.0;
    s1 += ga * (double)in[(int64_t)sl * 2 * p.C + c];
    s2 += ga * (double)in[(int64_t)sl * 2 * p.C + p.C + c];
  }
  s1 = pgv_wave_sum_d(s1);
  s2 = pgv_wave_sum_d(s2);
  if (lane == 0) {
    const double n = (double)p.P * (double)p.cg;
    p.coef[((int64_t)item * p.G + g) * 2] = (float)(s1 / n);
    p.coef[((int64_t)item * p.G + g) * 2 + 1] = (float)(s2 / n);
  }
}

template <typename T, bool VEC>
__global__ __launch_bounds__(256) void gn_bwd_apply_kernel(gn_args p) {
  const int item = blockIdx.z, slice = blockIdx.x, c0 = blockIdx.y * p.W;
  const place q = my_place(p, c0, 256);
  if (q.n == 0) return;
  const int r0 = (int)((int64_t)p.P * slice / p.slices), r1 = (int)((int64_t)p.P * (slice + 1) / p.slices);
  const int64_t base = (int64_t)item * p.P * p.C + q.c;
  const T* x = (const T*)p.x + base;
  const T* gy = (const T*)p.gy + base;
  chan ch;
  load_affine(p, q, ch);
  load_stats(p, q, item, ch);
  float c1[8], c2[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t g = (int64_t)item * p.G + (i < q.n ? (q.c + i) / p.cg : 0);
    c1[i] = p.coef[2 * g];
    c2[i] = p.coef[2 * g + 1];
  }
#pragma unroll 2
  for (int r = r0 + q.r; r < r1; r += q.rpp) {
    const raw8<T> d = load_raw<VEC>(x + (int64_t)r * p.C, q.n), e = load_raw<VEC>(gy + (int64_t)r * p.C, q.n);
    put_gx<VEC>(p, q, ch, c1, c2, (int64_t)item * p.P + r, d, e);
  }
}

// gbeta / ggamma: rows [rows][2][C] of channel sums, added in a fixed order (8 interleaved chains, then their sum)
__global__ __launch_bounds__(256) void gn_param_grads_kernel(const float* __restrict__ part, int64_t rows, int C,
                                                             float* __restrict__ ggamma, float* __restrict__ gbeta) {
  __shared__ double red[8][64];
  const int l = threadIdx.x & 31, ph = threadIdx.x >> 5, c = blockIdx.x * 32 + l;
  double a = 0.0, b = 0.0;
  if (c < C)
#pragma unroll 4
    for (int64_t r = ph; r < rows; r += 8) {
      a += (double)part[r * 2 * C + c];
      b += (double)part[(r * 2 + 1) * C + c];
    }
  red[ph][l] = a;
  red[ph][32 + l] = b;
  __syncthreads();
  if (threadIdx.x < 64) {
    double s = 0.0;
    for (int i = 0; i < 8; ++i) s += red[i][threadIdx.x];
    float* out = threadIdx.x < 32 ? gbeta : ggamma;
    if (out && c < C) out[c] = (float)s;
  }
}

// ---- which scheme: a function of the sizes and the element size -----------------------------------------------------------
struct gn_plan {
  bool fused;
  int W, tpr, nt, kv;      // fused
  int slices, colblocks;   // two-pass
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
  if (W > C) W = C;
  int64_t tpr = pgv_cdiv(W, 8);
  if (kind == 1) tpr = pgv_cdiv(W, F8B) * 16;
  const int64_t groups = pgv_cdiv(W, cg);
  static const int cfg[][2] = {{256, 1}, {256, 4}, {1024, 4}, {1024, 8}};
  if (groups <= MAXG)
    for (const auto& c : cfg) {
      if (kind == 2 && c[1] == 8) break;   // x and gy: twice the registers
      const int64_t rpp = c[0] / tpr;
      if (rpp >= 1 && P <= rpp * c[1]) {
        r.fused = true;
        r.W = (int)W;
        r.tpr = (int)tpr;
        r.nt = c[0];
        r.kv = c[1];
        r.colblocks = (int)pgv_cdiv(C, W);
        return r;
      }
    }
  r.W = (int)(C < 2048 ? C : 2048);
  r.tpr = (int)(kind == 1 ? pgv_cdiv(r.W, F8B) * 16 : pgv_cdiv(r.W, 8));
  r.colblocks = (int)pgv_cdiv(C, r.W);
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
  PGV_CHECK_ARG(N <= 65535 && P <= (1ll << 28) && C <= (1ll << 20), "%s: too large (items %lld, pixels %lld, channels %lld)", who,
                (long long)N, (long long)P, (long long)C);
  return PGV_OK;
}

template <typename T, bool VEC, bool Q, int FMT>
int gn_forward(gn_args p, const gn_plan& pl, hipStream_t st) {
  const bool same = p.cg % 8 == 0;
  p.W = pl.W;
  p.tpr = pl.tpr;
  p.slices = pl.slices;
  if (pl.fused) {
    const dim3 grid((unsigned)pl.colblocks, (unsigned)p.N);
#define PGV_F(NT, KV)                                                            \
  same ? gn_fwd_fused_kernel<T, NT, KV, VEC, Q, FMT, true><<<grid, NT, 0, st>>>(p) \
       : gn_fwd_fused_kernel<T, NT, KV, VEC, Q, FMT, false><<<grid, NT, 0, st>>>(p)
    if (pl.nt == 256)
      pl.kv == 1 ? (PGV_F(256, 1)) : (PGV_F(256, 4));
    else
      pl.kv == 4 ? (PGV_F(1024, 4)) : (PGV_F(1024, 8));
#undef PGV_F
    return PGV_OK;
  }
  const dim3 grid((unsigned)pl.slices, (unsigned)pl.colblocks, (unsigned)p.N);
  if (same)
    gn_stats_kernel<T, VEC, true><<<grid, 256, 0, st>>>(p);
  else
    gn_stats_kernel<T, VEC, false><<<grid, 256, 0, st>>>(p);
  gn_finalize_kernel<<<dim3((unsigned)p.G, (unsigned)p.N), 64, 0, st>>>(p, pl.slices * pl.colblocks);
  gn_apply_kernel<T, VEC, Q, FMT><<<grid, 256, 0, st>>>(p);
  return PGV_OK;
}

template <typename T, int NT, int KV, bool VEC>
int launch_bwd_fused(const gn_args& p, dim3 grid, hipStream_t st) {
  auto k = gn_bwd_fused_kernel<T, NT, KV, VEC>;
  constexpr int most = 3 * NT * 8 * (int)sizeof(float);   // W is at most 8 NT channels
  static const hipError_t once = hipFuncSetAttribute((const void*)k, hipFuncAttributeMaxDynamicSharedMemorySize, most);
  if (once != hipSuccess) {
    pgv_set_error("pgv_group_norm_act_bwd: %d bytes of LDS refused: %s", most, hipGetErrorString(once));
    return PGV_E_LAUNCH;
  }
  k<<<grid, NT, sizeof(float) * ((size_t)NT * 8 + 2 * (size_t)p.W), st>>>(p);
  return PGV_OK;
}

template <typename T, bool VEC>
int gn_backward(gn_args p, const gn_plan& pl, float* ggamma, float* gbeta, hipStream_t st) {
  p.W = pl.W;
  p.tpr = pl.tpr;
  p.slices = pl.fused ? 1 : pl.slices;
  if (pl.fused) {
    const dim3 grid((unsigned)pl.colblocks, (unsigned)p.N);
    const int rc = pl.nt == 1024 ? launch_bwd_fused<T, 1024, 4, VEC>(p, grid, st)
                   : pl.kv == 4  ? launch_bwd_fused<T, 256, 4, VEC>(p, grid, st)
                                 : launch_bwd_fused<T, 256, 1, VEC>(p, grid, st);
    if (rc != PGV_OK) return rc;
  } else {
    const dim3 grid((unsigned)pl.slices, (unsigned)pl.colblocks, (unsigned)p.N);
    gn_bwd_sums_kernel<T, VEC><<<grid, 256, 0, st>>>(p);
    gn_bwd_finalize_kernel<<<dim3((unsigned)p.G, (unsigned)p.N), 64, 0, st>>>(p);
    gn_bwd_apply_kernel<T, VEC><<<grid, 256, 0, st>>>(p);
  }
  if (ggamma || gbeta)
    gn_param_grads_kernel<<<dim3((unsigned)pgv_cdiv(p.C, 32)), 256, 0, st>>>(p.part, (int64_t)p.N * p.slices, p.C, ggamma, gbeta);
  return PGV_OK;
}

}  // namespace

extern "C" int64_t pgv_group_norm_workspace(int64_t N, int64_t P, int64_t C, int64_t G, int dtype, int kind) {
  if (N <= 0 || P <= 0 || C <= 0 || G <= 0 || C % G || !f8_dt_ok(dtype) || kind < 0 || kind > 2) return 0;
  const gn_plan pl = make_gn_plan(N, P, C, G, f8_dt_size(dtype), kind);
  if (kind == 2) return 4 * (pl.fused ? N * 2 * C : N * pl.slices * 2 * C + N * G * 2);
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
  p.N = (int)N, p.P = (int)P, p.C = (int)C, p.G = (int)G, p.cg = (int)(C / G);
  p.x = x, p.gamma = gamma, p.beta = beta, p.eps = eps, p.slope = slope, p.act = act;
  p.y = y, p.q = (uint8_t*)q, p.scale = scale, p.Kp = (int)(pgv_cdiv(C, F8B) * F8B);
  p.mean = mean, p.rstd = rstd;
  p.part = (float*)workspace;
  if (kind == 1 && !pl.fused) {
    float* tail = (float*)((char*)workspace + need - 8 * N * G);
    p.mean = tail, p.rstd = tail + N * G;
  }
  const bool vec = C % 8 == 0 && (uintptr_t)x % 16 == 0 && (q || (uintptr_t)y % 16 == 0);
  hipStream_t st = pgv_stream(stream);
  int r;
#define PGV_T(T, Q, FMT) (vec ? gn_forward<T, true, Q, FMT>(p, pl, st) : gn_forward<T, false, Q, FMT>(p, pl, st))
#define PGV_D(Q, FMT) (dtype == PGV_DT_F32 ? PGV_T(float, Q, FMT) : dtype == PGV_DT_BF16 ? PGV_T(__bf16, Q, FMT) : PGV_T(_Float16, Q, FMT))
  if (!q)
    r = PGV_D(false, PGV_F8_E4M3);
  else
    r = fmt == PGV_F8_E4M3 ? PGV_D(true, PGV_F8_E4M3) : PGV_D(true, PGV_F8_E5M2);
#undef PGV_D
#undef PGV_T
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
  p.N = (int)N, p.P = (int)P, p.C = (int)C, p.G = (int)G, p.cg = (int)(C / G);
  p.x = x, p.gy = gy, p.gx = gx, p.gamma = gamma, p.beta = beta, p.slope = slope, p.act = act;
  p.mean = const_cast<float*>(mean), p.rstd = const_cast<float*>(rstd);
  p.part = (float*)workspace;
  p.coef = pl.fused ? nullptr : p.part + N * pl.slices * 2 * C;
  const bool vec = C % 8 == 0 && (uintptr_t)x % 16 == 0 && (uintptr_t)gy % 16 == 0 && (uintptr_t)gx % 16 == 0;
  hipStream_t st = pgv_stream(stream);
#define PGV_T(T) (vec ? gn_backward<T, true>(p, pl, ggamma, gbeta, st) : gn_backward<T, false>(p, pl, ggamma, gbeta, st))
  const int r = dtype == PGV_DT_F32 ? PGV_T(float) : dtype == PGV_DT_BF16 ? PGV_T(__bf16) : PGV_T(_Float16);
#undef PGV_T
  if (r != PGV_OK) return r;
  PGV_CHECK_LAUNCH("pgv_group_norm_act_bwd");
  return PGV_OK;
}
