// Backward pass of GroupNorm + activation.
#include "group_norm_common.h"

namespace {

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

int pgv_gn_backward(const gn_args& p, const gn_plan& pl, int dtype, bool vec, float* ggamma, float* gbeta, hipStream_t st) {
  const bool same = p.cg % 8 == 0;
#define PGV_V(T, VEC) (same ? gn_backward<T, VEC, true>(p, pl, ggamma, gbeta, st) : gn_backward<T, VEC, false>(p, pl, ggamma, gbeta, st))
#define PGV_T(T) (vec ? PGV_V(T, true) : PGV_V(T, false))
  return dtype == PGV_DT_F32 ? PGV_T(float) : dtype == PGV_DT_BF16 ? PGV_T(__bf16) : PGV_T(_Float16);
#undef PGV_T
#undef PGV_V
}
