// Forward kernels of GroupNorm + activation, into values or into 8-bit blocks.
#pragma once
#include "group_norm_common.h"

namespace {

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

}  // namespace
