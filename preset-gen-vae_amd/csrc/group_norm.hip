// GroupNorm + activation: the C entry points, which scheme serves a call, and the forward pass (kernels: group_norm_fwd.h).
#include "group_norm_fwd.h"

namespace {

// ---- which scheme: a function of the sizes and the element size -----------------------------------------------------------
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

}  // namespace

int pgv_gn_forward(const gn_args& p, const gn_plan& pl, int dtype, bool vec, hipStream_t st) {
  const bool same = p.cg % 8 == 0;
#define PGV_V(T, VEC) (same ? gn_forward<T, VEC, false, 0, true>(p, pl, st) : gn_forward<T, VEC, false, 0, false>(p, pl, st))
#define PGV_T(T) (vec ? PGV_V(T, true) : PGV_V(T, false))
  return dtype == PGV_DT_F32 ? PGV_T(float) : dtype == PGV_DT_BF16 ? PGV_T(__bf16) : PGV_T(_Float16);
#undef PGV_T
#undef PGV_V
}

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
  const int r = q ? pgv_gn_forward_f8(p, pl, dtype, vec, fmt, st) : pgv_gn_forward(p, pl, dtype, vec, st);
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
  const int r = pgv_gn_backward(p, pl, dtype, vec, ggamma, gbeta, pgv_stream(stream));
  if (r != PGV_OK) return r;
  PGV_CHECK_LAUNCH("pgv_group_norm_act_bwd");
  return PGV_OK;
}
