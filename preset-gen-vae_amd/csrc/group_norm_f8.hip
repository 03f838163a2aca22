// GroupNorm + activation into 8-bit blocks (kernels: group_norm_fwd.h).
#include "group_norm_fwd.h"

int pgv_gn_forward_f8(const gn_args& p, const gn_plan& pl, int dtype, bool vec, int fmt, hipStream_t st) {
  const bool same = p.cg % 8 == 0;
#define PGV_V(T, VEC, FMT) (same ? gn_forward<T, VEC, true, FMT, true>(p, pl, st) : gn_forward<T, VEC, true, FMT, false>(p, pl, st))
#define PGV_T(T, FMT) (vec ? PGV_V(T, true, FMT) : PGV_V(T, false, FMT))
#define PGV_D(FMT) (dtype == PGV_DT_F32 ? PGV_T(float, FMT) : dtype == PGV_DT_BF16 ? PGV_T(__bf16, FMT) : PGV_T(_Float16, FMT))
  return fmt == PGV_F8_E4M3 ? PGV_D(PGV_F8_E4M3) : PGV_D(PGV_F8_E5M2);
#undef PGV_D
#undef PGV_T
#undef PGV_V
}
