// Launches of the residual step's forward for one storage type.
#pragma once

#include <algorithm>

#include "resnorm_rows.cuh"

namespace nblahip {

template <typename T, bool LN, bool POST, bool PRE, bool COPY, int MODE>
bool launch_fwd_rows(const StepPlan &pl, const StepArgs &a, hipStream_t st) {
#define NBLAHIP_CASE(TPR, NV)                                                                     \
  if (pl.tpr == TPR && pl.nv == NV) {                                                             \
    if constexpr (fwd_row_fits(Tok<T>::VEC, LN, POST, PRE, COPY, MODE, NV) && !(NV > 1 && MODE == kRagged)) { \
      NBLAHIP_LAUNCH("step_fwd_rows_kernel",                                                      \
                     (step_fwd_rows_kernel<T, LN, POST, PRE, COPY, MODE, TPR, NV>),               \
                     dim3(static_cast<unsigned>(a.grid)), dim3(fwd_block(TPR)), 0, st, a);        \
      return true;                                                                                \
    }                                                                                             \
  }
  NBLAHIP_STEP_LAYOUTS(NBLAHIP_CASE)
#undef NBLAHIP_CASE
  return false;
}

template <typename T, bool LN, bool POST, bool PRE>
int launch_fwd_kind(const StepPlan &pl, const StepArgs &a, hipStream_t st) {
  const bool copy = a.x8 || a.h8;
  if (pl.tpr != 0) {
    const bool known =
        pl.mode == kWhole ? copy ? launch_fwd_rows<T, LN, POST, PRE, true, kWhole>(pl, a, st)
                                 : launch_fwd_rows<T, LN, POST, PRE, false, kWhole>(pl, a, st)
        : copy                   ? launch_fwd_rows<T, LN, POST, PRE, true, kAny>(pl, a, st)
        : pl.mode == kRagged     ? launch_fwd_rows<T, LN, POST, PRE, false, kRagged>(pl, a, st)
                                 : launch_fwd_rows<T, LN, POST, PRE, false, kAny>(pl, a, st);
    return known ? last_launch_status() : NBLAHIP_EINVAL;
  }
  const dim3 grid(static_cast<unsigned>(std::min<int64_t>(a.rows, 1 << 20)));
  NBLAHIP_LAUNCH("step_fwd_long_kernel", (step_fwd_long_kernel<T, LN, POST, PRE>), grid,
                 dim3(kLongThreads), 0, st, a);
  return last_launch_status();
}

template <typename T> int launch_fwd(const StepPlan &pl, const StepArgs &a, hipStream_t st) {
  if (pl.layer) {
    if (pl.post && pl.pre) return launch_fwd_kind<T, true, true, true>(pl, a, st);
    if (pl.post) return launch_fwd_kind<T, true, true, false>(pl, a, st);
    return launch_fwd_kind<T, true, false, true>(pl, a, st);
  }
  if (pl.post && pl.pre) return launch_fwd_kind<T, false, true, true>(pl, a, st);
  if (pl.post) return launch_fwd_kind<T, false, true, false>(pl, a, st);
  return launch_fwd_kind<T, false, false, true>(pl, a, st);
}

} // namespace nblahip
