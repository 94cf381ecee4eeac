// Launches of the residual step's backward for one storage type, from the
// tensors (Q8 false) or from their 8-bit copies.
#pragma once

#include <algorithm>

#include "resnorm_rows.cuh"

namespace nblahip {

template <typename T, bool LN, bool POST, bool PRE, bool Q8, int MODE>
bool launch_bwd_rows(const StepPlan &pl, const StepArgs &a, hipStream_t st) {
#define NBLAHIP_CASE(TPR, NV)                                                                     \
  if (pl.tpr == TPR && pl.nv == NV) {                                                             \
    if constexpr (bwd_row_fits(Tok<T>::VEC, LN, POST, PRE, Q8, MODE, TPR, NV) &&                  \
                  !(NV > 1 && MODE == kRagged)) {                                                 \
      NBLAHIP_LAUNCH("step_bwd_rows_kernel",                                                      \
                     (step_bwd_rows_kernel<T, LN, POST, PRE, Q8, MODE, TPR, NV>),                 \
                     dim3(static_cast<unsigned>(a.grid)), dim3(bwd_block(TPR)), 0, st, a);        \
      return true;                                                                                \
    }                                                                                             \
  }
  NBLAHIP_STEP_LAYOUTS(NBLAHIP_CASE)
#undef NBLAHIP_CASE
  return false;
}

template <typename T, bool LN, bool POST, bool PRE, bool Q8>
int launch_bwd_kind(const StepPlan &pl, const StepArgs &a, hipStream_t st) {
  if (pl.tpr != 0) {
    const bool known = pl.mode == kWhole    ? launch_bwd_rows<T, LN, POST, PRE, Q8, kWhole>(pl, a, st)
                       : pl.mode == kRagged ? launch_bwd_rows<T, LN, POST, PRE, Q8, kRagged>(pl, a, st)
                                            : launch_bwd_rows<T, LN, POST, PRE, Q8, kAny>(pl, a, st);
    return known ? last_launch_status() : NBLAHIP_EINVAL; // (the workspace is not the long rows')
  }
  const dim3 rows(static_cast<unsigned>(std::min<int64_t>(a.rows, 1 << 20)));
  NBLAHIP_LAUNCH("step_bwd_long_sums_kernel", (step_bwd_long_sums_kernel<T, LN, POST, PRE, Q8>), rows,
                 dim3(kLongThreads), 0, st, a);
  if (const int e = last_launch_status()) return e;
  const int64_t span = static_cast<int64_t>(kLongThreads) * Tok<T>::VEC;
  const dim3 tiles(static_cast<unsigned>((a.pitch + span - 1) / span),
                   static_cast<unsigned>(std::min<int64_t>(a.chunks, 65535)));
  NBLAHIP_LAUNCH("step_bwd_long_cols_kernel", (step_bwd_long_cols_kernel<T, LN, POST, PRE, Q8>), tiles,
                 dim3(kLongThreads), 0, st, a);
  return last_launch_status();
}

template <typename T, bool LN, bool Q8>
int launch_bwd_norms(const StepPlan &pl, const StepArgs &a, hipStream_t st) {
  if (pl.post && pl.pre) return launch_bwd_kind<T, LN, true, true, Q8>(pl, a, st);
  if (pl.post) return launch_bwd_kind<T, LN, true, false, Q8>(pl, a, st);
  return launch_bwd_kind<T, LN, false, true, Q8>(pl, a, st);
}

template <typename T, bool Q8> int launch_bwd(const StepPlan &pl, const StepArgs &a, hipStream_t st) {
  return pl.layer ? launch_bwd_norms<T, true, Q8>(pl, a, st) : launch_bwd_norms<T, false, Q8>(pl, a, st);
}

} // namespace nblahip
