// Launches of the residual step's backward for one storage type.
#pragma once

#include <algorithm>

#include "resnorm_long.cuh"

namespace nblahip {

template <typename T, bool LN, bool POST, bool PRE, bool Q8>
int launch_bwd_kind(const StepPlan &pl, const StepArgs &a, hipStream_t st) {
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

template <typename T> int launch_bwd(const StepPlan &pl, const StepArgs &a, hipStream_t st) {
  if (pl.layer)
    return pl.kept8 ? launch_bwd_norms<T, true, true>(pl, a, st) : launch_bwd_norms<T, true, false>(pl, a, st);
  return pl.kept8 ? launch_bwd_norms<T, false, true>(pl, a, st) : launch_bwd_norms<T, false, false>(pl, a, st);
}

} // namespace nblahip
