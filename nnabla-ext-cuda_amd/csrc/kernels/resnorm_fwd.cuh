// Launches of the residual step's forward for one storage type.
#pragma once

#include <algorithm>

#include "resnorm_long.cuh"

namespace nblahip {

template <typename T, bool LN, bool POST, bool PRE>
int launch_fwd_kind(const StepPlan &pl, const StepArgs &a, hipStream_t st) {
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
