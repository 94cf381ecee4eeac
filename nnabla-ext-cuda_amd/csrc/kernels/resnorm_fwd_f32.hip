#include "resnorm_fwd.cuh"

namespace nblahip {
int launch_step_fwd_f32(const StepPlan &pl, const StepArgs &a, hipStream_t st) {
  return launch_fwd<float>(pl, a, st);
}
} // namespace nblahip
