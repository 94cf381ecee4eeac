#include "resnorm_fwd.cuh"

namespace nblahip {
int launch_step_fwd_bf16(const StepPlan &pl, const StepArgs &a, hipStream_t st) {
  return launch_fwd<bf16>(pl, a, st);
}
} // namespace nblahip
