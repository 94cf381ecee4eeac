#include "resnorm_bwd.cuh"

namespace nblahip {
int launch_step_bwd_bf16(const StepPlan &pl, const StepArgs &a, hipStream_t st) {
  return launch_bwd<bf16, false>(pl, a, st);
}
} // namespace nblahip
