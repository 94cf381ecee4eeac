#include "resnorm_bwd.cuh"

namespace nblahip {
int launch_step_bwd8_bf16(const StepPlan &pl, const StepArgs &a, hipStream_t st) {
  return launch_bwd<bf16, true>(pl, a, st);
}
} // namespace nblahip
