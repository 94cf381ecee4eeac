#include "resnorm_bwd.cuh"

namespace nblahip {
int launch_step_bwd8_f32(const StepPlan &pl, const StepArgs &a, hipStream_t st) {
  return launch_bwd<float, true>(pl, a, st);
}
} // namespace nblahip
