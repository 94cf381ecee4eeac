#include "resnorm_fwd.cuh"

namespace nblahip {
int launch_step_fwd_f16(const StepPlan &pl, const StepArgs &a, hipStream_t st) {
  return launch_fwd<__half>(pl, a, st);
}
} // namespace nblahip
