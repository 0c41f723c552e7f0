// Distillation kernels for f32 logits.
#include "distill_device.hpp"

namespace pcp {

hipError_t launch_distill_f32(const DistillArgs& a, bool f32_out, hipStream_t st) {
  (void)f32_out;
  return launch_pair<F32T, F32T>(a, st);
}

}  // namespace pcp
