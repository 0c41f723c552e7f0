// Distillation kernels for f16 logits.
#include "distill_device.hpp"

namespace pcp {

hipError_t launch_distill_f16(const DistillArgs& a, bool f32_out, hipStream_t st) {
  return f32_out ? launch_pair<F16T, F32T>(a, st) : launch_pair<F16T, F16T>(a, st);
}

}  // namespace pcp
