// Distillation kernels for bf16 logits.
#include "distill_device.hpp"

namespace pcp {

hipError_t launch_distill_bf16(const DistillArgs& a, bool f32_out, hipStream_t st) {
  return f32_out ? launch_pair<BF16T, F32T>(a, st) : launch_pair<BF16T, BF16T>(a, st);
}

}  // namespace pcp
