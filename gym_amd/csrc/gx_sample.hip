// Actions from a policy's logits, binary32 logits and the choice of the type (see gx_sample_kernel.h; a translation unit a
// type, so that they compile side by side).
#include "gx_sample_kernel.h"

namespace gx {

hipError_t launch_sample_f16(const SampleArgs& a, void* workspace, int num_cus, hipStream_t stream);
hipError_t launch_sample_bf16(const SampleArgs& a, void* workspace, int num_cus, hipStream_t stream);

size_t sample_workspace(const SampleArgs& a, int num_cus) { return a.rows && split_parts(a, num_cus) > 1 ? a.rows * sizeof(SplitRow) : 0; }

hipError_t launch_sample_logits(const SampleArgs& a, int dtype, void* workspace, int num_cus, hipStream_t stream) {
  if (dtype == GX_F16) return launch_sample_f16(a, workspace, num_cus, stream);
  if (dtype == GX_BF16) return launch_sample_bf16(a, workspace, num_cus, stream);
  return launch_sample_typed<float>(a, static_cast<SplitRow*>(workspace), num_cus, stream);
}

}  // namespace gx
