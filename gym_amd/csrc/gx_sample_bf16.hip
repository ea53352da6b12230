#include "gx_sample_kernel.h"

namespace gx {

hipError_t launch_sample_bf16(const SampleArgs& a, void* workspace, int num_cus, hipStream_t stream) {
  return launch_sample_typed<bf16>(a, static_cast<SplitRow*>(workspace), num_cus, stream);
}

}  // namespace gx
