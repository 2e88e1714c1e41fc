// Kernels of the logits head for one type of hidden states (a translation unit per type: they compile side by side).
#include "ets_head_launch.h"

namespace ets_host {

hipError_t launch_head_f16(const ets::HeadParams& p, const HeadForm& f, hipStream_t stream) {
  return launch_head<ets::kDtypeHalf>(p, f, stream);
}

}  // namespace ets_host
