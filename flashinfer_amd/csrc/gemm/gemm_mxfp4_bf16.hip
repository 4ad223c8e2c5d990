// Products with MXFP4 weights: the kernels for bf16 activations.
#include "fi/mxfp4_body.hpp"

namespace fi {
namespace mx4 {

hipError_t launch_bf16(int gated, const Plan& plan, const Params& p, hipStream_t stream) {
  return launch_act<kBf16>(gated, plan, p, stream);
}

}  // namespace mx4
}  // namespace fi
