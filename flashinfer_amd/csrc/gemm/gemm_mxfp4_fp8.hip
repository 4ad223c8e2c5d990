// Products with MXFP4 weights: the kernels for MXFP8 activations.
#include "fi/mxfp4_body.hpp"

namespace fi {
namespace mx4 {

hipError_t launch_fp8(int gated, const Plan& plan, const Params& p, hipStream_t stream) {
  return launch_act<kFp8>(gated, plan, p, stream);
}

}  // namespace mx4
}  // namespace fi
