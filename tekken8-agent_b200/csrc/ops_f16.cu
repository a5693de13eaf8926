// The linear map and the gated projection in f16.
#include "ops_linear.cuh"

namespace t8b {
namespace op {
template void linear_forward<f16>(const LinearCall&);
template void linear_backward<f16>(const LinearGradCall&);
}  // namespace op
}  // namespace t8b
