// The linear map and the gated projection in bf16.
#include "ops_linear.cuh"

namespace t8b {
namespace op {
template void linear_forward<bf16>(const LinearCall&);
template void linear_backward<bf16>(const LinearGradCall&);
}  // namespace op
}  // namespace t8b
