// The selective scan in bf16.
#include "ops_scan.cuh"

namespace t8b {
namespace op {
namespace scan {
template void launch_forward<bf16>(const Call&, const ForwardPlan&, int64_t, cudaStream_t);
template void launch_backward<bf16>(const Call&, const BackwardPlan&, float*, float*, float*, cudaStream_t);
template void launch_step<bf16>(const Call&, float*, bool, cudaStream_t);
}  // namespace scan
}  // namespace op
}  // namespace t8b
