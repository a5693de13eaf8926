// The selective scan in fp32.
#include "ops_scan.cuh"

namespace t8b {
namespace op {
namespace scan {
template void launch_forward<float>(const Call&, const ForwardPlan&, int64_t, cudaStream_t);
template void launch_backward<float>(const Call&, const BackwardPlan&, float*, float*, float*, cudaStream_t);
template void launch_step<float>(const Call&, float*, bool, cudaStream_t);
}  // namespace scan
}  // namespace op
}  // namespace t8b
