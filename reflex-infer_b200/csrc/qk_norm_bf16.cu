// The bf16 kernels of qk_norm.cuh.
#include "qk_norm.cuh"

namespace rfx {
namespace qkn {
cudaError_t launch_bf16(const QkNormParams& P, const Shape& s, cudaStream_t stream) { return launch_type<__nv_bfloat16>(P, s, stream); }
}  // namespace qkn
}  // namespace rfx
