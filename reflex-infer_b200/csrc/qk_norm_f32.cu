// The f32 kernels of qk_norm.cuh.
#include "qk_norm.cuh"

namespace rfx {
namespace qkn {
cudaError_t launch_f32(const QkNormParams& P, const Shape& s, cudaStream_t stream) { return launch_type<float>(P, s, stream); }
}  // namespace qkn
}  // namespace rfx
