// The residual join's kernels for x of type f32 and u of type f32 (residual_norm.cuh).
#include "residual_norm.cuh"

namespace sca2 {
namespace rnorm {

cudaError_t fwd_f32_f32(const Args& a, bool vec, cudaStream_t st) { return fwd_types<float, float>(a, vec, st); }
cudaError_t bwd_f32_f32(const Args& a, bool contig, cudaStream_t st) { return bwd_types<float, float>(a, contig, st); }

}  // namespace rnorm
}  // namespace sca2
