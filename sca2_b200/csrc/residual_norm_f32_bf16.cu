// The residual join's kernels for x of type f32 and u of type bf16 (residual_norm.cuh).
#include "residual_norm.cuh"

namespace sca2 {
namespace rnorm {

cudaError_t fwd_f32_bf16(const Args& a, bool vec, cudaStream_t st) { return fwd_types<float, __nv_bfloat16>(a, vec, st); }
cudaError_t bwd_f32_bf16(const Args& a, bool contig, cudaStream_t st) { return bwd_types<float, __nv_bfloat16>(a, contig, st); }

}  // namespace rnorm
}  // namespace sca2
