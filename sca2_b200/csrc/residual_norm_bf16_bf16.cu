// The residual join's kernels for x of type bf16 and u of type bf16 (residual_norm.cuh).
#include "residual_norm.cuh"

namespace sca2 {
namespace rnorm {

cudaError_t fwd_bf16_bf16(const Args& a, bool vec, cudaStream_t st) { return fwd_types<__nv_bfloat16, __nv_bfloat16>(a, vec, st); }
cudaError_t bwd_bf16_bf16(const Args& a, bool contig, cudaStream_t st) { return bwd_types<__nv_bfloat16, __nv_bfloat16>(a, contig, st); }

}  // namespace rnorm
}  // namespace sca2
