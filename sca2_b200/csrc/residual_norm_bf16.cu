// The residual join's kernels for an x of type bf16 (residual_norm.cuh).
#include "residual_norm.cuh"

namespace sca2 {
namespace rnorm {

cudaError_t fwd_bf16(const Args& a, int udt, bool vec, cudaStream_t st) {
  return udt == SCA2_BF16 ? fwd_types<__nv_bfloat16, __nv_bfloat16>(a, vec, st) : fwd_types<__nv_bfloat16, float>(a, vec, st);
}
cudaError_t bwd_bf16(const Args& a, int udt, bool contig, cudaStream_t st) {
  return udt == SCA2_BF16 ? bwd_types<__nv_bfloat16, __nv_bfloat16>(a, contig, st) : bwd_types<__nv_bfloat16, float>(a, contig, st);
}

}  // namespace rnorm
}  // namespace sca2
