// The residual join's kernels for an x of type f32 (residual_norm.cuh).
#include "residual_norm.cuh"

namespace sca2 {
namespace rnorm {

cudaError_t fwd_f32(const Args& a, int udt, bool vec, cudaStream_t st) {
  return udt == SCA2_BF16 ? fwd_types<float, __nv_bfloat16>(a, vec, st) : fwd_types<float, float>(a, vec, st);
}
cudaError_t bwd_f32(const Args& a, int udt, bool contig, cudaStream_t st) {
  return udt == SCA2_BF16 ? bwd_types<float, __nv_bfloat16>(a, contig, st) : bwd_types<float, float>(a, contig, st);
}

}  // namespace rnorm
}  // namespace sca2
