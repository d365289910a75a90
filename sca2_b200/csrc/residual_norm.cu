// Entry points of the residual join with norms, and the sum over the backward's partial parameter
// gradients.  The kernels are in residual_norm.cuh.
#include <string>

#include "residual_norm.cuh"

namespace sca2 {
void set_last_error(const std::string& msg);

namespace rnorm {

struct Outs {
  float* p[NPART];
};

// column sums of the CTAs' partials, 32 columns to a CTA, the partial rows over its 16 warps
constexpr int RW = 16;
__global__ void __launch_bounds__(32 * RW) reduce_kernel(const float* __restrict__ part, int nparts, int d, const Outs o) {
  __shared__ float s[RW][32];
  float* out = o.p[blockIdx.y];
  if (!out) return;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  float v = 0.f;
  if (c < d) {
#pragma unroll 8
    for (int i = w; i < nparts; i += RW) v += part[((int64_t)i * NPART + blockIdx.y) * d + c];
  }
  s[w][lane] = v;
  __syncthreads();
  if (w == 0 && c < d) {
#pragma unroll
    for (int k = 1; k < RW; ++k) v += s[k][lane];
    out[c] = v;
  }
}

int fail(int code, const char* msg) {
  set_last_error(msg);
  return code;
}
int cuda_fail(cudaError_t e, const char* where) {
  set_last_error(std::string(where) + ": " + cudaGetErrorString(e));
  return SCA2_ERR_CUDA;
}

int check(const sca2_rnorm_args* a) {
  if (!a) return fail(SCA2_ERR_ARG, "residual_norm: null argument struct");
  if (a->rows < 0 || a->d < 1) return fail(SCA2_ERR_ARG, "residual_norm: bad sizes");
  if (a->d > SCA2_RNORM_MAX_D) return fail(SCA2_ERR_UNSUPPORTED, "residual_norm: rows wider than 4096 are not supported");
  for (int t : {a->x_dtype, a->u_dtype, a->z_dtype})
    if (t != SCA2_F32 && t != SCA2_BF16) return fail(SCA2_ERR_ARG, "residual_norm: types are SCA2_F32 or SCA2_BF16");
  if (a->kind != SCA2_NORM_LAYER && a->kind != SCA2_NORM_RMS)
    return fail(SCA2_ERR_ARG, "residual_norm: kind must be SCA2_NORM_LAYER or SCA2_NORM_RMS");
  if (a->gate_mode < 0 || a->gate_mode > 2) return fail(SCA2_ERR_ARG, "residual_norm: gate_mode must be 0, 1 or 2");
  if (!(a->eps >= 0.f)) return fail(SCA2_ERR_ARG, "residual_norm: eps must be >= 0");
  if ((a->b && !a->w) || (a->pb && !a->pw)) return fail(SCA2_ERR_ARG, "residual_norm: a bias needs its weight");
  if (a->kind == SCA2_NORM_RMS && (a->b || a->pb)) return fail(SCA2_ERR_ARG, "residual_norm: the RMS norm has no bias");
  if (a->rows == 0) return SCA2_OK;
  if (!a->x || !a->u) return fail(SCA2_ERR_ARG, "residual_norm: x and u must be non-null");
  if (a->sx < a->d || a->su < a->d || (a->gate_mode == 2 && a->sg < a->d) || (a->gate_mode == 1 && a->sg < 1))
    return fail(SCA2_ERR_ARG, "residual_norm: a row stride is smaller than the row");
  if (a->gate_mode && !a->gate) return fail(SCA2_ERR_ARG, "residual_norm: gate_mode needs a gate");
  return SCA2_OK;
}

bool on(int align, std::initializer_list<const void*> ps) {
  uintptr_t u = 0;
  for (const void* p : ps) u |= reinterpret_cast<uintptr_t>(p);
  return u % align == 0;
}
bool strides(const sca2_rnorm_args& a, int m) {
  return a.d % m == 0 && a.sx % m == 0 && a.su % m == 0 && (a.gate_mode != 2 || a.sg % m == 0);
}

Args args(const sca2_rnorm_args& a) {
  Args k{};
  k.x = a.x, k.u = a.u, k.gate = a.gate_mode ? a.gate : nullptr;
  k.sx = a.sx, k.su = a.su, k.sg = a.sg;
  k.w = a.w, k.b = a.b, k.pw = a.pw, k.pb = a.pb, k.scale = a.scale;
  k.rows = a.rows, k.d = a.d, k.eps = a.eps;
  k.rms = a.kind == SCA2_NORM_RMS, k.gate_mode = a.gate_mode, k.zdt = a.z_dtype;
  return k;
}

}  // namespace rnorm
}  // namespace sca2

using namespace sca2::rnorm;

extern "C" {

int sca2_residual_norm_fwd(const sca2_rnorm_args* a, void* y, void* z, float* stats, void* stream) {
  if (int rc = check(a)) return rc;
  if (z && !a->w) return fail(SCA2_ERR_ARG, "residual_norm: z needs its weight");
  if (a->rows == 0) return SCA2_OK;
  if (!y) return fail(SCA2_ERR_ARG, "residual_norm: y must be non-null");
  if (!on(16, {stats})) return fail(SCA2_ERR_ARG, "residual_norm: stats must be 16-byte aligned");
  Args k = args(*a);
  k.y = y, k.z = z, k.stats = stats;
  const bool vec = strides(*a, 4) && on(16, {k.x, k.u, k.gate_mode == 2 ? k.gate : nullptr, y, z, k.w, k.b, k.pw, k.pb, k.scale});
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const auto f = a->x_dtype == SCA2_BF16 ? (a->u_dtype == SCA2_BF16 ? fwd_bf16_bf16 : fwd_bf16_f32)
                                         : (a->u_dtype == SCA2_BF16 ? fwd_f32_bf16 : fwd_f32_f32);
  const cudaError_t e = f(k, vec, st);
  return e == cudaSuccess ? SCA2_OK : cuda_fail(e, "sca2_residual_norm_fwd");
}

int64_t sca2_residual_norm_work_bytes(int64_t rows, int32_t d) {
  return rows > 0 && d > 0 && d <= SCA2_RNORM_MAX_D ? (int64_t)bwd_grid(rows, d) * NPART * d * 4 : 0;
}

int sca2_residual_norm_bwd(const sca2_rnorm_args* a, const float* stats, const void* dy, const void* dz,
                           const sca2_rnorm_grads* g, void* work, int64_t work_bytes, void* stream) {
  if (int rc = check(a)) return rc;
  if (!g) return fail(SCA2_ERR_ARG, "residual_norm: null gradient struct");
  if (dz && !a->w) return fail(SCA2_ERR_ARG, "residual_norm: dz needs the weight of z");
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  Outs o{{a->w ? g->dw : nullptr, a->b ? g->db : nullptr, a->scale ? g->dscale : nullptr, a->pw ? g->dpw : nullptr,
          a->pb ? g->dpb : nullptr}};
  const bool none = a->rows == 0;
  if (none || !dz) {  // gradients that nothing reaches
    for (int i = 0; i < (none ? NPART : 2); ++i) {
      if (o.p[i])
        if (cudaError_t e = cudaMemsetAsync(o.p[i], 0, (size_t)a->d * 4, st)) return cuda_fail(e, "sca2_residual_norm_bwd");
      o.p[i] = nullptr;
    }
    if (none) return SCA2_OK;
  }
  if (!stats || !on(16, {stats})) return fail(SCA2_ERR_ARG, "residual_norm: stats must be non-null and 16-byte aligned");
  if (!g->dx || !g->du || (a->gate_mode && !g->dgate)) return fail(SCA2_ERR_ARG, "residual_norm: null gradient buffer");
  if (!work || !on(16, {work}) || work_bytes < sca2_residual_norm_work_bytes(a->rows, a->d))
    return fail(SCA2_ERR_ARG, "residual_norm: workspace null, misaligned or too small");
  Args k = args(*a);
  k.stats = const_cast<float*>(stats);
  k.dy = dy, k.dz = dz, k.dx = g->dx, k.du = g->du, k.dgate = g->dgate, k.part = static_cast<float*>(work);
  const bool contig = strides(*a, 4) && on(16, {k.x, k.u, k.gate_mode == 2 ? k.gate : nullptr, dy, dz, k.dx, k.du,
                                                k.gate_mode == 2 ? k.dgate : nullptr, k.w, k.b, k.pw, k.pb, k.scale});
  const auto f = a->x_dtype == SCA2_BF16 ? (a->u_dtype == SCA2_BF16 ? bwd_bf16_bf16 : bwd_bf16_f32)
                                         : (a->u_dtype == SCA2_BF16 ? bwd_f32_bf16 : bwd_f32_f32);
  cudaError_t e = f(k, contig, st);
  if (e == cudaSuccess && (o.p[0] || o.p[1] || o.p[2] || o.p[3] || o.p[4])) {
    reduce_kernel<<<dim3((a->d + 31) / 32, NPART), 32 * RW, 0, st>>>(k.part, bwd_grid(a->rows, a->d), a->d, o);
    e = cudaGetLastError();
  }
  return e == cudaSuccess ? SCA2_OK : cuda_fail(e, "sca2_residual_norm_bwd");
}

}  // extern "C"
