// Global gradient norm over a list of tensors, and clipping to a largest norm:
//
//     norm = sqrt(sum_i sum_j g_i[j]^2),   out_i = g_i * min(1, max_norm / (norm + 1e-6))
//
// (the semantics of torch.nn.utils.clip_grad_norm_).  Two launches: `norm_kernel` leaves one
// partial sum of squares per CTA, `clip_kernel` adds the partials (every CTA in the same order,
// so the norm has one value and does not depend on the schedule) and writes the scaled values.
//
// Bound by memory: the values are read twice (the factor depends on all of them) and written
// once.  The tensor table travels in the kernel's parameters, so a call makes no copy to the
// device and its capture in a CUDA graph holds the addresses by value.  The chunks of all
// tensors form one sequence, of which every CTA takes a contiguous range (one search for its
// first tensor, then a walk), whatever the tensors' sizes.
#include <algorithm>
#include <string>
#include <vector>

#include "common.cuh"

namespace sca2 {
void set_last_error(const std::string& msg);

namespace clip {

constexpr int NT = 256;
constexpr int CHUNK = 4096;          // values of one chunk; 16 of each thread
constexpr int CTAS_PER_SM = 4;

struct Entry {
  const void* src;
  void* dst;
  int64_t n;
  int32_t first;      // its first chunk in the launch's sequence
  int16_t sdt, ddt;   // SCA2_F32 or SCA2_BF16
};

// The launch's tensors.  Kernel parameters hold up to 32 764 bytes: 1000 entries, or 100 where
// they suffice (the parameters are copied at each launch).
template <int N>
struct Table {
  int32_t count, chunks;
  Entry e[N];
};

template <int N>
__device__ __forceinline__ int find(const Table<N>& t, int chunk) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {  // last entry whose first chunk is <= chunk
    const int mid = (lo + hi + 1) >> 1;
    if (t.e[mid].first <= chunk) lo = mid; else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

__device__ __forceinline__ float2 unpack(uint32_t u) {
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u));
}

// f(j, v) for the 16 values of this thread in the chunk [c0, c0 + CHUNK) of a tensor of n values
// that lies on a 16-byte boundary and has the whole chunk: group k of 4 (fp32) or 8 (bf16) consecutive values.
template <class F>
__device__ __forceinline__ void vec_f32(const float* p, F f) {
  float4 q[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) q[k] = reinterpret_cast<const float4*>(p)[threadIdx.x + NT * k];
#pragma unroll
  for (int k = 0; k < 4; ++k) f(4 * (threadIdx.x + NT * k), q[k]);
}
template <class F>
__device__ __forceinline__ void vec_bf16(const __nv_bfloat16* p, F f) {
  uint4 q[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) q[k] = reinterpret_cast<const uint4*>(p)[threadIdx.x + NT * k];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int j = 8 * (threadIdx.x + NT * k);
    const float2 a = unpack(q[k].x), b = unpack(q[k].y), c = unpack(q[k].z), d = unpack(q[k].w);
    f(j, make_float4(a.x, a.y, b.x, b.y));
    f(j + 4, make_float4(c.x, c.y, d.x, d.y));
  }
}

// the sum of `v` over the CTA, in thread 0 (fixed order)
__device__ __forceinline__ double cta_sum(double v) {
  __shared__ double s[NT / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  if (threadIdx.x == 0)
    for (int w = 1; w < NT / 32; ++w) v += s[w];
  return v;
}

// Squares and sums are taken in 64 bits: in 32 a gradient above 1.8e19 or below 1e-23 would
// overflow or vanish although its norm is an fp32 number.
template <int N>
__global__ void __launch_bounds__(NT) norm_kernel(const __grid_constant__ Table<N> t, double* __restrict__ part) {
  const int64_t c0 = (int64_t)t.chunks * blockIdx.x / gridDim.x, c1 = (int64_t)t.chunks * (blockIdx.x + 1) / gridDim.x;
  double s0 = 0., s1 = 0., s2 = 0., s3 = 0.;
  int ti = find(t, (int)c0);
  for (int64_t c = c0; c < c1; ++c) {
    while (ti + 1 < t.count && t.e[ti + 1].first <= c) ++ti;
    const Entry& e = t.e[ti];
    const int64_t at = (c - e.first) * CHUNK;
    const int64_t left = e.n - at;
    const auto add = [&](int, float4 q) {
      s0 = fma((double)q.x, (double)q.x, s0), s1 = fma((double)q.y, (double)q.y, s1);
      s2 = fma((double)q.z, (double)q.z, s2), s3 = fma((double)q.w, (double)q.w, s3);
    };
    if (left >= CHUNK && aligned16(e.src)) {
      if (e.sdt == SCA2_F32) vec_f32(reinterpret_cast<const float*>(e.src) + at, add);
      else vec_bf16(reinterpret_cast<const __nv_bfloat16*>(e.src) + at, add);
    } else {
      const int m = (int)(left < CHUNK ? left : CHUNK);
#pragma unroll 4
      for (int j = threadIdx.x; j < m; j += NT) {
        const double v = ld_io(e.src, at + j, e.sdt);
        s0 = fma(v, v, s0);
      }
    }
  }
  const double s = cta_sum((s0 + s1) + (s2 + s3));
  if (threadIdx.x == 0) part[blockIdx.x] = s;
}

// the norm from the partials of every launch, the same in all threads of all CTAs
__device__ __forceinline__ float total_norm(const double* __restrict__ part, int nparts) {
  __shared__ float out;
  double v = 0.;
  for (int i = threadIdx.x; i < nparts; i += NT) v += part[i];
  v = cta_sum(v);
  if (threadIdx.x == 0) out = (float)sqrt(v);
  __syncthreads();
  return out;
}

template <int N>
__global__ void __launch_bounds__(NT) clip_kernel(const __grid_constant__ Table<N> t, const double* __restrict__ part,
                                                  int nparts, float max_norm, float* __restrict__ norm) {
  const float nrm = total_norm(part, nparts);
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = nrm;
  float coef = max_norm / (nrm + 1e-6f);
  coef = coef > 1.f ? 1.f : coef;  // a NaN norm stays NaN and reaches every value, as in torch
  const int64_t c0 = (int64_t)t.chunks * blockIdx.x / gridDim.x, c1 = (int64_t)t.chunks * (blockIdx.x + 1) / gridDim.x;
  int ti = find(t, (int)(c1 - 1));
  // backwards: what the norm's pass read last is still in L2
  for (int64_t c = c1 - 1; c >= c0; --c) {
    while (t.e[ti].first > c) --ti;
    const Entry& e = t.e[ti];
    if (coef == 1.f && e.dst == e.src) continue;  // in place, and every value keeps its bits
    const int64_t at = (c - e.first) * CHUNK;
    const int64_t left = e.n - at;
    if (left >= CHUNK && aligned16(e.src) && aligned16(e.dst)) {
      const auto put = [&](int j, float4 q) {
        q.x *= coef, q.y *= coef, q.z *= coef, q.w *= coef;
        if (e.ddt == SCA2_F32) {
          *reinterpret_cast<float4*>(reinterpret_cast<float*>(e.dst) + at + j) = q;
        } else {
          __nv_bfloat162 a = __floats2bfloat162_rn(q.x, q.y), b = __floats2bfloat162_rn(q.z, q.w);
          uint2 o;
          o.x = *reinterpret_cast<uint32_t*>(&a), o.y = *reinterpret_cast<uint32_t*>(&b);
          *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(e.dst) + at + j) = o;
        }
      };
      if (e.sdt == SCA2_F32) vec_f32(reinterpret_cast<const float*>(e.src) + at, put);
      else vec_bf16(reinterpret_cast<const __nv_bfloat16*>(e.src) + at, put);
    } else {
      const int m = (int)(left < CHUNK ? left : CHUNK);
#pragma unroll 4
      for (int j = threadIdx.x; j < m; j += NT) st_io(e.dst, at + j, ld_io(e.src, at + j, e.sdt) * coef, e.ddt);
    }
  }
}

__global__ void __launch_bounds__(NT) finish_kernel(const double* __restrict__ part, int nparts, float* __restrict__ norm) {
  const float nrm = total_norm(part, nparts);
  if (threadIdx.x == 0) *norm = nrm;
}

constexpr int SMALL = 100, LARGE = 1000;
static_assert(sizeof(Table<LARGE>) <= 32764 - 64, "kernel parameters are limited to 32764 bytes");

int grid_of(int chunks) { return std::max(1, std::min(chunks, 148 * CTAS_PER_SM)); }

struct Group {  // the tensors of one launch
  int begin, end, chunks, grid, part;
};

template <int N>
void fill(Table<N>& t, const sca2_grad_tensor* list, const Group& g) {
  t.count = 0, t.chunks = g.chunks;
  int first = 0;
  for (int i = g.begin; i < g.end; ++i) {
    if (list[i].n == 0) continue;
    t.e[t.count++] = Entry{list[i].src, list[i].dst, list[i].n, first, (int16_t)list[i].src_dtype,
                           (int16_t)list[i].dst_dtype};
    first += (int)((list[i].n + CHUNK - 1) / CHUNK);
  }
}

template <int N>
cudaError_t run(const sca2_grad_tensor* list, const std::vector<Group>& groups, int nparts, float max_norm, bool write,
                float* norm, double* part, cudaStream_t st) {
  Table<N> t;
  for (const Group& g : groups) {
    fill(t, list, g);
    norm_kernel<N><<<g.grid, NT, 0, st>>>(t, part + g.part);
    if (cudaError_t e = cudaGetLastError()) return e;
  }
  if (!write || groups.empty()) {
    finish_kernel<<<1, NT, 0, st>>>(part, nparts, norm);
    return cudaGetLastError();
  }
  for (size_t k = 0; k < groups.size(); ++k) {
    if (groups.size() > 1) fill(t, list, groups[k]);
    clip_kernel<N><<<groups[k].grid, NT, 0, st>>>(t, part, nparts, max_norm, k == 0 ? norm : nullptr);
    if (cudaError_t e = cudaGetLastError()) return e;
  }
  return cudaSuccess;
}

int fail(int code, const char* msg) {
  set_last_error(msg);
  return code;
}

// launches of LARGE tensors each, and of at most 2^30 chunks
std::vector<Group> groups_of(const sca2_grad_tensor* list, int count) {
  std::vector<Group> v;
  int part = 0;
  for (int i = 0; i < count;) {
    Group g{i, i, 0, 0, part};
    int64_t chunks = 0;
    while (g.end < count && g.end - g.begin < LARGE) {
      const int64_t c = (list[g.end].n + CHUNK - 1) / CHUNK;
      if (chunks + c > (1LL << 30)) break;
      chunks += c, ++g.end;
    }
    g.chunks = (int)chunks, g.grid = grid_of(g.chunks);
    i = g.end;
    if (!g.chunks) continue;
    part += g.grid;
    v.push_back(g);
  }
  return v;
}

int width(int dt) { return dt == SCA2_BF16 ? 2 : 4; }

// A value that a call writes must not be read or written by another tensor of the list (the
// chunks run in no order); the one allowed overlap is a tensor with its own destination.
bool overlaps(const sca2_grad_tensor* list, int count) {
  struct Range {
    uintptr_t b, e;
    bool write;
  };
  std::vector<Range> r;
  r.reserve(2 * (size_t)count);
  for (int i = 0; i < count; ++i) {
    const sca2_grad_tensor& t = list[i];
    if (t.n == 0) continue;
    const uintptr_t s = reinterpret_cast<uintptr_t>(t.src), d = reinterpret_cast<uintptr_t>(t.dst);
    if (!(s == d && t.src_dtype == t.dst_dtype)) r.push_back({s, s + (uintptr_t)t.n * width(t.src_dtype), false});
    r.push_back({d, d + (uintptr_t)t.n * width(t.dst_dtype), true});
  }
  std::sort(r.begin(), r.end(), [](const Range& a, const Range& b) { return a.b < b.b; });
  uintptr_t any = 0, wr = 0;
  for (const Range& x : r) {
    if (x.b < (x.write ? any : wr)) return true;
    any = std::max(any, x.e);
    if (x.write) wr = std::max(wr, x.e);
  }
  return false;
}

int check(const sca2_grad_tensor* list, int32_t count, bool write) {
  if (count < 0 || (count > 0 && !list)) return fail(SCA2_ERR_ARG, "clip_grads: null or negative tensor list");
  for (int i = 0; i < count; ++i) {
    const sca2_grad_tensor& t = list[i];
    if (t.n < 0 || t.n > (1LL << 41)) return fail(SCA2_ERR_ARG, "clip_grads: a tensor's size must be 0 ... 2^41");
    if (t.n > 0 && (!t.src || (write && !t.dst))) return fail(SCA2_ERR_ARG, "clip_grads: null tensor");
    if ((t.src_dtype != SCA2_F32 && t.src_dtype != SCA2_BF16) ||
        (write && t.dst_dtype != SCA2_F32 && t.dst_dtype != SCA2_BF16))
      return fail(SCA2_ERR_ARG, "clip_grads: tensors are SCA2_F32 or SCA2_BF16");
    if (t.n > 0 && ((reinterpret_cast<uintptr_t>(t.src) % width(t.src_dtype)) ||
                    (write && reinterpret_cast<uintptr_t>(t.dst) % width(t.dst_dtype))))
      return fail(SCA2_ERR_ARG, "clip_grads: a tensor is not aligned to its values");
  }
  return SCA2_OK;
}

int go(const sca2_grad_tensor* list, int32_t count, float max_norm, bool write, float* norm, void* work,
       int64_t work_bytes, void* stream) {
  if (int rc = check(list, count, write)) return rc;
  if (!norm || !work || (reinterpret_cast<uintptr_t>(work) & 7u))
    return fail(SCA2_ERR_ARG, "clip_grads: norm and an 8-byte aligned workspace are needed");
  if (write && !(max_norm >= 0.f)) return fail(SCA2_ERR_ARG, "clip_grads: max_norm must be >= 0");
  try {
    if (write && overlaps(list, count))
      return fail(SCA2_ERR_ARG, "clip_grads: a destination overlaps another tensor of the list");
    const std::vector<Group> groups = groups_of(list, count);
    const int nparts = groups.empty() ? 0 : groups.back().part + groups.back().grid;
    if (work_bytes < (int64_t)nparts * 8) return fail(SCA2_ERR_ARG, "clip_grads: workspace too small");
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    double* part = static_cast<double*>(work);
    const cudaError_t e = count <= SMALL ? run<SMALL>(list, groups, nparts, max_norm, write, norm, part, st)
                                         : run<LARGE>(list, groups, nparts, max_norm, write, norm, part, st);
    if (e != cudaSuccess) {
      set_last_error(std::string("sca2_clip_grads: ") + cudaGetErrorString(e));
      return SCA2_ERR_CUDA;
    }
    return SCA2_OK;
  } catch (const std::exception&) {
    return fail(SCA2_ERR_ARG, "clip_grads: out of host memory");
  }
}

}  // namespace clip
}  // namespace sca2

extern "C" {

int64_t sca2_clip_grads_work_bytes(const sca2_grad_tensor* list, int32_t count) {
  if (sca2::clip::check(list, count, false)) return 0;
  try {
    const auto groups = sca2::clip::groups_of(list, count);
    return 8 * (int64_t)(groups.empty() ? 1 : groups.back().part + groups.back().grid);
  } catch (const std::exception&) {
    return 0;
  }
}

int sca2_grad_norm(const sca2_grad_tensor* list, int32_t count, float* norm, void* work, int64_t work_bytes,
                   void* stream) {
  return sca2::clip::go(list, count, 0.f, false, norm, work, work_bytes, stream);
}

int sca2_clip_grads(const sca2_grad_tensor* list, int32_t count, float max_norm, float* norm, void* work,
                    int64_t work_bytes, void* stream) {
  return sca2::clip::go(list, count, max_norm, true, norm, work, work_bytes, stream);
}

}  // extern "C"
