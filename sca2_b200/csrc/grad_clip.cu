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
// tensors form one sequence, dealt to the CTAs in turn whatever the tensors' sizes; the second pass
// takes it from the end, whose values are still in L2.  Measured, 97.5 M fp32 values (390 MB): 74 and
// 120 us; the same passes over a contiguous range for each CTA 77 and 123 us.
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

// The launch's tensors.  Kernel parameters hold up to 32 764 bytes: 1000 entries, or a smaller table
// where it suffices (the parameters are copied at each launch).
template <int N>
struct Table {
  int32_t count, chunks;
  Entry e[N];
};

// the tensor that chunk c belongs to; `at` is the one of the CTA's chunk before (-1: none)
template <int N>
__device__ __forceinline__ int tensor_of(const Table<N>& t, int c, int at) {
  if (at >= 0 && t.e[at].first <= c && (at + 1 == t.count || c < t.e[at + 1].first)) return at;
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {  // last entry whose first chunk is <= c
    const int mid = (lo + hi + 1) >> 1;
    if (t.e[mid].first <= c) lo = mid; else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

__device__ __forceinline__ float2 unpack(uint32_t u) {
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u));
}

// The 16 values of a chunk that thread t takes: groups of consecutive values where the chunk is
// whole and on a 16-byte boundary, every NT-th value otherwise.  All loads are issued before the
// first value is used.
template <class T>
__device__ __forceinline__ void load_vec(const T* p, float (&v)[16]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float4 q = reinterpret_cast<const float4*>(p)[threadIdx.x + NT * k];
      v[4 * k] = q.x, v[4 * k + 1] = q.y, v[4 * k + 2] = q.z, v[4 * k + 3] = q.w;
    }
  } else {
    uint4 q[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) q[k] = reinterpret_cast<const uint4*>(p)[threadIdx.x + NT * k];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float2 a = unpack(q[k].x), b = unpack(q[k].y), c = unpack(q[k].z), d = unpack(q[k].w);
      v[8 * k] = a.x, v[8 * k + 1] = a.y, v[8 * k + 2] = b.x, v[8 * k + 3] = b.y;
      v[8 * k + 4] = c.x, v[8 * k + 5] = c.y, v[8 * k + 6] = d.x, v[8 * k + 7] = d.y;
    }
  }
}
__device__ __forceinline__ float value(float v) { return v; }
__device__ __forceinline__ float value(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ void load_each(const T* p, int m, float (&v)[16]) {
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const int j = threadIdx.x + NT * k;
    v[k] = j < m ? value(p[j]) : 0.f;
  }
}
// vec: the source is whole and aligned (its groups: 4 values of fp32, 8 of bf16)
template <class T>
__device__ __forceinline__ void load16(const void* src, int64_t at, int m, bool vec, float (&v)[16]) {
  const T* p = reinterpret_cast<const T*>(src) + at;
  if (vec) load_vec(p, v);
  else load_each(p, m, v);
}
// the first value's place and the distance of the groups, as load_vec<T> took them
template <class TS, class TD>
__device__ __forceinline__ void store_vec(TD* p, const float (&v)[16]) {
  constexpr int G = sizeof(TS) == 4 ? 4 : 8;  // values of a group
#pragma unroll
  for (int k = 0; k < 16; k += 4) {
    const int j = G * (threadIdx.x + NT * (k / G)) + k % G;
    if constexpr (sizeof(TD) == 4) {
      __stcs(reinterpret_cast<float4*>(p + j), make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]));
    } else {
      const __nv_bfloat162 a = __floats2bfloat162_rn(v[k], v[k + 1]), b = __floats2bfloat162_rn(v[k + 2], v[k + 3]);
      __stcs(reinterpret_cast<uint2*>(p + j), make_uint2(*reinterpret_cast<const uint32_t*>(&a),
                                                         *reinterpret_cast<const uint32_t*>(&b)));
    }
  }
}
__device__ __forceinline__ void put(float* p, float v) { __stcs(p, v); }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

template <class TS, class TD>
__device__ __forceinline__ void scale_chunk(const Entry& e, int64_t at, int m, bool vec, float coef) {
  float v[16];
  load16<TS>(e.src, at, m, vec, v);
#pragma unroll
  for (int k = 0; k < 16; ++k) v[k] *= coef;
  TD* p = reinterpret_cast<TD*>(e.dst) + at;
  if (vec) {
    store_vec<TS>(p, v);
  } else {
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const int j = threadIdx.x + NT * k;
      if (j < m) put(p + j, v[k]);
    }
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
  double s0 = 0., s1 = 0., s2 = 0., s3 = 0.;
  for (int c = blockIdx.x, ti = -1; c < t.chunks; c += gridDim.x) {
    ti = tensor_of(t, c, ti);
    const Entry& e = t.e[ti];
    const int64_t at = (int64_t)(c - e.first) * CHUNK;
    const int m = (int)(e.n - at < CHUNK ? e.n - at : CHUNK);
    const bool vec = m == CHUNK && aligned16(e.src);
    float v[16];
    if (e.sdt == SCA2_F32) load16<float>(e.src, at, m, vec, v);
    else load16<__nv_bfloat16>(e.src, at, m, vec, v);
#pragma unroll
    for (int k = 0; k < 16; k += 4) {
      s0 = fma((double)v[k], (double)v[k], s0), s1 = fma((double)v[k + 1], (double)v[k + 1], s1);
      s2 = fma((double)v[k + 2], (double)v[k + 2], s2), s3 = fma((double)v[k + 3], (double)v[k + 3], s3);
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
  // backwards: what the norm's pass read last is still in L2
  const int last = t.chunks - 1 - (t.chunks - 1 - (int)blockIdx.x) % (int)gridDim.x;
  for (int c = last, ti = -1; c >= 0; c -= gridDim.x) {
    ti = tensor_of(t, c, ti);
    const Entry& e = t.e[ti];
    if (coef == 1.f && e.dst == e.src) continue;  // in place, and every value keeps its bits
    const int64_t at = (int64_t)(c - e.first) * CHUNK;
    const int m = (int)(e.n - at < CHUNK ? e.n - at : CHUNK);
    const bool vec = m == CHUNK && aligned16(e.src) && aligned16(e.dst);
    if (e.sdt == SCA2_F32) {
      if (e.ddt == SCA2_F32) scale_chunk<float, float>(e, at, m, vec, coef);
      else scale_chunk<float, __nv_bfloat16>(e, at, m, vec, coef);
    } else {
      if (e.ddt == SCA2_F32) scale_chunk<__nv_bfloat16, float>(e, at, m, vec, coef);
      else scale_chunk<__nv_bfloat16, __nv_bfloat16>(e, at, m, vec, coef);
    }
  }
}

__global__ void __launch_bounds__(NT) finish_kernel(const double* __restrict__ part, int nparts, float* __restrict__ norm) {
  const float nrm = total_norm(part, nparts);
  if (threadIdx.x == 0) *norm = nrm;
}

constexpr int SMALL = 64, MIDDLE = 256, LARGE = 1000;
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

constexpr int64_t PARTS = 148 * CTAS_PER_SM;  // partials of one launch, at most

// launches of LARGE tensors each; false where one would have 2^30 chunks or more
bool groups_of(const sca2_grad_tensor* list, int count, std::vector<Group>& v) {
  int part = 0;
  for (int i = 0; i < count; i += LARGE) {
    Group g{i, std::min(count, i + LARGE), 0, 0, part};
    int64_t chunks = 0;
    for (int k = g.begin; k < g.end; ++k) chunks += (list[k].n + CHUNK - 1) / CHUNK;
    if (chunks >= (1LL << 30)) return false;
    g.chunks = (int)chunks, g.grid = grid_of(g.chunks);
    if (!g.chunks) continue;
    part += g.grid;
    v.push_back(g);
  }
  return true;
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
  if (work_bytes < sca2_clip_grads_work_bytes(count)) return fail(SCA2_ERR_ARG, "clip_grads: workspace too small");
  if (write && !(max_norm >= 0.f)) return fail(SCA2_ERR_ARG, "clip_grads: max_norm must be >= 0");
  try {
    if (write && overlaps(list, count))
      return fail(SCA2_ERR_ARG, "clip_grads: a destination overlaps another tensor of the list");
    std::vector<Group> groups;
    if (!groups_of(list, count, groups)) return fail(SCA2_ERR_UNSUPPORTED, "clip_grads: too many values");
    const int nparts = groups.empty() ? 0 : groups.back().part + groups.back().grid;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    double* part = static_cast<double*>(work);
    const cudaError_t e = count <= SMALL ? run<SMALL>(list, groups, nparts, max_norm, write, norm, part, st)
                          : count <= MIDDLE ? run<MIDDLE>(list, groups, nparts, max_norm, write, norm, part, st)
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

int64_t sca2_clip_grads_work_bytes(int32_t count) {
  return count < 0 ? 0 : 8 * sca2::clip::PARTS * std::max<int64_t>(1, ((int64_t)count + sca2::clip::LARGE - 1) / sca2::clip::LARGE);
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
