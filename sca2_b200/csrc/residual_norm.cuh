// Residual join with the norms on both sides of it, forward and backward.  Per row of width d:
//
//     p = N_post(u)  (or u),   y = x + scale * sigmoid(gate) * p,   z = N(y)
//
// N is LayerNorm (biased variance, eps inside the root, weight and optional bias) or the RMS norm
// with weight; gate is one logit for each value or for each row.  All arithmetic in fp32: y and z
// are rounded once, when stored, and z is formed from the unrounded y.  Instantiated per type of
// x and u (residual_norm_*.cu).
//
// Bound by memory.  Forward: the row stays in registers between its (up to four) reductions, so
// everything is read and written once.  Backward: recomputes p, y and the normalised rows from the
// inputs and the saved means and deviations (16 bytes a row) instead of keeping them.
#pragma once

#include <algorithm>

#include "common.cuh"

namespace sca2 {
namespace rnorm {

struct Args {
  const void *x, *u, *gate;
  int64_t sx, su, sg;              // row strides in values
  const float *w, *b, *pw, *pb, *scale;
  float* stats;                    // (rows, 4): mean and 1 / deviation of u, then of y
  int64_t rows;
  int d;
  float eps;
  int rms, gate_mode, zdt;         // gate_mode 0 none, 1 one logit a row, 2 one a value
  // forward
  void *y, *z;
  // backward
  const void *dy, *dz;
  void *dx, *du, *dgate;
  float* part;                     // (CTAs, 5, d): partial dw, db, dscale, dpw, dpb
};

enum { PART_W, PART_B, PART_SCALE, PART_PW, PART_PB, NPART };

// sigmoid by the special function unit's 2^x and 1 / x (relative error about 2^-22; 2^x overflows to
// inf, whose reciprocal is the 0 that belongs there)
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_fast(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float LOG2E = 1.4426950408889634f;
__device__ __forceinline__ float sigmoid(float v) { return rcp_fast(1.f + exp2_fast(-LOG2E * v)); }

// two fp32 values in one instruction (add, mul, fma of sm_100), each rounded as by itself: the
// kernels of aligned rows issue about half the instructions with them
struct F2 {
  uint64_t v;
};
__device__ __forceinline__ F2 pair(float a, float b) {
  return {((uint64_t)__float_as_uint(b) << 32) | __float_as_uint(a)};
}
__device__ __forceinline__ F2 both(float a) { return pair(a, a); }
__device__ __forceinline__ float first(F2 a) { return __uint_as_float((uint32_t)a.v); }
__device__ __forceinline__ float second(F2 a) { return __uint_as_float((uint32_t)(a.v >> 32)); }
__device__ __forceinline__ float sum(F2 a) { return first(a) + second(a); }
__device__ __forceinline__ F2 operator+(F2 a, F2 b) {
  F2 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
  return d;
}
__device__ __forceinline__ F2 operator*(F2 a, F2 b) {
  F2 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
  return d;
}
__device__ __forceinline__ F2 fma(F2 a, F2 b, F2 c) {
  F2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return d;
}
__device__ __forceinline__ F2 sigmoid(F2 v) {
  const F2 t = v * both(-LOG2E);
  const F2 e = pair(exp2_fast(first(t)), exp2_fast(second(t))) + both(1.f);
  return pair(rcp_fast(first(e)), rcp_fast(second(e)));
}

__device__ __forceinline__ void unpack2(uint32_t u, float* v) {
  v[0] = __uint_as_float(u << 16), v[1] = __uint_as_float(u & 0xFFFF0000u);
}
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&p);
}

// ---- four values at consecutive columns (VEC = 4: aligned) or one ------------------------------
template <int VEC>
__device__ __forceinline__ void loadv(const float* p, float* v) {
  if constexpr (VEC == 1) {
    v[0] = *p;
  } else {
    const float4 q = *reinterpret_cast<const float4*>(p);
    v[0] = q.x, v[1] = q.y, v[2] = q.z, v[3] = q.w;
  }
}
template <int VEC>
__device__ __forceinline__ void loadv(const __nv_bfloat16* p, float* v) {
  if constexpr (VEC == 1) {
    v[0] = __bfloat162float(*p);
  } else {
    const uint2 q = *reinterpret_cast<const uint2*>(p);
    unpack2(q.x, v), unpack2(q.y, v + 2);
  }
}
template <int VEC>
__device__ __forceinline__ void storev(float* p, const float* v) {
  if constexpr (VEC == 1) {
    *p = v[0];
  } else {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  }
}
template <int VEC>
__device__ __forceinline__ void storev(__nv_bfloat16* p, const float* v) {
  if constexpr (VEC == 1) {
    *p = __float2bfloat16_rn(v[0]);
  } else {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack2(v[0], v[1]), pack2(v[2], v[3]));
  }
}

// ---- forward --------------------------------------------------------------------------------
constexpr int FT = 256;

__device__ __forceinline__ float row_sum(float v, int& flip) {
  __shared__ float s[2][FT / 32];
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) s[flip][threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.f;
#pragma unroll
  for (int w = 0; w < FT / 32; ++w) v += s[flip][w];
  flip ^= 1;  // the next sum's writes pass this one's reads only after its own barrier
  return v;
}

// four consecutive values as two pairs
template <class T>
__device__ __forceinline__ void load2(const T* p, F2 (&v)[2]) {
  float q[4];
  loadv<4>(p, q);
  v[0] = pair(q[0], q[1]), v[1] = pair(q[2], q[3]);
}
template <class T>
__device__ __forceinline__ void store2(T* p, const F2 (&v)[2]) {
  const float q[4] = {first(v[0]), second(v[0]), first(v[1]), second(v[1])};
  storev<4>(p, q);
}

// ---- asynchronous copies: a thread's own values of the rows to come, into its own slots of shared
// memory, which no other thread reads: its wait for its copies is the only synchronisation.
template <int BYTES>
__device__ __forceinline__ void copy_async(void* dst, const void* src) {
  const uint32_t d = static_cast<uint32_t>(__cvta_generic_to_shared(dst));
  if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d), "l"(src) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(d), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// A group of four columns of a row, n of them inside it, in a thread's slot (GB bytes).  ANY: rows of
// any alignment.  Values of 32 bits then travel one by one; of 16 bits, the two aligned 8-byte words
// around the group, from which reading shifts it out (word by value at the tensor's two ends [lo, hi),
// so that nothing outside is read).
template <bool ANY, class T>
constexpr int GB = ANY ? 16 : 4 * (int)sizeof(T);

template <bool ANY, class T>
__device__ __forceinline__ void group_copy(void* slot, const T* p, int n, const T* lo, const T* hi) {
  if constexpr (!ANY) {
    copy_async<4 * sizeof(T)>(slot, p);
  } else if constexpr (sizeof(T) == 4) {
    const uint32_t s = static_cast<uint32_t>(__cvta_generic_to_shared(slot));
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < n) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(s + 4 * k), "l"(p + k) : "memory");
  } else {
    const T* w = reinterpret_cast<const T*>(reinterpret_cast<uintptr_t>(p) & ~(uintptr_t)7);
    const int m = (int)(p - w);  // the group's place in the words
    if (w >= lo && w + 8 <= hi) {
      copy_async<8>(slot, w);
      if (m + n > 4) copy_async<8>(static_cast<uint8_t*>(slot) + 8, w + 4);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (k < n) static_cast<T*>(slot)[m + k] = p[k];
    }
  }
}
template <bool ANY, class T>
__device__ __forceinline__ void group_read(const void* slot, const T* p, int n, F2 (&v)[2]) {
  if constexpr (!ANY) {
    load2(static_cast<const T*>(slot), v);
  } else {
    float q[4];
    if constexpr (sizeof(T) == 4) {
      loadv<4>(static_cast<const float*>(slot), q);
    } else {
      const ulonglong2 w = *static_cast<const ulonglong2*>(slot);
      const int sh = 16 * (int)((reinterpret_cast<uintptr_t>(p) >> 1) & 3);
      const unsigned long long u = sh ? (w.x >> sh) | (w.y << (64 - sh)) : w.x;
      unpack2((uint32_t)u, q), unpack2((uint32_t)(u >> 32), q + 2);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k >= n) q[k] = 0.f;
    v[0] = pair(q[0], q[1]), v[1] = pair(q[2], q[3]);
  }
}
template <bool ANY, class T>
__device__ __forceinline__ void group_store(T* p, int n, const F2 (&v)[2]) {
  if constexpr (!ANY) {
    store2(p, v);
  } else {
    const float q[4] = {first(v[0]), second(v[0]), first(v[1]), second(v[1])};
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < n) storev<1>(p + k, q + k);
  }
}
// n values of a parameter, `fill` beyond
template <bool ANY>
__device__ __forceinline__ void group_param(const float* p, int n, float fill, F2 (&v)[2]) {
  if constexpr (!ANY) {
    load2(p, v);
  } else {
    float q[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) q[k] = k < n ? p[k] : fill;
    v[0] = pair(q[0], q[1]), v[1] = pair(q[2], q[3]);
  }
}
// zeros beyond the n values inside the row
template <bool ANY>
__device__ __forceinline__ void group_clean(int n, F2 (&v)[2]) {
  if constexpr (ANY) {
    if (n < 4) {
      if (n < 1) v[0] = both(0.f);
      else if (n < 2) v[0] = pair(first(v[0]), 0.f);
      v[1] = n < 3 ? both(0.f) : pair(first(v[1]), 0.f);
    }
  }
}

// Forward for rows of up to 1024 values: a warp owns a row, each lane NG groups of four
// values, so that every copy, load and store of the warp is one run of whole sectors in either type.
// The slots hold one row: the next row's u is asked for once this row's is in registers, its x and
// gate once the join has read this row's, and both travel under the rest of the row's work.  The
// parameters lie in shared memory too: read from L1 their latency was the kernel's bound (65536 x
// 768, everything on: 141 us, 116 us so; 705 MB are 109 us at the copy rate).
template <int NG, int GATE, bool ANY, class TX, class TU>
struct FwdRing {  // bytes of a thread's group in each array; the arrays' slots lie thread by thread
  static constexpr int BU = GB<ANY, TU>, BX = GB<ANY, TX>, BG = GATE == 2 ? BU : 0;
  static constexpr int OX = NG * BU * FT, OG = OX + NG * BX * FT, OP = OG + NG * BG * FT;
  static constexpr int D = NG * 128;  // floats of a parameter, from OP
};

template <int NG, int GATE, bool POST, bool ANY, class TX, class TU>
__global__ void __launch_bounds__(FT, 3) fwd_ring(const Args a) {
  using L = FwdRing<NG, GATE, ANY, TX, TU>;
  extern __shared__ __align__(16) uint8_t slots[];
  const int lane = threadIdx.x & 31, d = a.d;
  const float inv = 1.f / (float)d;
  const auto col = [&](int k) { return 4 * (lane + 32 * k); };
  const auto in = [&](int k) { return ANY ? min(4, d - col(k)) : 4; };
  const auto slot = [&](int off, int k, int bytes) { return slots + off + (k * FT + threadIdx.x) * bytes; };
  const int64_t step = (int64_t)gridDim.x * (FT / 32);
  int64_t row = (int64_t)blockIdx.x * (FT / 32) + (threadIdx.x >> 5);
  const auto fetch_u = [&](int64_t r) {
    if (r < a.rows) {
      const TU *p = reinterpret_cast<const TU*>(a.u), *e = p + (a.rows - 1) * a.su + d;
#pragma unroll
      for (int k = 0; k < NG; ++k)
        if (col(k) < d) group_copy<ANY>(slot(0, k, L::BU), p + r * a.su + col(k), in(k), p, e);
    }
    copies_commit();
  };
  const auto fetch_x = [&](int64_t r) {
    if (r < a.rows) {
      const TX *p = reinterpret_cast<const TX*>(a.x), *e = p + (a.rows - 1) * a.sx + d;
      const TU *q = reinterpret_cast<const TU*>(a.gate), *f = q + (a.rows - 1) * a.sg + d;
#pragma unroll
      for (int k = 0; k < NG; ++k)
        if (col(k) < d) {
          group_copy<ANY>(slot(L::OX, k, L::BX), p + r * a.sx + col(k), in(k), p, e);
          if constexpr (GATE == 2) group_copy<ANY>(slot(L::OG, k, L::BU), q + r * a.sg + col(k), in(k), q, f);
        }
    }
    copies_commit();
  };
  F2 y[NG][2];
  const auto normalise = [&](float& mu, float& rs) {  // y <- y - mean
    mu = 0.f;
    if (!a.rms) {
      F2 s = both(0.f);
#pragma unroll
      for (int k = 0; k < NG; ++k) s = s + (y[k][0] + y[k][1]);  // columns past d hold 0
      mu = warp_sum(sum(s)) * inv;
    }
    const F2 m = both(-mu);
    F2 q0 = both(0.f), q1 = q0;
#pragma unroll
    for (int k = 0; k < NG; ++k)
      if (col(k) < d) {
        y[k][0] = y[k][0] + m, y[k][1] = y[k][1] + m;
        group_clean<ANY>(in(k), y[k]);
        q0 = fma(y[k][0], y[k][0], q0), q1 = fma(y[k][1], y[k][1], q1);
      }
    rs = rsqrtf(warp_sum(sum(q0 + q1)) * inv + a.eps);
  };
  const auto affine = [&](int k, float rs, const float* w, const float* b) {  // y <- y rs w + b
    F2 q[2], c[2] = {both(0.f), both(0.f)};
    load2(w + col(k), q);
    if (b) load2(b + col(k), c);
#pragma unroll
    for (int j = 0; j < 2; ++j) y[k][j] = fma(y[k][j] * both(rs), q[j], c[j]);
  };

  fetch_u(row), fetch_x(row);
  float* par = reinterpret_cast<float*>(slots + L::OP);
  const auto stage = [&](const float* p) -> const float* {
    if (!p) return nullptr;
    float* q = par;
    for (int c = threadIdx.x; c < L::D; c += FT) q[c] = c < d ? p[c] : 0.f;
    par += L::D;
    return q;
  };
  const float *w = stage(a.w), *b = stage(a.b), *pw = stage(a.pw), *pb = stage(a.pb), *scale = stage(a.scale);
  __syncthreads();
  for (; row < a.rows; row += step) {
    float gt = 1.f;
    if constexpr (GATE == 1) {
      loadv<1>(reinterpret_cast<const TU*>(a.gate) + row * a.sg, &gt);
      gt = sigmoid(gt);
    }
    copies_wait<1>();
    float mu = 0.f, rs = 0.f;
#pragma unroll
    for (int k = 0; k < NG; ++k) {
      y[k][0] = y[k][1] = both(0.f);
      if (col(k) < d) group_read<ANY>(slot(0, k, L::BU), reinterpret_cast<const TU*>(a.u) + row * a.su, in(k), y[k]);
    }
    fetch_u(row + step);
    if constexpr (POST) {
      normalise(mu, rs);
#pragma unroll
      for (int k = 0; k < NG; ++k)
        if (col(k) < d) affine(k, rs, pw, pb);
    }
    if (a.stats && lane == 0) a.stats[4 * row] = mu, a.stats[4 * row + 1] = rs;
    copies_wait<1>();
#pragma unroll
    for (int k = 0; k < NG; ++k)
      if (col(k) < d) {
        F2 q[2];
        if (scale) {
          load2(scale + col(k), q);
          y[k][0] = y[k][0] * q[0], y[k][1] = y[k][1] * q[1];
        }
        if constexpr (GATE == 2) {
          group_read<ANY>(slot(L::OG, k, L::BU), reinterpret_cast<const TU*>(a.gate) + row * a.sg, in(k), q);
          y[k][0] = y[k][0] * sigmoid(q[0]), y[k][1] = y[k][1] * sigmoid(q[1]);
        }
        group_read<ANY>(slot(L::OX, k, L::BX), reinterpret_cast<const TX*>(a.x) + row * a.sx, in(k), q);
#pragma unroll
        for (int j = 0; j < 2; ++j) y[k][j] = GATE == 1 ? fma(both(gt), y[k][j], q[j]) : y[k][j] + q[j];
        group_clean<ANY>(in(k), y[k]);
        group_store<ANY>(reinterpret_cast<TX*>(a.y) + row * d + col(k), in(k), y[k]);
      }
    fetch_x(row + step);
    if (!a.z) continue;
    normalise(mu, rs);
    if (a.stats && lane == 0) a.stats[4 * row + 2] = mu, a.stats[4 * row + 3] = rs;
#pragma unroll
    for (int k = 0; k < NG; ++k)
      if (col(k) < d) {
        affine(k, rs, w, b);
        if (a.zdt == SCA2_BF16) group_store<ANY>(reinterpret_cast<__nv_bfloat16*>(a.z) + row * d + col(k), in(k), y[k]);
        else group_store<ANY>(reinterpret_cast<float*>(a.z) + row * d + col(k), in(k), y[k]);
      }
  }
  copies_wait<0>();
}

// Forward for wider rows, and from 513 values for those of any alignment (whose slots are larger: 32768 x
// 1001 in bf16 317 us with fwd_ring, 184 so): a CTA owns a row, each thread NG groups of four columns and
// their parameters; the next row travels as in fwd_ring.
template <int NG, int GATE, bool POST, bool ANY, class TX, class TU>
__global__ void __launch_bounds__(FT, NG == 1 ? 4 : 2) fwd_wide(const Args a) {
  using L = FwdRing<NG, GATE, ANY, TX, TU>;
  extern __shared__ __align__(16) uint8_t slots[];
  const int t = threadIdx.x, d = a.d;
  const float inv = 1.f / (float)d;
  const auto col = [&](int k) { return 4 * (t + FT * k); };
  const auto in = [&](int k) { return ANY ? min(4, d - col(k)) : 4; };
  const auto slot = [&](int off, int k, int bytes) { return slots + off + (k * FT + t) * bytes; };
  const auto fetch_u = [&](int64_t r) {
    if (r < a.rows) {
      const TU *p = reinterpret_cast<const TU*>(a.u), *e = p + (a.rows - 1) * a.su + d;
#pragma unroll
      for (int k = 0; k < NG; ++k)
        if (col(k) < d) group_copy<ANY>(slot(0, k, L::BU), p + r * a.su + col(k), in(k), p, e);
    }
    copies_commit();
  };
  const auto fetch_x = [&](int64_t r) {
    if (r < a.rows) {
      const TX *p = reinterpret_cast<const TX*>(a.x), *e = p + (a.rows - 1) * a.sx + d;
      const TU *q = reinterpret_cast<const TU*>(a.gate), *f = q + (a.rows - 1) * a.sg + d;
#pragma unroll
      for (int k = 0; k < NG; ++k)
        if (col(k) < d) {
          group_copy<ANY>(slot(L::OX, k, L::BX), p + r * a.sx + col(k), in(k), p, e);
          if constexpr (GATE == 2) group_copy<ANY>(slot(L::OG, k, L::BU), q + r * a.sg + col(k), in(k), q, f);
        }
    }
    copies_commit();
  };
  int64_t row = blockIdx.x;
  fetch_u(row), fetch_x(row);
  F2 w[NG][2], b[NG][2], pw[NG][2], pb[NG][2], sc[NG][2], y[NG][2];
  const auto param = [&](const float* p, float fill, F2 (&v)[NG][2]) {
#pragma unroll
    for (int k = 0; k < NG; ++k) {
      v[k][0] = v[k][1] = both(fill);
      if (p && col(k) < d) group_param<ANY>(p + col(k), in(k), fill, v[k]);
    }
  };
  param(a.w, 0.f, w), param(a.b, 0.f, b), param(a.scale, 1.f, sc);
  if constexpr (POST) param(a.pw, 0.f, pw), param(a.pb, 0.f, pb);
  int flip = 0;
  const auto normalise = [&](float& mu, float& rs) {  // y <- y - mean
    mu = 0.f;
    if (!a.rms) {
      F2 s = both(0.f);
#pragma unroll
      for (int k = 0; k < NG; ++k) s = s + (y[k][0] + y[k][1]);  // columns past d hold 0
      mu = row_sum(sum(s), flip) * inv;
    }
    const F2 m = both(-mu);
    F2 q0 = both(0.f), q1 = q0;
#pragma unroll
    for (int k = 0; k < NG; ++k)
      if (col(k) < d) {
        y[k][0] = y[k][0] + m, y[k][1] = y[k][1] + m;
        group_clean<ANY>(in(k), y[k]);
        q0 = fma(y[k][0], y[k][0], q0), q1 = fma(y[k][1], y[k][1], q1);
      }
    rs = rsqrtf(row_sum(sum(q0 + q1), flip) * inv + a.eps);
  };
  for (; row < a.rows; row += gridDim.x) {
    float gt = 1.f;
    if constexpr (GATE == 1) {
      loadv<1>(reinterpret_cast<const TU*>(a.gate) + row * a.sg, &gt);
      gt = sigmoid(gt);
    }
    copies_wait<1>();
    float mu = 0.f, rs = 0.f;
#pragma unroll
    for (int k = 0; k < NG; ++k) {
      y[k][0] = y[k][1] = both(0.f);
      if (col(k) < d) group_read<ANY>(slot(0, k, L::BU), reinterpret_cast<const TU*>(a.u) + row * a.su, in(k), y[k]);
    }
    fetch_u(row + gridDim.x);
    if constexpr (POST) {
      normalise(mu, rs);
#pragma unroll
      for (int k = 0; k < NG; ++k)
#pragma unroll
        for (int j = 0; j < 2; ++j) y[k][j] = fma(y[k][j] * both(rs), pw[k][j], pb[k][j]);  // 0 past d
    }
    if (a.stats && t == 0) a.stats[4 * row] = mu, a.stats[4 * row + 1] = rs;
    copies_wait<1>();
#pragma unroll
    for (int k = 0; k < NG; ++k)
      if (col(k) < d) {
        F2 q[2];
        if constexpr (GATE == 2) {
          group_read<ANY>(slot(L::OG, k, L::BU), reinterpret_cast<const TU*>(a.gate) + row * a.sg, in(k), q);
          y[k][0] = y[k][0] * sigmoid(q[0]), y[k][1] = y[k][1] * sigmoid(q[1]);
        }
        group_read<ANY>(slot(L::OX, k, L::BX), reinterpret_cast<const TX*>(a.x) + row * a.sx, in(k), q);
#pragma unroll
        for (int j = 0; j < 2; ++j) y[k][j] = fma(GATE == 1 ? both(gt) * sc[k][j] : sc[k][j], y[k][j], q[j]);
        group_clean<ANY>(in(k), y[k]);
        group_store<ANY>(reinterpret_cast<TX*>(a.y) + row * d + col(k), in(k), y[k]);
      }
    fetch_x(row + gridDim.x);
    if (!a.z) continue;
    normalise(mu, rs);
    if (a.stats && t == 0) a.stats[4 * row + 2] = mu, a.stats[4 * row + 3] = rs;
#pragma unroll
    for (int k = 0; k < NG; ++k)
      if (col(k) < d) {
#pragma unroll
        for (int j = 0; j < 2; ++j) y[k][j] = fma(y[k][j] * both(rs), w[k][j], b[k][j]);
        if (a.zdt == SCA2_BF16) group_store<ANY>(reinterpret_cast<__nv_bfloat16*>(a.z) + row * d + col(k), in(k), y[k]);
        else group_store<ANY>(reinterpret_cast<float*>(a.z) + row * d + col(k), in(k), y[k]);
      }
  }
  copies_wait<0>();
}

// ---- backward -------------------------------------------------------------------------------
// A thread owns four columns of every row (4t ... 4t+3, or t + T k where rows are not aligned), so
// the five column sums stay in its registers over all its rows.  bwd_kernel takes few rows (and the few
// widest forms that bwd_ring's shared memory does not hold): a row at a time, by as many CTAs as the rows feed.
template <int N, int O>
__device__ __forceinline__ void warp_sums(float* v, int lane) {
  // after the halving steps a lane holds N / 2^s of the values, chosen by its upper lane bits
  if constexpr (O > 0) {
    if constexpr (N % 2 == 0) {
      const bool hi = lane & O;
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        const float give = hi ? v[i] : v[i + N / 2], keep = hi ? v[i + N / 2] : v[i];
        v[i] = keep + __shfl_xor_sync(0xffffffffu, give, O);
      }
      warp_sums<N / 2, O / 2>(v, lane);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], O);
      warp_sums<N, O / 2>(v, lane);
    }
  }
}
constexpr int halvings(int n) { return n % 2 == 0 ? 1 + halvings(n / 2) : 0; }

// CTA sums of N values over at most W warps; `s` has (N, W) floats whose unused warps hold zeros.
// After the barrier every warp adds the warps' parts itself, W lanes to a value, and hands the
// totals round: few instructions, and no second barrier.
template <int N, int W>
__device__ __forceinline__ void cta_sums(float* v, float* s) {
  constexpr int H = halvings(N) < 5 ? halvings(N) : 5, LEFT = N >> H;
  constexpr int P = 32 / W, J = (N + P - 1) / P;  // values of one pass over the warp, passes
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  warp_sums<N, 16>(v, lane);
  if ((lane & ((1 << (5 - H)) - 1)) == 0) {
    int first = 0;  // the lane's upper H bits, the topmost choosing between halves of N
#pragma unroll
    for (int h = 0; h < H; ++h)
      if (lane & (16 >> h)) first += N >> (h + 1);
#pragma unroll
    for (int i = 0; i < LEFT; ++i) s[(first + i) * W + warp] = v[i];
  }
  __syncthreads();
  float q[J];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int at = P * W * j + lane;
    q[j] = at < N * W ? s[at] : 0.f;
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) q[j] += __shfl_xor_sync(0xffffffffu, q[j], o);
  }
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = __shfl_sync(0xffffffffu, q[i / P], (i % P) * W);
}

template <int MAXT, int MINB, bool CONTIG, class TX, class TU>
__global__ void __launch_bounds__(MAXT, MINB) bwd_kernel(const Args a) {
  constexpr int W = MAXT <= 256 ? 8 : MAXT / 32;
  __shared__ __align__(16) float red[2][3 * W];
  const int t = threadIdx.x, T = blockDim.x, d = a.d;
  const float inv = 1.f / (float)d;
  for (int i = t; i < 2 * 3 * W; i += T) (&red[0][0])[i] = 0.f;
  __syncthreads();
  const auto col = [&](int k) { return CONTIG ? 4 * t : t + T * k; };  // CONTIG: d % 4 == 0, all four or none
  const auto load = [&](const auto* p, float* v) {
    if constexpr (CONTIG) {
      if (4 * t < d) loadv<4>(p + 4 * t, v);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (col(k) < d) loadv<1>(p + col(k), v + k);
    }
  };
  const auto store = [&](auto* p, const float* v) {
    if constexpr (CONTIG) {
      if (4 * t < d) storev<4>(p + 4 * t, v);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (col(k) < d) storev<1>(p + col(k), v + k);
    }
  };
  // Columns past d get parameters of 0, which keep whatever a row's statistics make of them out of
  // the row's sums.
  const auto param = [&](const float* p, float fill, float* v) {
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = col(k) < d ? fill : 0.f;
    if (p) load(p, v);
  };
  const bool post = a.pw != nullptr, token = a.gate_mode == 1, chan = a.gate_mode == 2, has_z = a.dz != nullptr;
  float w[4], sc[4], pw[4], pb[4];
  param(a.w, 0.f, w);
  param(a.scale, 1.f, sc);
  param(a.pw, 1.f, pw);
  param(a.pb, 0.f, pb);
  float aw[4] = {}, ab[4] = {}, as[4] = {}, apw[4] = {}, apb[4] = {};
  int flip = 0;

  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    // un (normalised u, or u), s (the gate), dy, then yn and dn of z
    float un[4] = {}, s[4] = {}, dy[4] = {}, yn[4] = {}, dn[4] = {}, st[4];
    load(reinterpret_cast<const TU*>(a.u) + r * a.su, un);
    load(reinterpret_cast<const TX*>(a.x) + r * a.sx, yn);
    if (chan) load(reinterpret_cast<const TU*>(a.gate) + r * a.sg, s);
    if (token) {
      float g;
      loadv<1>(reinterpret_cast<const TU*>(a.gate) + r * a.sg, &g);
#pragma unroll
      for (int k = 0; k < 4; ++k) s[k] = g;
    }
    if (a.dy) load(reinterpret_cast<const TX*>(a.dy) + r * d, dy);
    if (has_z) {
      if (a.zdt == SCA2_BF16) load(reinterpret_cast<const __nv_bfloat16*>(a.dz) + r * d, dn);
      else load(reinterpret_cast<const float*>(a.dz) + r * d, dn);
    }
    loadv<4>(a.stats + 4 * r, st);
    float v[2] = {}, q[3] = {}, dg[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (post) un[k] = (un[k] - st[0]) * st[1];
      s[k] = a.gate_mode ? sigmoid(s[k]) : 1.f;
      if (has_z) {
        const float y = fmaf(sc[k] * s[k], fmaf(un[k], pw[k], pb[k]), yn[k]);
        yn[k] = (y - st[2]) * st[3];
        aw[k] = fmaf(dn[k], yn[k], aw[k]);
        ab[k] += dn[k];
        dn[k] *= w[k];
        v[0] += dn[k];
        v[1] = fmaf(dn[k], yn[k], v[1]);
      }
    }
    if (has_z) {
      cta_sums<2, W>(v, red[flip]);
      flip ^= 1;
      const float m1 = a.rms ? 0.f : v[0] * inv, m2 = v[1] * inv;
#pragma unroll
      for (int k = 0; k < 4; ++k) dy[k] += st[3] * (dn[k] - m1 - yn[k] * m2);
    }
    store(reinterpret_cast<TX*>(a.dx) + r * d, dy);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float e = dy[k], p = fmaf(un[k], pw[k], pb[k]), dp = e * sc[k] * s[k];
      as[k] = fmaf(e * s[k], p, as[k]);
      dg[k] = e * sc[k] * p * s[k] * (1.f - s[k]);
      q[2] += dg[k];
      apw[k] = fmaf(dp, un[k], apw[k]);
      apb[k] += dp;
      dn[k] = dp * pw[k];
      q[0] += dn[k];
      q[1] = fmaf(dn[k], un[k], q[1]);
    }
    if (chan) store(reinterpret_cast<TU*>(a.dgate) + r * d, dg);
    if (post || token) {
      cta_sums<3, W>(q, red[flip]);
      flip ^= 1;
    }
    if (post) {
      const float m1 = a.rms ? 0.f : q[0] * inv, m2 = q[1] * inv;
#pragma unroll
      for (int k = 0; k < 4; ++k) dn[k] = st[1] * (dn[k] - m1 - un[k] * m2);
    }
    store(reinterpret_cast<TU*>(a.du) + r * d, dn);
    if (token && t == 0) storev<1>(reinterpret_cast<TU*>(a.dgate) + r, &q[2]);
  }
  float* part = a.part + (int64_t)blockIdx.x * NPART * d;
  if (has_z) store(part + PART_W * d, aw);
  if (has_z && a.b) store(part + PART_B * d, ab);
  if (a.scale) store(part + PART_SCALE * d, as);
  if (post) store(part + PART_PW * d, apw);
  if (post && a.pb) store(part + PART_PB * d, apb);
}

// Backward for many rows: as bwd_kernel with the options that cost instructions as
// template parameters, and the next rows on their way into shared memory while the present ones are
// reduced.  A thread owns C groups of four columns (4t and, C = 2, 4(t + T)) of R rows at a time, C R = 2:
// two rows to 1024 values, one beyond.  One step ahead: three ahead need so much shared memory that one
// CTA an SM is left (65536 x 768: 226 us, 340 so; one row a step 249, three 246).  With C = 2 the
// parameters lie in the thread's slots too; their sums fill the registers.  Aligned rows have their copies,
// reads and stores written out: through the group functions the compiler orders them so that C = 2 loses
// 4 to 8 % (24576 x 1536: 176 us, 191 so).  Rows of any alignment on bwd_kernel instead: 49152 x 333
// 200 us, 135 here; 32768 x 1001 in bf16 417, 267; 12288 x 3001 in fp32 522, 412.
template <int C, int GATE, bool HASZ, bool ANY, class TX, class TU>
struct BwdRing {
  static constexpr int R = 2 / C, STAGES = 2, MAXT = C == 1 ? 256 : 512, MINB = C == 1 ? 2 : 1;
  // offsets of a group's slots, in bytes of one thread; every array's slots lie thread by thread
  static constexpr int BX = GB<ANY, TX>, BU = GB<ANY, TU>;
  static constexpr int OU = 0, OX = OU + BU, ODY = OX + BX, OG = ODY + BX, OZ = OG + (GATE == 2 ? BU : 0);
  static __host__ __device__ int z_bytes(bool bf16) { return bf16 && !ANY ? 8 : 16; }
  // bytes of a thread: a group with z of zb bytes a group; all of it
  static __host__ __device__ int group(int zb) { return OZ + (HASZ ? zb : 0); }
  static __host__ __device__ int thread(int zb) {
    return STAGES * R * (C * group(zb) + 16) + (C == 2 ? C * 4 * 16 : 0);  // 16: the row's statistics
  }
};
template <int C, int GATE, bool POST, bool HASZ, bool ANY, class TX, class TU>
__global__ void __launch_bounds__(BwdRing<C, GATE, HASZ, ANY, TX, TU>::MAXT, BwdRing<C, GATE, HASZ, ANY, TX, TU>::MINB)
    bwd_ring(const Args a) {
  using L = BwdRing<C, GATE, HASZ, ANY, TX, TU>;
  constexpr int W = L::MAXT / 32, R = L::R, ST = L::STAGES, N = 2 * C;  // N pairs of a row
  __shared__ __align__(16) float red[2][3 * R * W];
  extern __shared__ __align__(16) uint8_t slots[];
  const int t = threadIdx.x, T = blockDim.x, d = a.d;
  const float inv = 1.f / (float)d;
  const auto col = [&](int g) { return 4 * (t + T * g); };
  const auto inside = [&](int g) { return ANY ? min(4, d - col(g)) : 4; };
  for (int i = t; i < 2 * 3 * R * W; i += T) (&red[0][0])[i] = 0.f;
  __syncthreads();
  const bool zb16 = a.zdt == SCA2_BF16;
  const int zb = L::z_bytes(zb16), grp = L::group(zb);
  const auto slot = [&](int stage, int i, int g, int off, int bytes) {
    return slots + ((stage * R + i) * C + g) * grp * T + off * T + bytes * t;
  };
  uint8_t* const stat0 = slots + ST * R * C * grp * T + 16 * t;  // statistics of (stage, row): + (stage R + row) 16 T
  float* const par0 = reinterpret_cast<float*>(slots + ST * R * (C * grp + 16) * T) + 4 * t;  // parameter i of group g: + (4 g + i) 4 T
  const F2 zero = both(0.f), one = both(1.f), minus = both(-1.f);
  // w, scale, pw, pb of the thread's columns; 0 past d, which keeps those out of the sums
  F2 reg[4][2];
  {
    const float* src[4] = {HASZ ? a.w : nullptr, a.scale, POST ? a.pw : nullptr, POST ? a.pb : nullptr};
#pragma unroll
    for (int g = 0; g < C; ++g)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool mine = col(g) < d;
        F2 v[2];
        v[0] = v[1] = both(mine && (i == 1 || i == 2) ? 1.f : 0.f);
        if constexpr (!ANY) {
          if (src[i] && mine) load2(src[i] + col(g), v);
        } else if (mine) {
          if (src[i]) group_param<ANY>(src[i] + col(g), inside(g), 0.f, v);
          else group_clean<ANY>(inside(g), v);
        }
        if constexpr (C == 1) reg[i][0] = v[0], reg[i][1] = v[1];
        else store2(par0 + (4 * g + i) * 4 * T, v);
      }
  }
  const auto param = [&](int i, int g, F2 (&v)[2]) {
    if constexpr (C == 1) v[0] = reg[i][0], v[1] = reg[i][1];
    else load2(par0 + (4 * g + i) * 4 * T, v);
  };
  F2 aw[N], ab[N], as[N], apw[N], apb[N];
#pragma unroll
  for (int j = 0; j < N; ++j) aw[j] = ab[j] = as[j] = apw[j] = apb[j] = zero;

  const int64_t step = (int64_t)gridDim.x * R;
  const auto fetch = [&](int64_t r0, int stage) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int64_t r = r0 + i;
      if (r < a.rows) {
#pragma unroll
        for (int g = 0; g < C; ++g) {
          const int c = col(g);
          if (c >= d) continue;
          if constexpr (!ANY) {
            copy_async<L::BU>(slot(stage, i, g, L::OU, L::BU), reinterpret_cast<const TU*>(a.u) + r * a.su + c);
            copy_async<L::BX>(slot(stage, i, g, L::OX, L::BX), reinterpret_cast<const TX*>(a.x) + r * a.sx + c);
            if (a.dy) copy_async<L::BX>(slot(stage, i, g, L::ODY, L::BX), reinterpret_cast<const TX*>(a.dy) + r * d + c);
            if constexpr (GATE == 2)
              copy_async<L::BU>(slot(stage, i, g, L::OG, L::BU), reinterpret_cast<const TU*>(a.gate) + r * a.sg + c);
            if constexpr (HASZ) {
              if (zb16) copy_async<8>(slot(stage, i, g, L::OZ, 8), reinterpret_cast<const __nv_bfloat16*>(a.dz) + r * d + c);
              else copy_async<16>(slot(stage, i, g, L::OZ, 16), reinterpret_cast<const float*>(a.dz) + r * d + c);
            }
          } else {
            const auto copy = [&](uint8_t* s, const auto* p, int64_t stride) {
              group_copy<ANY>(s, p + r * stride + c, inside(g), p, p + (a.rows - 1) * stride + d);
            };
            copy(slot(stage, i, g, L::OU, L::BU), reinterpret_cast<const TU*>(a.u), a.su);
            copy(slot(stage, i, g, L::OX, L::BX), reinterpret_cast<const TX*>(a.x), a.sx);
            if (a.dy) copy(slot(stage, i, g, L::ODY, L::BX), reinterpret_cast<const TX*>(a.dy), d);
            if constexpr (GATE == 2) copy(slot(stage, i, g, L::OG, L::BU), reinterpret_cast<const TU*>(a.gate), a.sg);
            if constexpr (HASZ) {
              if (zb16) copy(slot(stage, i, g, L::OZ, 16), reinterpret_cast<const __nv_bfloat16*>(a.dz), d);
              else copy(slot(stage, i, g, L::OZ, 16), reinterpret_cast<const float*>(a.dz), d);
            }
          }
        }
        copy_async<16>(stat0 + (stage * R + i) * 16 * T, a.stats + 4 * r);
      }
    }
    copies_commit();
  };
  int flip = 0;
  int64_t r0 = (int64_t)blockIdx.x * R;
#pragma unroll
  for (int s = 0; s < ST - 1; ++s) fetch(r0 + s * step, s);
  for (int stage = 0; r0 < a.rows; r0 += step, stage = stage + 1 == ST ? 0 : stage + 1) {
    fetch(r0 + (ST - 1) * step, stage == 0 ? ST - 1 : stage - 1);
    float tok[R];
    if constexpr (GATE == 1) {
#pragma unroll
      for (int i = 0; i < R; ++i) {
        tok[i] = 0.f;
        if (r0 + i < a.rows) loadv<1>(reinterpret_cast<const TU*>(a.gate) + (r0 + i) * a.sg, &tok[i]);
      }
    }
    copies_wait<ST - 1>();
    F2 un[R][N], s[R][N], dy[R][N], yn[R][N], dn[R][N];
    float v[2 * R], ru[R], ry[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      float st[4] = {0.f, 0.f, 0.f, 0.f};
      const bool in = r0 + i < a.rows;
      if (in) loadv<4>(reinterpret_cast<const float*>(stat0 + (stage * R + i) * 16 * T), st);
      ru[i] = st[1], ry[i] = st[3];
      const F2 g1 = both(GATE == 1 ? sigmoid(tok[i]) : 1.f);
      F2 v0 = zero, v1 = zero;
#pragma unroll
      for (int g = 0; g < C; ++g) {
        F2 lu[2] = {zero, zero}, lx[2] = {zero, zero}, ly[2] = {zero, zero}, lg[2] = {one, one}, lz[2] = {zero, zero};
        if (in && col(g) < d) {
          if constexpr (!ANY) {
            load2(reinterpret_cast<const TU*>(slot(stage, i, g, L::OU, L::BU)), lu);
            if constexpr (HASZ) load2(reinterpret_cast<const TX*>(slot(stage, i, g, L::OX, L::BX)), lx);
            if (a.dy) load2(reinterpret_cast<const TX*>(slot(stage, i, g, L::ODY, L::BX)), ly);
            if constexpr (GATE == 2) load2(reinterpret_cast<const TU*>(slot(stage, i, g, L::OG, L::BU)), lg);
            if constexpr (HASZ) {
              if (zb16) load2(reinterpret_cast<const __nv_bfloat16*>(slot(stage, i, g, L::OZ, 8)), lz);
              else load2(reinterpret_cast<const float*>(slot(stage, i, g, L::OZ, 16)), lz);
            }
          } else {
            const int64_t r = r0 + i;
            const int n = inside(g);
            group_read<ANY>(slot(stage, i, g, L::OU, L::BU), reinterpret_cast<const TU*>(a.u) + r * a.su, n, lu);
            if constexpr (HASZ) group_read<ANY>(slot(stage, i, g, L::OX, L::BX), reinterpret_cast<const TX*>(a.x) + r * a.sx, n, lx);
            if (a.dy) group_read<ANY>(slot(stage, i, g, L::ODY, L::BX), reinterpret_cast<const TX*>(a.dy) + r * d, n, ly);
            if constexpr (GATE == 2)
              group_read<ANY>(slot(stage, i, g, L::OG, L::BU), reinterpret_cast<const TU*>(a.gate) + r * a.sg, n, lg);
            if constexpr (HASZ) {
              if (zb16) group_read<ANY>(slot(stage, i, g, L::OZ, 16), reinterpret_cast<const __nv_bfloat16*>(a.dz) + r * d, n, lz);
              else group_read<ANY>(slot(stage, i, g, L::OZ, 16), reinterpret_cast<const float*>(a.dz) + r * d, n, lz);
            }
          }
        }
        F2 w[2], sc[2], pw[2], pb[2];
        if constexpr (HASZ) param(0, g, w), param(1, g, sc);
        if constexpr (POST && HASZ) param(2, g, pw), param(3, g, pb);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int k = 2 * g + j;
          un[i][k] = POST ? (lu[j] + both(-st[0])) * both(ru[i]) : lu[j];
          s[i][k] = GATE == 1 ? g1 : GATE == 2 ? sigmoid(lg[j]) : one;
          dy[i][k] = ly[j];
          dn[i][k] = lz[j];
          if constexpr (HASZ) {
            const F2 p = POST ? fma(un[i][k], pw[j], pb[j]) : un[i][k];
            const F2 y = fma(GATE ? sc[j] * s[i][k] : sc[j], p, lx[j]);
            yn[i][k] = (y + both(-st[2])) * both(ry[i]);
            aw[k] = fma(dn[i][k], yn[i][k], aw[k]);
            ab[k] = ab[k] + dn[i][k];
            dn[i][k] = dn[i][k] * w[j];
            v0 = v0 + dn[i][k];
            v1 = fma(dn[i][k], yn[i][k], v1);
          }
        }
      }
      v[2 * i] = sum(v0), v[2 * i + 1] = sum(v1);
    }
    if constexpr (HASZ) {
      cta_sums<2 * R, W>(v, red[flip]);
      flip ^= 1;
    }
    float q[3 * R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int64_t r = r0 + i;
      F2 m1 = zero, m2 = zero;
      const F2 rr = both(ry[i]);
      if constexpr (HASZ) m1 = both(a.rms ? 0.f : -v[2 * i] * inv), m2 = both(-v[2 * i + 1] * inv);
      F2 q0 = zero, q1 = zero, q2 = zero;
#pragma unroll
      for (int g = 0; g < C; ++g) {
        F2 sc[2], pw[2], pb[2], ey[2], dg[2];
        param(1, g, sc);
        if constexpr (POST) param(2, g, pw), param(3, g, pb);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int k = 2 * g + j;
          if constexpr (HASZ) dy[i][k] = fma(rr, fma(yn[i][k], m2, dn[i][k] + m1), dy[i][k]);
          ey[j] = dy[i][k];
          const F2 p = POST ? fma(un[i][k], pw[j], pb[j]) : un[i][k];
          const F2 es = GATE ? ey[j] * s[i][k] : ey[j], dp = es * sc[j];
          as[k] = fma(es, p, as[k]);
          if constexpr (GATE != 0) {
            dg[j] = dp * p * fma(s[i][k], minus, one);
            if constexpr (GATE == 1) q2 = q2 + dg[j];
          }
          if constexpr (POST) {
            apw[k] = fma(dp, un[i][k], apw[k]);
            apb[k] = apb[k] + dp;
            dn[i][k] = dp * pw[j];
            q0 = q0 + dn[i][k];
            q1 = fma(dn[i][k], un[i][k], q1);
          } else {
            dn[i][k] = dp;
          }
        }
        if (r < a.rows && col(g) < d) {
          if constexpr (ANY) group_store<ANY>(reinterpret_cast<TX*>(a.dx) + r * d + col(g), inside(g), ey);
          else store2(reinterpret_cast<TX*>(a.dx) + r * d + col(g), ey);
          if constexpr (GATE == 2) if constexpr (ANY) group_store<ANY>(reinterpret_cast<TU*>(a.dgate) + r * d + col(g), inside(g), dg);
          else store2(reinterpret_cast<TU*>(a.dgate) + r * d + col(g), dg);
        }
      }
      q[3 * i] = sum(q0), q[3 * i + 1] = sum(q1), q[3 * i + 2] = sum(q2);
    }
    if constexpr (POST && GATE == 1) {
      cta_sums<3 * R, W>(q, red[flip]);
      flip ^= 1;
    } else if constexpr (POST || GATE == 1) {
      float h[2 * R];  // two sums a row, or one
      constexpr int M = POST ? 2 * R : R;
#pragma unroll
      for (int i = 0; i < R; ++i) {
        if constexpr (POST) h[2 * i] = q[3 * i], h[2 * i + 1] = q[3 * i + 1];
        else h[i] = q[3 * i + 2];
      }
      cta_sums<M, W>(h, red[flip]);
      flip ^= 1;
#pragma unroll
      for (int i = 0; i < R; ++i) {
        if constexpr (POST) q[3 * i] = h[2 * i], q[3 * i + 1] = h[2 * i + 1];
        else q[3 * i + 2] = h[i];
      }
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int64_t r = r0 + i;
      if (r >= a.rows) continue;
      const F2 m1 = both(POST && !a.rms ? -q[3 * i] * inv : 0.f), m2 = both(-q[3 * i + 1] * inv), rr = both(ru[i]);
#pragma unroll
      for (int g = 0; g < C; ++g) {
        F2 o[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int k = 2 * g + j;
          o[j] = POST ? rr * fma(un[i][k], m2, dn[i][k] + m1) : dn[i][k];
        }
        if (col(g) < d) if constexpr (ANY) group_store<ANY>(reinterpret_cast<TU*>(a.du) + r * d + col(g), inside(g), o);
        else store2(reinterpret_cast<TU*>(a.du) + r * d + col(g), o);
      }
      if constexpr (GATE == 1)
        if (t == 0) storev<1>(reinterpret_cast<TU*>(a.dgate) + r, &q[3 * i + 2]);
    }
  }
  copies_wait<0>();
#pragma unroll
  for (int g = 0; g < C; ++g) {
    if (col(g) >= d) continue;
    float* part = a.part + (int64_t)blockIdx.x * NPART * d + col(g);
    const auto put = [&](int which, const F2* v) {
      const F2 q[2] = {v[2 * g], v[2 * g + 1]};
      if constexpr (ANY) group_store<ANY>(part + which * d, inside(g), q);
      else store2(part + which * d, q);
    };
    if constexpr (HASZ) {
      put(PART_W, aw);
      if (a.b) put(PART_B, ab);
    }
    if (a.scale) put(PART_SCALE, as);
    if constexpr (POST) {
      put(PART_PW, apw);
      if (a.pb) put(PART_PB, apb);
    }
  }
}

// Threads of a backward CTA: a row's groups of four columns, in warps; C = 2: half as many.
inline int bwd_threads(int d, int c) { return ((d + 4 * c - 1) / (4 * c) + 31) / 32 * 32; }
// `many`: rows from which bwd_ring wins to 1024 values (backward of 1184, 2368, 4736 rows, bwd_kernel against
// bwd_ring: d = 256 7.2 / 5.6, 12.1 / 7.7, 20.6 / 12.4 us; d = 768 8.5 / 12.4, 13.8 / 16.1, 30.8 / 24.1;
// d = 1024 9.5 / 14.6, 16.4 / 21.1, 36.4 / 33.1; odd rows: d = 333 9.4 / 7.9, 16.1 / 12.6, 27.6 / 18.2;
// d = 1001 13.3 / 19.8, 22.0 / 29.9, 49.8 / 49.0).
inline bool many(int64_t rows, int d) { return d <= 1024 && rows >= 4 * d; }
// The same for wider rows (592, 1184, 2368 rows of 1536 values 8.0 / 10.4, 13.0 / 14.8, 28.4 / 23.5 us; of 4096
// 18.3 / 25.5, 40.0 / 37.5, 80.2 / 63.4; odd: 2368 and 4736 of 2001 55.2 / 61.9 and 113 / 111).
inline bool many_wide(int64_t rows, int d, bool any) { return d > 1024 && rows >= (any ? 4096 : d > 2048 ? 1184 : 2048); }
// The CTAs, each of which leaves one row of partials: two to an SM, more of narrow rows.
inline int bwd_grid(int64_t rows, int d) {
  const bool m = many(rows, d);
  const int T = bwd_threads(d, 1);
  const int most = 148 * (d > 2048 ? 1 : d > 1024 ? 2 : m ? std::max(2, std::min(8, 512 / T)) : 3);
  const int64_t want = m ? (rows + 1) / 2 : rows;
  return (int)(want < most ? want : most);
}

template <int NG, int GATE, bool POST, bool ANY, class TX, class TU>
cudaError_t fwd_ring_launch(const Args& a, cudaStream_t st) {
  using L = FwdRing<NG, GATE, ANY, TX, TU>;
  int params = 0;
  for (const float* p : {a.w, a.b, a.pw, a.pb, a.scale}) params += p != nullptr;
  const int smem = L::OP + params * L::D * 4;
  const auto k = fwd_ring<NG, GATE, POST, ANY, TX, TU>;
  if (smem > 48 * 1024)
    if (cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)) return e;
  // the CTAs that run at once (444 where 296 fit, 49152 x 1024: 133 us, 121 so)
  const int most = 148 * std::min(3, 228 * 1024 / (smem + 1024));
  const int64_t want = (a.rows + 7) / 8;
  k<<<(int)(want < most ? want : most), FT, smem, st>>>(a);
  return cudaGetLastError();
}
template <int NG, int GATE, bool POST, bool ANY, class TX, class TU>
cudaError_t fwd_wide_launch(const Args& a, cudaStream_t st) {
  constexpr int smem = FwdRing<NG, GATE, ANY, TX, TU>::OP;
  const auto k = fwd_wide<NG, GATE, POST, ANY, TX, TU>;
  if (smem > 47 * 1024)  // and the row sums beside it
    if (cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)) return e;
  constexpr int most = 148 * (NG == 1 ? 4 : 2);
  k<<<(int)(a.rows < most ? a.rows : most), FT, smem, st>>>(a);
  return cudaGetLastError();
}
// A CTA a row (fwd_wide) for rows wider than fwd_ring takes, for odd rows from 513 values, and for few rows,
// each by more threads (against fwd_ring, everything on: 1184 and 1776 rows of 768 values 6.2 / 8.8 and 8.1 /
// 9.0 us; 64 rows 2.7 / 7.1).  The bound is one for all widths to 768 and too high for narrow rows, most of
// whose threads hold no column: 1184 and 1776 rows of 256 values take 5.5 / 4.7 and 7.2 / 4.7 us.  Beyond 768
// values fwd_ring's slots leave two CTAs an SM (one where x and u are fp32 with a channel gate and all five
// parameters), and few means more rows (3552, 7104, 10656 rows of 1024 values 15.0 / 21.0, 27.0 / 28.2,
// 38.9 / 38.1 us; of 896 14.3 / 19.1, 26.1 / 26.1, 37.4 / 35.2; measured where two fit).
inline int few_rows(int d) { return 148 * (d > 768 ? 48 : 8); }
template <int GATE, bool POST, bool ANY, class TX, class TU>
cudaError_t fwd_width(const Args& a, cudaStream_t st) {
  const int d = a.d;
  if (d > 2048) return fwd_wide_launch<4, GATE, POST, ANY, TX, TU>(a, st);
  if (d > 1024) return fwd_wide_launch<2, GATE, POST, ANY, TX, TU>(a, st);
  if (a.rows <= few_rows(d) || (ANY && d > 512)) return fwd_wide_launch<1, GATE, POST, ANY, TX, TU>(a, st);
  if (d <= 256) return fwd_ring_launch<2, GATE, POST, ANY, TX, TU>(a, st);
  if constexpr (!ANY)
    if (d > 512) return d <= 768 ? fwd_ring_launch<6, GATE, POST, ANY, TX, TU>(a, st) : fwd_ring_launch<8, GATE, POST, ANY, TX, TU>(a, st);
  return fwd_ring_launch<4, GATE, POST, ANY, TX, TU>(a, st);
}
template <bool ANY, class TX, class TU>
cudaError_t fwd_options(const Args& a, cudaStream_t st) {
  if (a.pw)
    return a.gate_mode == 0 ? fwd_width<0, true, ANY, TX, TU>(a, st)
           : a.gate_mode == 1 ? fwd_width<1, true, ANY, TX, TU>(a, st) : fwd_width<2, true, ANY, TX, TU>(a, st);
  return a.gate_mode == 0 ? fwd_width<0, false, ANY, TX, TU>(a, st)
         : a.gate_mode == 1 ? fwd_width<1, false, ANY, TX, TU>(a, st) : fwd_width<2, false, ANY, TX, TU>(a, st);
}
template <class TX, class TU>
cudaError_t fwd_types(const Args& a, bool vec, cudaStream_t st) {
  return vec ? fwd_options<false, TX, TU>(a, st) : fwd_options<true, TX, TU>(a, st);
}

constexpr int SMEM_MOST = 227 * 1024 - 2 * 3 * 16 * 4;  // a CTA's dynamic shared memory beside bwd_ring's sums

template <int C, int GATE, bool POST, bool HASZ, bool ANY, class TX, class TU>
cudaError_t bwd_ring_launch(const Args& a, cudaStream_t st) {
  using L = BwdRing<C, GATE, HASZ, ANY, TX, TU>;
  const int T = bwd_threads(a.d, C), smem = L::thread(L::z_bytes(a.zdt == SCA2_BF16)) * T;
  const auto k = bwd_ring<C, GATE, POST, HASZ, ANY, TX, TU>;
  if (cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)) return e;
  k<<<bwd_grid(a.rows, a.d), T, smem, st>>>(a);
  return cudaGetLastError();
}
template <int C, int GATE, bool ANY, class TX, class TU>
cudaError_t bwd_ring_options(const Args& a, cudaStream_t st) {
  if (a.pw)
    return a.dz ? bwd_ring_launch<C, GATE, true, true, ANY, TX, TU>(a, st) : bwd_ring_launch<C, GATE, true, false, ANY, TX, TU>(a, st);
  return a.dz ? bwd_ring_launch<C, GATE, false, true, ANY, TX, TU>(a, st) : bwd_ring_launch<C, GATE, false, false, ANY, TX, TU>(a, st);
}
template <int C, bool ANY, class TX, class TU>
cudaError_t bwd_ring_gate(const Args& a, cudaStream_t st) {
  return a.gate_mode == 0 ? bwd_ring_options<C, 0, ANY, TX, TU>(a, st)
         : a.gate_mode == 1 ? bwd_ring_options<C, 1, ANY, TX, TU>(a, st) : bwd_ring_options<C, 2, ANY, TX, TU>(a, st);
}
template <bool CONTIG, class TX, class TU>
cudaError_t bwd_launch(const Args& a, cudaStream_t st) {
  const int d = a.d, grid = bwd_grid(a.rows, d), T = bwd_threads(d, 1);
  // The slots are counted for a channel gate and z, whatever the call has: above 3840 values rows with no
  // type of 16 bits, and those of any alignment, count as too large.
  using L = BwdRing<2, 2, true, !CONTIG, TX, TU>;
  const bool fits = d <= 1024 || L::thread(L::z_bytes(a.zdt == SCA2_BF16)) * bwd_threads(d, 2) <= SMEM_MOST;
  if ((many(a.rows, d) || many_wide(a.rows, d, !CONTIG)) && fits)
    return d <= 1024 ? bwd_ring_gate<1, !CONTIG, TX, TU>(a, st) : bwd_ring_gate<2, !CONTIG, TX, TU>(a, st);
  if (d > 2048) bwd_kernel<1024, 1, CONTIG, TX, TU><<<grid, T, 0, st>>>(a);
  else if (d > 1024) bwd_kernel<512, 2, CONTIG, TX, TU><<<grid, T, 0, st>>>(a);
  else bwd_kernel<256, 3, CONTIG, TX, TU><<<grid, T, 0, st>>>(a);
  return cudaGetLastError();
}
template <class TX, class TU>
cudaError_t bwd_types(const Args& a, bool contig, cudaStream_t st) {
  return contig ? bwd_launch<true, TX, TU>(a, st) : bwd_launch<false, TX, TU>(a, st);
}

// one translation unit for each pair of types
cudaError_t fwd_f32_f32(const Args& a, bool vec, cudaStream_t st);
cudaError_t fwd_f32_bf16(const Args& a, bool vec, cudaStream_t st);
cudaError_t fwd_bf16_f32(const Args& a, bool vec, cudaStream_t st);
cudaError_t fwd_bf16_bf16(const Args& a, bool vec, cudaStream_t st);
cudaError_t bwd_f32_f32(const Args& a, bool contig, cudaStream_t st);
cudaError_t bwd_f32_bf16(const Args& a, bool contig, cudaStream_t st);
cudaError_t bwd_bf16_f32(const Args& a, bool contig, cudaStream_t st);
cudaError_t bwd_bf16_bf16(const Args& a, bool contig, cudaStream_t st);

}  // namespace rnorm
}  // namespace sca2
