// Residual join with the norms on both sides of it, forward and backward.  Per row of width d:
//
//     p = N_post(u)  (or u),   y = x + scale * sigmoid(gate) * p,   z = N(y)
//
// N is LayerNorm (biased variance, eps inside the root, weight and optional bias) or the RMS norm
// with weight; gate is one logit for each value or for each row.  All arithmetic in fp32: y and z
// are rounded once, when stored, and z is formed from the unrounded y.  Instantiated per type of
// x and u (residual_norm_*.cu); z's type and the options are uniform runtime branches.
//
// Bound by memory.  Forward: the row stays in registers between its (up to four) reductions, so
// everything is read and written once.  Backward: recomputes p, y and the normalised rows from the
// inputs and the saved means and deviations (16 bytes a row) instead of keeping them.
#pragma once

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

__device__ __forceinline__ float sigmoid(float v) { return __fdividef(1.f, 1.f + __expf(-v)); }

__device__ __forceinline__ void unpack2(uint32_t u, float* v) {
  v[0] = __uint_as_float(u << 16), v[1] = __uint_as_float(u & 0xFFFF0000u);
}
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&p);
}

// ---- VEC values at consecutive columns (VEC = 8, 4: aligned) or one value -----------------------
template <int VEC>
__device__ __forceinline__ void loadv(const float* p, float* v) {
  if constexpr (VEC == 1) {
    v[0] = *p;
  } else {
#pragma unroll
    for (int k = 0; k < VEC / 4; ++k) {
      const float4 q = reinterpret_cast<const float4*>(p)[k];
      v[4 * k] = q.x, v[4 * k + 1] = q.y, v[4 * k + 2] = q.z, v[4 * k + 3] = q.w;
    }
  }
}
template <int VEC>
__device__ __forceinline__ void loadv(const __nv_bfloat16* p, float* v) {
  if constexpr (VEC == 1) {
    v[0] = __bfloat162float(*p);
  } else if constexpr (VEC == 4) {
    const uint2 q = *reinterpret_cast<const uint2*>(p);
    unpack2(q.x, v), unpack2(q.y, v + 2);
  } else {
    const uint4 q = *reinterpret_cast<const uint4*>(p);
    unpack2(q.x, v), unpack2(q.y, v + 2), unpack2(q.z, v + 4), unpack2(q.w, v + 6);
  }
}
template <int VEC>
__device__ __forceinline__ void storev(float* p, const float* v) {
  if constexpr (VEC == 1) {
    *p = v[0];
  } else {
#pragma unroll
    for (int k = 0; k < VEC / 4; ++k)
      reinterpret_cast<float4*>(p)[k] = make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
  }
}
template <int VEC>
__device__ __forceinline__ void storev(__nv_bfloat16* p, const float* v) {
  if constexpr (VEC == 1) {
    *p = __float2bfloat16_rn(v[0]);
  } else if constexpr (VEC == 4) {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack2(v[0], v[1]), pack2(v[2], v[3]));
  } else {
    *reinterpret_cast<uint4*>(p) =
        make_uint4(pack2(v[0], v[1]), pack2(v[2], v[3]), pack2(v[4], v[5]), pack2(v[6], v[7]));
  }
}
template <int VEC>
__device__ __forceinline__ void load_dt(const void* p, int64_t i, int dt, float* v) {
  if (dt == SCA2_BF16) loadv<VEC>(reinterpret_cast<const __nv_bfloat16*>(p) + i, v);
  else loadv<VEC>(reinterpret_cast<const float*>(p) + i, v);
}
template <int VEC>
__device__ __forceinline__ void store_dt(void* p, int64_t i, int dt, const float* v) {
  if (dt == SCA2_BF16) storev<VEC>(reinterpret_cast<__nv_bfloat16*>(p) + i, v);
  else storev<VEC>(reinterpret_cast<float*>(p) + i, v);
}

// ---- forward --------------------------------------------------------------------------------
// NT threads own a row (a warp, or the whole CTA of 256), each NV groups of VEC values: group k of
// thread t starts at column VEC (t + NT k).
constexpr int FT = 256;

template <int NT>
__device__ __forceinline__ float row_sum(float v, int& flip) {
  v = warp_sum(v);
  if constexpr (NT > 32) {
    __shared__ float s[2][NT / 32];
    if ((threadIdx.x & 31) == 0) s[flip][threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int w = 0; w < NT / 32; ++w) v += s[flip][w];
    flip ^= 1;  // the next sum's writes pass this one's reads only after its own barrier
  }
  return v;
}

template <int NT, int NV, int VEC, class TX, class TU>
__global__ void __launch_bounds__(FT, NT == 32 && NV > 2 ? 2 : 3) fwd_kernel(const Args a) {
  const int t = threadIdx.x % NT;
  const int d = a.d;
  const float inv = 1.f / (float)d;
  int flip = 0;
  const auto col = [&](int k) { return VEC * (t + NT * k); };
  // mean and 1 / deviation of v, then v <- (v - mean) / deviation
  const auto normalise = [&](float (&v)[NV][VEC], float& mu, float& rs) {
    mu = 0.f;
    if (!a.rms) {
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int j = 0; j < VEC; ++j) s += v[k][j];  // columns past d hold 0
      mu = row_sum<NT>(s, flip) * inv;
    }
    float q = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (col(k) < d) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[k][j] -= mu, q = fmaf(v[k][j], v[k][j], q);
      }
    rs = rsqrtf(row_sum<NT>(q, flip) * inv + a.eps);
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[k][j] *= rs;
  };
  const auto affine = [&](float (&v)[VEC], const float* w, const float* b, int c) {
    float q[VEC];
    loadv<VEC>(w + c, q);
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] *= q[j];
    if (b) {
      loadv<VEC>(b + c, q);
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[j] += q[j];
    }
  };

  const int64_t step = (int64_t)gridDim.x * (FT / NT);
  for (int64_t row = (int64_t)blockIdx.x * (FT / NT) + threadIdx.x / NT; row < a.rows; row += step) {
    const TX* xr = reinterpret_cast<const TX*>(a.x) + row * a.sx;
    const TU* ur = reinterpret_cast<const TU*>(a.u) + row * a.su;
    const TU* gr = reinterpret_cast<const TU*>(a.gate) + row * a.sg;
    float x[NV][VEC], p[NV][VEC], g[NV][VEC];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) x[k][j] = p[k][j] = g[k][j] = 0.f;
      if (col(k) < d) {
        loadv<VEC>(ur + col(k), p[k]);
        loadv<VEC>(xr + col(k), x[k]);
        if (a.gate_mode == 2) loadv<VEC>(gr + col(k), g[k]);
      }
    }
    float gt = 1.f;
    if (a.gate_mode == 1) loadv<1>(gr, &gt), gt = sigmoid(gt);
    float mu = 0.f, rs = 0.f;
    if (a.pw) {
      normalise(p, mu, rs);
#pragma unroll
      for (int k = 0; k < NV; ++k)
        if (col(k) < d) affine(p[k], a.pw, a.pb, col(k));
    }
    if (a.stats && t == 0) a.stats[4 * row] = mu, a.stats[4 * row + 1] = rs;
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (col(k) < d) {
        float s[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) s[j] = 1.f;
        if (a.scale) loadv<VEC>(a.scale + col(k), s);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          if (a.gate_mode == 2) s[j] *= sigmoid(g[k][j]);
          else s[j] *= gt;
          x[k][j] = fmaf(s[j], p[k][j], x[k][j]);
        }
        storev<VEC>(reinterpret_cast<TX*>(a.y) + row * d + col(k), x[k]);
      }
    if (!a.z) continue;
    normalise(x, mu, rs);
    if (a.stats && t == 0) a.stats[4 * row + 2] = mu, a.stats[4 * row + 3] = rs;
#pragma unroll
    for (int k = 0; k < NV; ++k)
      if (col(k) < d) {
        affine(x[k], a.w, a.b, col(k));
        store_dt<VEC>(a.z, row * d + col(k), a.zdt, x[k]);
      }
  }
}

// ---- backward -------------------------------------------------------------------------------
// A thread owns four columns of every row (4t ... 4t+3, or t + T k where rows are not aligned), so
// the five column sums stay in its registers over all its rows; R rows are in flight at once,
// which hides their loads and shares the two barriers of their row sums.
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

template <int MAXT, int R, int MINB, bool CONTIG, class TX, class TU>
__global__ void __launch_bounds__(MAXT, MINB) bwd_kernel(const Args a) {
  constexpr int W = MAXT <= 256 ? 8 : MAXT / 32;
  __shared__ __align__(16) float red[2][3 * R * W];
  const int t = threadIdx.x, T = blockDim.x, d = a.d;
  const float inv = 1.f / (float)d;
  for (int i = t; i < 2 * 3 * R * W; i += T) (&red[0][0])[i] = 0.f;
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

  for (int64_t r0 = (int64_t)blockIdx.x * R; r0 < a.rows; r0 += (int64_t)gridDim.x * R) {
    // per row: un (normalised u, or u), s (the gate), dy, then yn and dn of z
    float un[R][4], s[R][4], dy[R][4], yn[R][4], dn[R][4], st[R][4];
#pragma unroll
    for (int i = 0; i < R; ++i) {
#pragma unroll
      for (int k = 0; k < 4; ++k) un[i][k] = s[i][k] = dy[i][k] = yn[i][k] = dn[i][k] = st[i][k] = 0.f;
      const int64_t r = r0 + i;
      if (r < a.rows) {
        load(reinterpret_cast<const TU*>(a.u) + r * a.su, un[i]);
        load(reinterpret_cast<const TX*>(a.x) + r * a.sx, yn[i]);
        if (chan) load(reinterpret_cast<const TU*>(a.gate) + r * a.sg, s[i]);
        if (token) {
          float g;
          loadv<1>(reinterpret_cast<const TU*>(a.gate) + r * a.sg, &g);
#pragma unroll
          for (int k = 0; k < 4; ++k) s[i][k] = g;
        }
        if (a.dy) load(reinterpret_cast<const TX*>(a.dy) + r * d, dy[i]);
        if (has_z) {
          if (a.zdt == SCA2_BF16) load(reinterpret_cast<const __nv_bfloat16*>(a.dz) + r * d, dn[i]);
          else load(reinterpret_cast<const float*>(a.dz) + r * d, dn[i]);
        }
        loadv<4>(a.stats + 4 * r, st[i]);
      }
    }
    float v[3 * R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      v[2 * i] = v[2 * i + 1] = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (post) un[i][k] = (un[i][k] - st[i][0]) * st[i][1];
        s[i][k] = a.gate_mode ? sigmoid(s[i][k]) : 1.f;
        if (has_z) {
          const float y = fmaf(sc[k] * s[i][k], fmaf(un[i][k], pw[k], pb[k]), yn[i][k]);
          yn[i][k] = (y - st[i][2]) * st[i][3];
          aw[k] = fmaf(dn[i][k], yn[i][k], aw[k]);
          ab[k] += dn[i][k];
          dn[i][k] *= w[k];
          v[2 * i] += dn[i][k];
          v[2 * i + 1] = fmaf(dn[i][k], yn[i][k], v[2 * i + 1]);
        }
      }
    }
    if (has_z) {
      cta_sums<2 * R, W>(v, red[flip]);
      flip ^= 1;
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int64_t r = r0 + i;
      float dg[4];
      if (has_z) {
        const float m1 = a.rms ? 0.f : v[2 * i] * inv, m2 = v[2 * i + 1] * inv;
#pragma unroll
        for (int k = 0; k < 4; ++k) dy[i][k] += st[i][3] * (dn[i][k] - m1 - yn[i][k] * m2);
      }
      if (r < a.rows) store(reinterpret_cast<TX*>(a.dx) + r * d, dy[i]);
      float q0 = 0.f, q1 = 0.f, q2 = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float e = dy[i][k];
        const float p = fmaf(un[i][k], pw[k], pb[k]);
        as[k] = fmaf(e * s[i][k], p, as[k]);
        dg[k] = e * sc[k] * p * s[i][k] * (1.f - s[i][k]);
        q2 += dg[k];
        const float dp = e * sc[k] * s[i][k];
        apw[k] = fmaf(dp, un[i][k], apw[k]);
        apb[k] += dp;
        dn[i][k] = dp * pw[k];
        q0 += dn[i][k];
        q1 = fmaf(dn[i][k], un[i][k], q1);
      }
      if (chan && r < a.rows) store(reinterpret_cast<TU*>(a.dgate) + r * d, dg);
      s[i][0] = q0, s[i][1] = q1, s[i][2] = q2;  // the gate's values are done with
    }
    if (post || token) {
#pragma unroll
      for (int i = 0; i < R; ++i) v[3 * i] = s[i][0], v[3 * i + 1] = s[i][1], v[3 * i + 2] = s[i][2];
      cta_sums<3 * R, W>(v, red[flip]);
      flip ^= 1;
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int64_t r = r0 + i;
      if (r >= a.rows) continue;
      if (post) {
        const float m1 = a.rms ? 0.f : v[3 * i] * inv, m2 = v[3 * i + 1] * inv;
#pragma unroll
        for (int k = 0; k < 4; ++k) dn[i][k] = st[i][1] * (dn[i][k] - m1 - un[i][k] * m2);
      }
      store(reinterpret_cast<TU*>(a.du) + r * d, dn[i]);
      if (token && t == 0) storev<1>(reinterpret_cast<TU*>(a.dgate) + r, &v[3 * i + 2]);
    }
  }
  float* part = a.part + (int64_t)blockIdx.x * NPART * d;
  if (has_z) store(part + PART_W * d, aw);
  if (has_z && a.b) store(part + PART_B * d, ab);
  if (a.scale) store(part + PART_SCALE * d, as);
  if (post) store(part + PART_PW * d, apw);
  if (post && a.pb) store(part + PART_PB * d, apb);
}

// rows in flight in a CTA, and the CTAs (each leaves one row of partials)
inline int bwd_rows_per_step(int64_t rows, int d) { return d > 1024 ? 1 : rows >= 148 * 6 ? 2 : 1; }
inline int bwd_grid(int64_t rows, int d) {
  const int R = bwd_rows_per_step(rows, d), most = 148 * (d > 2048 ? 1 : d > 1024 ? 2 : 3);
  const int64_t want = (rows + R - 1) / R;
  return (int)(want < most ? want : most);
}

template <class TX, class TU>
cudaError_t fwd_types(const Args& a, bool vec, cudaStream_t st) {
  const int d = a.d;
  const bool warp = vec && d <= 1024;
  const int64_t want = warp ? (a.rows + 7) / 8 : a.rows;
  const int grid = (int)(want < 148 * 8 ? want : 148 * 8);
  if (warp) {
    switch ((d + 255) / 256) {
      case 1: fwd_kernel<32, 1, 8, TX, TU><<<grid, FT, 0, st>>>(a); break;
      case 2: fwd_kernel<32, 2, 8, TX, TU><<<grid, FT, 0, st>>>(a); break;
      case 3: fwd_kernel<32, 3, 8, TX, TU><<<grid, FT, 0, st>>>(a); break;
      default: fwd_kernel<32, 4, 8, TX, TU><<<grid, FT, 0, st>>>(a); break;
    }
  } else if (vec) {
    if (d <= 2048) fwd_kernel<256, 1, 8, TX, TU><<<grid, FT, 0, st>>>(a);
    else fwd_kernel<256, 2, 8, TX, TU><<<grid, FT, 0, st>>>(a);
  } else {
    if (d <= 1024) fwd_kernel<256, 4, 1, TX, TU><<<grid, FT, 0, st>>>(a);
    else fwd_kernel<256, 16, 1, TX, TU><<<grid, FT, 0, st>>>(a);
  }
  return cudaGetLastError();
}

template <bool CONTIG, class TX, class TU>
cudaError_t bwd_launch(const Args& a, cudaStream_t st) {
  const int d = a.d, R = bwd_rows_per_step(a.rows, d), grid = bwd_grid(a.rows, d);
  const int T = ((d + 3) / 4 + 31) / 32 * 32;
  if (d > 2048) bwd_kernel<1024, 1, 1, CONTIG, TX, TU><<<grid, T, 0, st>>>(a);
  else if (d > 1024) bwd_kernel<512, 1, 2, CONTIG, TX, TU><<<grid, T, 0, st>>>(a);
  else if (R == 2 && T <= 192) bwd_kernel<192, 2, 3, CONTIG, TX, TU><<<grid, T, 0, st>>>(a);
  else if (R == 2) bwd_kernel<256, 2, 2, CONTIG, TX, TU><<<grid, T, 0, st>>>(a);
  else bwd_kernel<256, 1, 3, CONTIG, TX, TU><<<grid, T, 0, st>>>(a);
  return cudaGetLastError();
}
template <class TX, class TU>
cudaError_t bwd_types(const Args& a, bool contig, cudaStream_t st) {
  return contig ? bwd_launch<true, TX, TU>(a, st) : bwd_launch<false, TX, TU>(a, st);
}

// one translation unit for each type of x
cudaError_t fwd_f32(const Args& a, int udt, bool vec, cudaStream_t st);
cudaError_t fwd_bf16(const Args& a, int udt, bool vec, cudaStream_t st);
cudaError_t bwd_f32(const Args& a, int udt, bool contig, cudaStream_t st);
cudaError_t bwd_bf16(const Args& a, int udt, bool contig, cudaStream_t st);

}  // namespace rnorm
}  // namespace sca2
