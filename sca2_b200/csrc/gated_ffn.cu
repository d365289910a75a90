// Gated feed-forward projections, forward and backward (bf16 in and out, fp32 accumulation):
//
//     g = x Wg^T,  u = x Wu^T,  h = act(g) * u                     x (rows, d), W (f, d), h (rows, f)
//     dg = dh u act'(g),  du = dh act(g)
//     dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x
//
// Four kinds of product share one kernel, `ffn_gemm<KIND>`: a pair of CTAs (cta_group::2) computes a
// 256 x 256 tile with tcgen05.mma, the operands staged by TMA in 128-byte swizzled tiles of 64
// contraction steps, one mbarrier ring, the accumulator double-buffered in TMEM (2 x 256 columns)
// so that the epilogue of a tile runs under the products of the next; tiles are dealt to the pairs
// in a fixed order.  The launches: FWD; BACK; GRADS, which holds DW and DX.
//   FWD   tile = 256 rows x (128 gate columns | the same 128 up columns): CTA 0 of the pair stages
//         Wg's rows and CTA 1 Wu's, so one accumulator row holds g and u of a column and the
//         epilogue forms h without a trip to memory.
//   BACK  the same product again with dh: g and u are recomputed in fp32 rather than kept (which
//         would cost 2 rows f bf16 values of memory for the whole step and a rounding of both).
//         dg and du are rounded to bf16 once, as operands of the next two products (two bf16 terms of
//         each would double those).  That shows in the gradients: in the 2-norm they are 0.0023 off 64
//         bits, 0.0017 if dg and du kept 32 bits until the gradients themselves are rounded.
//   DX    contraction over f twice, (dg, Wg) then (du, Wu), one accumulator; the weights are read
//         as they lie (MN-major operand), no transposed copy.
//   DW    contraction over the rows, both operands MN-major; split over the rows where the tiles
//         alone do not fill the machine, the fp32 parts added in a fixed order by `dw_reduce`.
//   GRADS gives each pair its DW tiles (few and long) and then as many of the DX tiles (many and
//         short) as even out the pairs' contraction blocks, so neither has a last round of its own:
//         65536 x 768 -> 2048 555 us for both, 580 as two launches and a pass over split parts.
// Ragged sizes: TMA fills what lies outside with zeros and clips what is stored there.
//
// Measured (one B200): 32768 x 1024 -> 4096 forward 420 to 430 us called back to back (1280 to 1310
// TFLOP/s, 92% of what cuBLAS sustains under the power limit), 360 us in short bursts (1530, 91% of its
// burst).  In short bursts 65536 x 768 -> 2048: forward 290 us, BACK 340, GRADS 555.  Bound by
// the tensor cores under the power limit: a contraction block of a tile takes 0.37 us at any width,
// which is cuBLAS's rate; at d = 768 the epilogue and the switch of tiles add 15%, in BACK 30% (half of
// that its stores).  L2 prefetches of the operands by TMA slowed every product (360 -> 400 us).
//
// Up to FEW_ROWS rows (decode) the forward is bound by reading the weights and by latency:
// `ffn_few` keeps no tiles, each warp streams weight rows straight into mma.sync fragments.
//
// Every wait is bounded: a wait that runs out sets the fault word, and the kernel leaves once its copies
// and products in flight are done (waits that are bounded too).
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <cstring>
#include <string>

#include "common.cuh"
#include "umma.cuh"

namespace sca2 {
void set_last_error(const std::string& msg);
PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder();

namespace ffn {

using umma::smem_u32;

__device__ unsigned int g_fault_ffn;

enum Mode { FWD, BACK, DX, DW, GRADS };
enum Act { SILU, GELU };

constexpr int BK = 64;               // contraction steps of a stage: 128 bytes, one swizzle row
constexpr int HALF = 128 * BK * 2;   // one operand of one CTA's stage, 16 KB
constexpr int EPI_WARPS = 16;        // four to a quarter of the rows, each a quarter of the columns
constexpr int NT = 128 + 32 * EPI_WARPS;
constexpr int STG = 2048;            // one staged output block: 32 rows of 64 bytes
constexpr uint64_t WAIT_NS = 4000000000ull;  // a wait gives up after this

template <int KIND>
struct Layout {
  static constexpr int STAGES = KIND == FWD ? 6 : 5;
  static constexpr int NSTG = KIND == FWD ? 1 : 2;  // staged output blocks of a warp
  static constexpr int RING = STAGES * 2 * HALF;
  static constexpr int BARS = RING + EPI_WARPS * NSTG * STG;
  static constexpr int TOTAL = BARS + 320 + 1024;  // 1024: room to align the ring
};

struct Geo {
  int rows, d, f;
  int tiles_n, tiles_m, slices, splits;  // unit = ((split * slices + slice) * tiles_m + m) * tiles_n + n
  int units;                             // of FWD or BACK, or those of DW
  int kb, kb_half;                       // contraction blocks of a whole tile; DX: those of one half
  int kb_split, kb_more;                 // those of a split, and how many splits have one more
  int sn, sm, ss, sp;                    // the grid's pairs as digits of a unit
  int x_units, x_pairs, x_a, x_b;        // DX: units; a pair below x_pairs takes up to x_a of them, another x_b
};

struct Maps {
  CUtensorMap a0, a1, b0, b1, o0, o1, dh;  // GRADS: a0, a1, b0, o0, o1 of DW
  CUtensorMap xa0, xa1, xb0, xb1, xo;      // and those of DX
};

// ---- cluster, barrier and TMA primitives ---------------------------------------------------
__device__ __forceinline__ uint32_t cta_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t map_to(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ bool try_wait(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return done;
}
__device__ __forceinline__ uint64_t now_ns() {
  uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
__device__ __forceinline__ bool wait_for(uint32_t bar, uint32_t parity) {
  if (try_wait(bar, parity)) return true;
  const uint64_t t0 = now_ns();
  while (!try_wait(bar, parity))
    if (now_ns() - t0 > WAIT_NS) {
      atomicOr(&g_fault_ffn, 1u);
      return false;
    }
  return true;
}
__device__ __forceinline__ void expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
// load of a box into this CTA's shared memory, completing on a barrier of either CTA of the pair
__device__ __forceinline__ void load2(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, "
      "%3}], [%4];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void load1(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::
          "r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void store2d(const CUtensorMap* map, uint32_t src, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(x),
               "r"(y), "r"(src)
               : "memory");
}
__device__ __forceinline__ void store3d(const CUtensorMap* map, uint32_t src, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(map),
               "r"(x), "r"(y), "r"(z), "r"(src)
               : "memory");
}
__device__ __forceinline__ void stores_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void stores_read() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void stores_done() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

__device__ __forceinline__ void mma2(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
// arrive on the barrier at this offset in the CTAs of `mask` (both) once the products issued so far are done
__device__ __forceinline__ void commit2(uint32_t bar, uint16_t mask = 3) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
      "h"(mask)
      : "memory");
}
__device__ __forceinline__ void ld32(uint32_t t, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,"
      "%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(t));
}

// Descriptors of a 128-byte swizzled tile (layout type 2 in bits 61-63, version 1 in bit 46).
// K-major: rows of 64 contraction steps, 8-row groups 1024 bytes apart; 16 steps on are 32 bytes on.
// MN-major: blocks of 64 columns, in each one 128-byte row per contraction step; 8 steps are 1024
// bytes apart, the next 64 columns 8192; 16 steps on are 2048 bytes on.
__device__ __forceinline__ uint64_t desc_k(uint32_t s) {
  return (uint64_t)((s >> 4) & 0x3FFFu) | (uint64_t)1 << 16 | (uint64_t)64 << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
__device__ __forceinline__ uint64_t desc_mn(uint32_t s) {
  return (uint64_t)((s >> 4) & 0x3FFFu) | (uint64_t)512 << 16 | (uint64_t)64 << 32 | (uint64_t)1 << 46 |
         (uint64_t)2 << 61;
}

// ---- activations -----------------------------------------------------------------------------
// The special function unit's 2^x and 1 / x without the handling of denormals around them: the
// epilogues run beside the products and are bound by their instructions.  Relative error about
// 2^-22; an overflow gives inf, and its reciprocal the 0 that the sigmoid has there.
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
__device__ __forceinline__ float sigmoid(float g) { return rcp_fast(1.f + exp2_fast(-LOG2E * g)); }

template <int ACT>
__device__ __forceinline__ float act_of(float g) {
  if constexpr (ACT == SILU) return g * sigmoid(g);
  else return g * fmaf(0.5f, erff(g * 0.70710678f), 0.5f);
}
// the activation and its derivative
template <int ACT>
__device__ __forceinline__ void act_grad(float g, float& a, float& da) {
  if constexpr (ACT == SILU) {
    const float s = sigmoid(g);
    a = g * s;
    da = fmaf(a, 1.f - s, s);  // s (1 + g (1 - s))
  } else {
    const float p = fmaf(0.5f, erff(g * 0.70710678f), 0.5f);
    a = g * p;
    da = fmaf(g * 0.39894228f, exp2_fast(-0.5f * LOG2E * g * g), p);
  }
}
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&p);
}
__device__ __forceinline__ float lo(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float hi(uint32_t u) { return __uint_as_float(u & 0xFFFF0000u); }

// 16-byte chunk c of row r of a staged block, in the 64-byte swizzle (8 rows' stores of one chunk
// fall on 8 different 16-byte columns of the banks)
__device__ __forceinline__ uint32_t chunk(uint32_t base, int r, int c) {
  return base + (uint32_t)(r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
}
__device__ __forceinline__ void sts4(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ uint4 lds4(uint32_t a) {
  uint4 q;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w) : "r"(a) : "memory");
  return q;
}

// A pair's units, `step` apart.  The step is kept as digits (Geo::s*) and added with carries: a
// division for each tile would stall the one thread that issues the products between two tiles.
struct Unit {
  int n, m, slice, split;
  __device__ __forceinline__ void first(const Geo& g, int u) {
    n = u % g.tiles_n, u /= g.tiles_n;
    m = u % g.tiles_m, u /= g.tiles_m;
    slice = u % g.slices, split = u / g.slices;
  }
  __device__ __forceinline__ void next(const Geo& g) {
    n += g.sn;
    const int c = n >= g.tiles_n;
    n -= c ? g.tiles_n : 0;
    m += g.sm + c;
    const int e = m >= g.tiles_m;
    m -= e ? g.tiles_m : 0;
    slice += g.ss + e;
    const int f = slice >= g.slices;
    slice -= f ? g.slices : 0;
    split += g.sp + f;
  }
  // DX: a unit, and the one `step` (as digits) on
  __device__ __forceinline__ void first_x(const Geo& g, int u) { n = u % g.tiles_n, m = u / g.tiles_n, slice = split = 0; }
  __device__ __forceinline__ void next_x(const Geo& g, int step_n, int step_m) {
    n += step_n;
    const int c = n >= g.tiles_n;
    n -= c ? g.tiles_n : 0, m += step_m + c;
  }
  // its contraction blocks: the first `kb_more` splits have one more
  __device__ __forceinline__ int k0(const Geo& g) const { return split * g.kb_split + (split < g.kb_more ? split : g.kb_more); }
  __device__ __forceinline__ int k1(const Geo& g) const { return k0(g) + g.kb_split + (split < g.kb_more ? 1 : 0); }
};

template <int M>
struct ModeOf {
  static constexpr int value = M;
};

// f(mode, unit) for the pair's units in order; false from f ends it
template <int KIND, class F>
__device__ __forceinline__ void for_units(const Geo& g, int pair, int pairs, F f) {
  Unit t;
  if (pair < g.units) {
    t.first(g, pair);
    for (int u = pair; u < g.units; u += pairs, t.next(g))
      if (!f(ModeOf<KIND == GRADS ? DW : KIND>{}, t)) return;
  }
  if constexpr (KIND == GRADS) {
    // pairs with equally many DW units come here together and take the DX units of their share in
    // turn: neighbours have the same rows, which reach L2 once
    const bool a = pair < g.x_pairs;
    const int step = a ? g.x_pairs : pairs - g.x_pairs, count = a ? g.x_a : g.x_b;
    int u = a ? pair : g.x_a * g.x_pairs + (pair - g.x_pairs);
    if (count == 0 || u >= g.x_units) return;
    t.first_x(g, u);
    const int step_n = step % g.tiles_n, step_m = step / g.tiles_n;
    for (int i = 0; i < count && u < g.x_units; ++i, u += step, t.next_x(g, step_n, step_m))
      if (!f(ModeOf<DX>{}, t)) return;
  }
}

template <int KIND, int ACT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(NT, 1) ffn_gemm(const __grid_constant__ Maps maps, const Geo g) {
  using L = Layout<KIND>;
  constexpr int ST = L::STAGES;
  extern __shared__ uint8_t raw[];
  const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;  // the same offset in both CTAs
  const uint32_t stg0 = base + L::RING, bars = base + L::BARS;
  const uint32_t full = bars, empty = bars + 8 * ST, tfull = bars + 16 * ST, tempty = tfull + 16, dhbar = tempty + 16,
                 slot = dhbar + 8 * EPI_WARPS, done = slot + 8;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cta_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    const auto init = [](uint32_t b, uint32_t n) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(b), "r"(n) : "memory");
    };
    for (int s = 0; s < ST; ++s) init(full + 8 * s, 1), init(empty + 8 * s, 1);
    for (int s = 0; s < 2; ++s) init(tfull + 8 * s, 1), init(tempty + 8 * s, 2 * EPI_WARPS);
    for (int s = 0; s < EPI_WARPS; ++s) init(dhbar + 8 * s, 1);
    init(done, 1);
    umma::fence_mbar_init();
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(slot) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  umma::fence_before_sync();
  __syncthreads();
  cluster_sync();
  umma::fence_after_sync();
  uint32_t tmem;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(tmem) : "r"(slot));

  if (warp == 0) {
    if (lane == 0) {  // ---- producer: this CTA's half of both operands
      const uint32_t full0 = map_to(full, 0);
      int s = 0, ph = 1, issued = 0;
      bool ok = true;
      for_units<KIND>(g, pair, pairs, [&](auto mode, const Unit& t) {
        constexpr int MODE = decltype(mode)::value;
        const int k0 = MODE == DW ? t.k0(g) : 0, k1 = MODE == DX ? 2 * g.kb_half : MODE == DW ? t.k1(g) : g.kb;
        for (int k = k0; k < k1; ++k) {
          if (!(ok = wait_for(empty + 8 * s, ph))) return false;
          if (rank == 0) expect(full + 8 * s, 4 * HALF);
          const uint32_t A = base + s * 2 * HALF, B = A + HALF, bar = full0 + 8 * s;
          if constexpr (MODE == FWD || MODE == BACK) {
            load2(A, &maps.a0, k * BK, t.m * 256 + 128 * rank, bar);
            load2(B, rank ? &maps.b1 : &maps.b0, k * BK, t.n * 128, bar);
          } else if constexpr (MODE == DX) {
            const bool up = k >= g.kb_half;
            const int kk = (up ? k - g.kb_half : k) * BK, n = t.n * 256 + 128 * rank;
            const CUtensorMap* w = up ? &maps.xb1 : &maps.xb0;
            load2(A, up ? &maps.xa1 : &maps.xa0, kk, t.m * 256 + 128 * rank, bar);
            load2(B, w, n, kk, bar);
            load2(B + HALF / 2, w, n + 64, kk, bar);
          } else {
            const CUtensorMap* a = t.slice ? &maps.a1 : &maps.a0;
            const int m = t.m * 256 + 128 * rank, n = t.n * 256 + 128 * rank;
            load2(A, a, m, k * BK, bar);
            load2(A + HALF / 2, a, m + 64, k * BK, bar);
            load2(B, &maps.b0, n, k * BK, bar);
            load2(B + HALF / 2, &maps.b0, n + 64, k * BK, bar);
          }
          if (++s == ST) s = 0, ph ^= 1;
          issued = issued < ST ? issued + 1 : ST;
        }
        return true;
      });
      if (rank == 0)  // leave no copy in flight, whichever wait ran out: both CTAs' copies complete on these
        for (; issued > 0; --issued) {
          if (--s < 0) s = ST - 1, ph ^= 1;
          if (!wait_for(full + 8 * s, ph ^ 1)) break;
        }
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {  // ---- products of both CTAs
      int n = 0, s = 0, ph = 0;
      for_units<KIND>(g, pair, pairs, [&](auto mode, const Unit& t) {
        constexpr int MODE = decltype(mode)::value;
        constexpr bool a_mn = MODE == DW, b_mn = MODE == DX || MODE == DW;
        constexpr uint32_t id = umma::idesc_bf16_t(256, 256, a_mn, b_mn);
        const int acc = n & 1, kn = MODE == DX ? 2 * g.kb_half : MODE == DW ? t.k1(g) - t.k0(g) : g.kb;
        if (!wait_for(tempty + 8 * acc, ((n >> 1) & 1) ^ 1)) return false;
        umma::fence_after_sync();
        for (int k = 0; k < kn; ++k) {
          if (!wait_for(full + 8 * s, ph)) return false;
          umma::fence_after_sync();
          const uint32_t A = base + s * 2 * HALF, B = A + HALF;
          const uint64_t da = a_mn ? desc_mn(A) : desc_k(A), db = b_mn ? desc_mn(B) : desc_k(B);
#pragma unroll
          for (int j = 0; j < BK / 16; ++j)  // 16 steps on: 2048 / 16 or 32 / 16 in the address field
            mma2(tmem + 256 * acc, da + (a_mn ? 128 : 2) * j, db + (b_mn ? 128 : 2) * j, id, k > 0 || j > 0);
          commit2(empty + 8 * s);
          if (++s == ST) s = 0, ph ^= 1;
        }
        commit2(tfull + 8 * acc);
        ++n;
        return true;
      });
      commit2(done, 1);  // nor a product, whose operands and accumulator are about to be given up
      wait_for(done, 0);
    }
  } else if (warp >= 4) {  // ---- epilogue: 32 rows (the warp's quarter of TMEM) x a quarter of the columns
    const int e = warp - 4, q = warp & 3, part = e >> 2;
    const uint32_t stg = stg0 + e * L::NSTG * STG, dhb = dhbar + 8 * e, tempty0 = map_to(tempty, 0);
    int n = 0;
    for_units<KIND>(g, pair, pairs, [&](auto mode, const Unit& t) {
      constexpr int MODE = decltype(mode)::value;
      const int acc = n & 1;
      const int row = t.m * 256 + 128 * rank + 32 * q;
      const uint32_t tm = umma::taddr(tmem, 32 * q, 256 * acc);
      const int hc = t.n * 128 + 32 * part;  // FWD, BACK: first of the warp's 32 columns of h
      if constexpr (MODE == BACK) {
        if (lane == 0) {
          stores_read<0>();
          expect(dhb, STG);
          load1(stg, &maps.dh, hc, row, dhb);
        }
      }
      if (!__all_sync(0xffffffffu, wait_for(tfull + 8 * acc, (n >> 1) & 1))) {
        if constexpr (MODE == BACK) wait_for(dhb, n & 1);  // the copy of dh is in flight
        return false;
      }
      umma::fence_after_sync();
      if constexpr (MODE == FWD || MODE == BACK) {
        uint32_t rg[32], ru[32];
        float vg[32], vu[32];
        ld32(tm + 32 * part, rg);
        ld32(tm + 128 + 32 * part, ru);
        umma::ld_wait();
        umma::take<32>(rg, vg);
        umma::take<32>(ru, vu);
        // the accumulator is in registers: the products of the tile after next may have it
        umma::fence_before_sync();
        __syncwarp();
        if (lane == 0) arrive_cluster(tempty0 + 8 * acc);
        if constexpr (MODE == BACK) {
          if (!__all_sync(0xffffffffu, wait_for(dhb, n & 1))) return false;
        } else {
          if (lane == 0) stores_read<0>();
          __syncwarp();
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t at = chunk(stg, lane, j);
          if constexpr (MODE == FWD) {
            float h[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) h[i] = act_of<ACT>(vg[8 * j + i]) * vu[8 * j + i];
            sts4(at, pack2(h[0], h[1]), pack2(h[2], h[3]), pack2(h[4], h[5]), pack2(h[6], h[7]));
          } else {
            const uint4 w = lds4(at);
            const float dh[8] = {lo(w.x), hi(w.x), lo(w.y), hi(w.y), lo(w.z), hi(w.z), lo(w.w), hi(w.w)};
            float dg[8], du[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              float a, da;
              act_grad<ACT>(vg[8 * j + i], a, da);
              dg[i] = dh[i] * vu[8 * j + i] * da;
              du[i] = dh[i] * a;
            }
            sts4(chunk(stg + STG, lane, j), pack2(dg[0], dg[1]), pack2(dg[2], dg[3]), pack2(dg[4], dg[5]),
                 pack2(dg[6], dg[7]));
            sts4(at, pack2(du[0], du[1]), pack2(du[2], du[3]), pack2(du[4], du[5]), pack2(du[6], du[7]));
          }
        }
        umma::fence_async_smem();
        __syncwarp();
        if (lane == 0) {
          if (row < g.rows && hc < g.f) {
            if constexpr (MODE == FWD) {
              store2d(&maps.o0, stg, hc, row);
            } else {
              store2d(&maps.o0, stg + STG, hc, row);
              store2d(&maps.o1, stg, hc, row);
            }
          }
          stores_commit();
        }
      } else {
        const int limit = MODE == DX ? g.rows : g.f;
        const bool parts = MODE == DW && g.splits > 1;
#pragma unroll
        for (int c = 0; c < 2; ++c) {  // 32 columns at a time
          uint32_t r[32];
          float v[32];
          ld32(tm + 64 * part + 32 * c, r);
          umma::ld_wait();
          umma::take<32>(r, v);
          if (c == 1) {
            umma::fence_before_sync();
            __syncwarp();
            if (lane == 0) arrive_cluster(tempty0 + 8 * acc);
          }
          const int col = t.n * 256 + 64 * part + 32 * c;
          if (parts) {  // 16 fp32 columns fill a staged block
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              if (lane == 0) stores_read<1>();
              __syncwarp();
#pragma unroll
              for (int j = 0; j < 4; ++j)
                sts4(chunk(stg + k * STG, lane, j), __float_as_uint(v[16 * k + 4 * j]), __float_as_uint(v[16 * k + 4 * j + 1]),
                     __float_as_uint(v[16 * k + 4 * j + 2]), __float_as_uint(v[16 * k + 4 * j + 3]));
              umma::fence_async_smem();
              __syncwarp();
              if (lane == 0) {
                if (row < limit && col + 16 * k < g.d)
                  store3d(&maps.o0, stg + k * STG, col + 16 * k, row, t.split * 2 + t.slice);
                stores_commit();
              }
            }
          } else {  // 32 bf16 columns do
            if (lane == 0) stores_read<1>();
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 4; ++j)
              sts4(chunk(stg + c * STG, lane, j), pack2(v[8 * j], v[8 * j + 1]), pack2(v[8 * j + 2], v[8 * j + 3]),
                   pack2(v[8 * j + 4], v[8 * j + 5]), pack2(v[8 * j + 6], v[8 * j + 7]));
            umma::fence_async_smem();
            __syncwarp();
            if (lane == 0) {
              if (row < limit && col < g.d)
                store2d(MODE == DX ? &maps.xo : t.slice ? &maps.o1 : &maps.o0, stg + c * STG, col, row);
              stores_commit();
            }
          }
        }
      }
      ++n;
      return true;
    });
    if (lane == 0) stores_done();
  }
  __syncthreads();
  cluster_sync();
  if (warp == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

// dW = the sum of the splits' fp32 parts, (splits, 2, f, d), four values a thread
__global__ void __launch_bounds__(256) dw_reduce(const float4* __restrict__ part, int splits, int64_t n4,
                                                 uint2* __restrict__ dwg, uint2* __restrict__ dwu) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= 2 * n4) return;
  float4 v = part[i];
  for (int s = 1; s < splits; ++s) {
    const float4 q = part[2 * n4 * s + i];
    v.x += q.x, v.y += q.y, v.z += q.z, v.w += q.w;
  }
  uint2* o = i < n4 ? dwg : dwu;
  if (o) o[i < n4 ? i : i - n4] = make_uint2(pack2(v.x, v.y), pack2(v.z, v.w));
}

// ---- few rows ---------------------------------------------------------------------------------
// One CTA computes 16 columns of h for all rows; its 8 warps share the contraction.  The weights'
// 16 x 16 fragments come straight from memory: a lane reads 16 bytes (8 steps) of its two rows, and
// takes them as the fragments of two products; the steps' order inside a group of 32 does not
// matter as long as x, read the same way, agrees.  NG groups of 8 rows of x.
//
// Two CTAs to an SM hide each other's loads (768 -> 2048, one row 3.6 -> 2.6 us; 1024 -> 2736, 4.6 us:
// 11.2 MB of weights, 1.7 us at the copy rate).  With more than 32 rows the accumulators take 64
// registers: where the grid leaves no SM a second CTA, one with twice the loads in flight is faster
// (64 rows, 768 -> 2048: 6.0 against 7.4 us), otherwise two with fewer (1024 -> 2736: 11.3 against 13.0).
constexpr int FT = 256;
constexpr int RED_ROW = 20;  // floats of a row of 16 sums: a fragment's 32 lanes on 32 banks

__device__ __forceinline__ void mma16816(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

template <int NG, int ACT, int MINB>
__global__ void __launch_bounds__(FT, MINB) ffn_few(const __nv_bfloat16* __restrict__ x, int64_t ldx,
                                              const __nv_bfloat16* __restrict__ wg, int64_t ldg,
                                              const __nv_bfloat16* __restrict__ wu, int64_t ldu,
                                              __nv_bfloat16* __restrict__ h, int rows, int d, int f) {
  extern __shared__ float red[];  // (8 warps, gate | up, 8 NG rows, RED_ROW)
  constexpr int PART = 8 * NG * RED_ROW;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gr = lane >> 2, tq = lane & 3;
  const int f0 = blockIdx.x * 16;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  const bool r0 = f0 + gr < f, r1 = f0 + gr + 8 < f;
  const __nv_bfloat16 *g0 = wg + (int64_t)(f0 + gr) * ldg, *g1 = g0 + 8 * ldg;
  const __nv_bfloat16 *u0 = wu + (int64_t)(f0 + gr) * ldu, *u1 = u0 + 8 * ldu;
  float cg[NG][4], cu[NG][4];
#pragma unroll
  for (int i = 0; i < NG; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) cg[i][k] = cu[i][k] = 0.f;
  const auto ld = [&](const __nv_bfloat16* p, bool ok) {
    return ok ? __ldg(reinterpret_cast<const uint4*>(p)) : zero;
  };
  constexpr int UN = NG == 8 && MINB == 2 ? 2 : 4;  // groups of 32 steps whose weights are in flight at once
  for (int kb = 32 * warp; kb < d; kb += 32 * 8 * UN) {
    uint4 a[UN][4];
#pragma unroll
    for (int i = 0; i < UN; ++i) {
      const int k = kb + 256 * i + 8 * tq;
      const bool in = k < d;
      a[i][0] = ld(g0 + k, in && r0), a[i][1] = ld(g1 + k, in && r1);
      a[i][2] = ld(u0 + k, in && r0), a[i][3] = ld(u1 + k, in && r1);
    }
#pragma unroll
    for (int i = 0; i < UN; ++i) {
      const int k = kb + 256 * i + 8 * tq;
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        const int r = 8 * j + gr;
        const uint4 b = ld(x + (int64_t)r * ldx + k, k < d && r < rows);
        mma16816(cg[j], a[i][0].x, a[i][1].x, a[i][0].y, a[i][1].y, b.x, b.y);
        mma16816(cu[j], a[i][2].x, a[i][3].x, a[i][2].y, a[i][3].y, b.x, b.y);
        mma16816(cg[j], a[i][0].z, a[i][1].z, a[i][0].w, a[i][1].w, b.z, b.w);
        mma16816(cu[j], a[i][2].z, a[i][3].z, a[i][2].w, a[i][3].w, b.z, b.w);
      }
    }
  }
  // fragment (row gr or gr + 8 of the weights, rows 2 tq and 2 tq + 1 of x) -> red[warp][gate|up][row][column]
  float* mine = red + warp * 2 * PART;
#pragma unroll
  for (int j = 0; j < NG; ++j)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int at = (8 * j + 2 * tq + (k & 1)) * RED_ROW + gr + 8 * (k >> 1);
      mine[at] = cg[j][k];
      mine[PART + at] = cu[j][k];
    }
  __syncthreads();
  for (int i = threadIdx.x; i < 8 * NG * 16; i += FT) {
    const int r = i >> 4, c = i & 15;
    if (r >= rows || f0 + c >= f) continue;
    float sg = 0.f, su = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      sg += red[w * 2 * PART + r * RED_ROW + c];
      su += red[w * 2 * PART + PART + r * RED_ROW + c];
    }
    h[(int64_t)r * f + f0 + c] = __float2bfloat16_rn(act_of<ACT>(sg) * su);
  }
}

// ---- host -------------------------------------------------------------------------------------
constexpr int FEW_ROWS = 64;

int fail(int code, const char* msg) {
  set_last_error(msg);
  return code;
}
int cuda_fail(cudaError_t e, const char* where) {
  set_last_error(std::string(where) + ": " + cudaGetErrorString(e));
  return SCA2_ERR_CUDA;
}

// map of a (rows, cols) matrix with row stride ld values; swizzled boxes: 64 columns x `box` rows of
// an operand, 32 x 32 of what the epilogue stages (box = 0)
bool map2(CUtensorMap* m, const void* p, int64_t rows, int64_t cols, int64_t ld, int box) {
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld * 2};
  const cuuint32_t bx[2] = {box ? 64u : 32u, box ? (cuuint32_t)box : 32u}, es[2] = {1, 1};
  return tensor_map_encoder()(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(p), dims, strides, bx, es,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, box ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// map of the fp32 parts (splits * 2, f, d)
bool map3(CUtensorMap* m, const void* p, int64_t slices, int64_t f, int64_t d) {
  const cuuint64_t dims[3] = {(cuuint64_t)d, (cuuint64_t)f, (cuuint64_t)slices};
  const cuuint64_t strides[2] = {(cuuint64_t)d * 4, (cuuint64_t)(f * d * 4)};
  const cuuint32_t bx[3] = {16, 32, 1}, es[3] = {1, 1, 1};
  return tensor_map_encoder()(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, const_cast<void*>(p), dims, strides, bx, es,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

constexpr int PAIRS = 74;  // 148 SMs

// The kernels' shared memory.  Before any tensor map is encoded: as a call of the runtime it also
// makes the device's context current in this thread (autograd's threads come without one, and the
// driver then refuses to encode).
template <int KIND, int ACT>
cudaError_t allow() {
  return cudaFuncSetAttribute(ffn_gemm<KIND, ACT>, cudaFuncAttributeMaxDynamicSharedMemorySize, Layout<KIND>::TOTAL);
}
template <int KIND>
cudaError_t allow_act(int act) {
  return act == SCA2_ACT_SILU ? allow<KIND, SILU>() : allow<KIND, GELU>();
}
int pairs_of(const Geo& g) { return std::min(PAIRS, g.units + g.x_units); }
template <int KIND, int ACT>
cudaError_t launch(const Maps& maps, const Geo& g, cudaStream_t st) {
  const int pairs = pairs_of(g);
  Geo k = g;
  k.kb_split = g.kb / g.splits, k.kb_more = g.kb % g.splits;
  int u = pairs;
  k.sn = u % g.tiles_n, u /= g.tiles_n;
  k.sm = u % g.tiles_m, u /= g.tiles_m;
  k.ss = u % g.slices, k.sp = u / g.slices;
  ffn_gemm<KIND, ACT><<<2 * pairs, NT, Layout<KIND>::TOTAL, st>>>(maps, k);
  return cudaGetLastError();
}
template <int KIND>
cudaError_t launch_act(int act, const Maps& maps, const Geo& g, cudaStream_t st) {
  return act == SCA2_ACT_SILU ? launch<KIND, SILU>(maps, g, st) : launch<KIND, GELU>(maps, g, st);
}

template <int NG, int MINB = 2>
cudaError_t launch_few(const sca2_ffn_args& a, void* h, cudaStream_t st) {
  const auto bf = [](const void* p) { return static_cast<const __nv_bfloat16*>(p); };
  const int smem = 8 * 2 * 8 * NG * RED_ROW * 4, grid = (a.f + 15) / 16;
  const auto k = a.act == SCA2_ACT_SILU ? ffn_few<NG, SILU, MINB> : ffn_few<NG, GELU, MINB>;
  if (smem > 48 * 1024)
    if (cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)) return e;
  k<<<grid, FT, smem, st>>>(bf(a.x), a.ldx, bf(a.w_gate), a.ldg, bf(a.w_up), a.ldu, static_cast<__nv_bfloat16*>(h),
                            (int)a.rows, a.d, a.f);
  return cudaGetLastError();
}

int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

Geo geo_proj(const sca2_ffn_args& a) {
  Geo g{};
  g.rows = (int)a.rows, g.d = a.d, g.f = a.f;
  g.tiles_n = ceil_div(a.f, 128), g.tiles_m = ceil_div(a.rows, 256), g.slices = g.splits = 1;
  g.units = g.tiles_n * g.tiles_m, g.kb = ceil_div(a.d, BK);
  return g;
}
// The pairs' share of the DX tiles beside their DW tiles (pair p has DW units p, p + pairs, ...): x_a
// for those with one DW unit more than the others, x_b for the others.  Returns the longest pair's
// contraction blocks, a tile's start and end counted as `LAP` blocks.
constexpr int LAP = 4;
double share(Geo& g) {
  const int pairs = pairs_of(g);
  const double cw = (double)g.kb / g.splits + LAP, cx = 2.0 * g.kb_half + LAP;
  const int q = g.units / pairs;
  g.x_pairs = g.units % pairs;
  const int rest = pairs - g.x_pairs;
  const double even = (g.units * cw + g.x_units * cx) / pairs;
  double best = 1e30;
  for (int i = 0; i < 2; ++i) {
    const int xa = std::max(0, (int)((even - (q + 1) * cw) / cx) + i);
    const int64_t left = std::max<int64_t>(0, g.x_units - (int64_t)xa * g.x_pairs);
    const int xb = (int)((left + rest - 1) / rest);
    const double longest = std::max(g.x_pairs ? (q + 1) * cw + xa * cx : 0.0, q * cw + xb * cx);
    if (longest < best) best = longest, g.x_a = xa, g.x_b = xb;
  }
  return best;
}
// DW and DX.  Splits of the rows: the fewest whose longest pair is shortest, each split keeping at
// least 16 contraction blocks; from two on, the parts cost a launch and a pass over them.
Geo geo_grads(const sca2_ffn_args& a, bool need_x, bool need_w) {
  Geo g = geo_proj(a);
  g.tiles_n = ceil_div(a.d, 256), g.tiles_m = ceil_div(a.f, 256), g.slices = 2;
  g.kb = ceil_div(a.rows, BK), g.kb_half = ceil_div(a.f, BK);
  g.x_units = need_x ? g.tiles_n * ceil_div(a.rows, 256) : 0;
  const int tiles = need_w ? g.tiles_n * g.tiles_m * 2 : 0;
  Geo best = g;
  double least = 1e30;
  for (int s = 1; s <= (need_w ? 32 : 1) && (s == 1 || g.kb / s >= 16); ++s) {
    g.splits = s, g.units = tiles * s;
    const double cost = share(g) + (s > 1 ? 12 + 2 * s : 0);
    if (cost < least * 0.97) least = cost, best = g;
  }
  return best;
}

int check(const sca2_ffn_args* a) {
  if (!a) return fail(SCA2_ERR_ARG, "gated_ffn: null argument struct");
  if (a->rows < 0 || a->d < 1 || a->f < 1) return fail(SCA2_ERR_ARG, "gated_ffn: bad sizes");
  if (a->d % 8 || a->f % 8) return fail(SCA2_ERR_UNSUPPORTED, "gated_ffn: d and f must be multiples of 8");
  if (a->rows > (1LL << 30) || a->d > (1 << 20) || a->f > (1 << 20))
    return fail(SCA2_ERR_UNSUPPORTED, "gated_ffn: at most 2^30 rows and widths of 2^20");
  if (a->act != SCA2_ACT_SILU && a->act != SCA2_ACT_GELU)
    return fail(SCA2_ERR_ARG, "gated_ffn: act must be SCA2_ACT_SILU or SCA2_ACT_GELU");
  if ((int64_t)ceil_div(a->rows, 256) * ceil_div(a->f, 128) > (1 << 30) ||
      (int64_t)ceil_div(a->rows, 256) * ceil_div(a->d, 256) > (1 << 30))
    return fail(SCA2_ERR_UNSUPPORTED, "gated_ffn: too many tiles");
  if (!a->w_gate || !a->w_up || (a->rows > 0 && !a->x)) return fail(SCA2_ERR_ARG, "gated_ffn: null input");
  if (((uintptr_t)a->x | (uintptr_t)a->w_gate | (uintptr_t)a->w_up) & 15u)
    return fail(SCA2_ERR_ARG, "gated_ffn: inputs must be 16-byte aligned");
  for (int64_t ld : {a->ldx, a->ldg, a->ldu})
    if (ld < a->d || ld % 8 || ld > (1LL << 31)) return fail(SCA2_ERR_ARG, "gated_ffn: row strides must be multiples of 8, at least d");
  return SCA2_OK;
}

int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }

}  // namespace ffn

cudaError_t ffn_read_faults(unsigned int* out) {
  unsigned int zero = 0;
  cudaError_t e = cudaMemcpyFromSymbol(out, ffn::g_fault_ffn, sizeof(unsigned int));
  if (e != cudaSuccess) return e;
  return cudaMemcpyToSymbol(ffn::g_fault_ffn, &zero, sizeof(unsigned int));
}

}  // namespace sca2

using namespace sca2::ffn;

extern "C" {

int sca2_gated_ffn_fwd(const sca2_ffn_args* a, void* h, void* stream) {
  if (int rc = check(a)) return rc;
  if (a->rows == 0) return SCA2_OK;
  if (!h || ((uintptr_t)h & 15u)) return fail(SCA2_ERR_ARG, "gated_ffn: h must be non-null and 16-byte aligned");
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (a->rows <= FEW_ROWS) {
    e = a->rows <= 8 ? launch_few<1>(*a, h, st) : a->rows <= 16 ? launch_few<2>(*a, h, st)
        : a->rows <= 32 ? launch_few<4>(*a, h, st)
        : a->f <= 16 * 148 ? launch_few<8, 1>(*a, h, st) : launch_few<8, 2>(*a, h, st);
  } else {
    if ((e = allow_act<FWD>(a->act)) != cudaSuccess) return cuda_fail(e, "sca2_gated_ffn_fwd");
    if (!sca2::tensor_map_encoder()) return fail(SCA2_ERR_CUDA, "gated_ffn: no tensor-map encoder in the driver");
    Maps m;
    memset(&m, 0, sizeof(m));
    if (!map2(&m.a0, a->x, a->rows, a->d, a->ldx, 128) || !map2(&m.b0, a->w_gate, a->f, a->d, a->ldg, 128) ||
        !map2(&m.b1, a->w_up, a->f, a->d, a->ldu, 128) || !map2(&m.o0, h, a->rows, a->f, a->f, 0))
      return fail(SCA2_ERR_CUDA, "gated_ffn: tensor map refused");
    e = launch_act<FWD>(a->act, m, geo_proj(*a), st);
  }
  return e == cudaSuccess ? SCA2_OK : cuda_fail(e, "sca2_gated_ffn_fwd");
}

int64_t sca2_gated_ffn_work_bytes(int64_t rows, int32_t d, int32_t f) {
  if (rows < 1 || d < 1 || f < 1 || rows > (1LL << 30)) return 0;
  sca2_ffn_args a{};
  a.rows = rows, a.d = d, a.f = f;
  const int s = std::max(geo_grads(a, true, true).splits, geo_grads(a, false, true).splits);
  return 2 * up256(rows * f * 2) + (s > 1 ? (int64_t)s * 2 * f * d * 4 : 0);
}

int sca2_gated_ffn_bwd(const sca2_ffn_args* a, const void* dh, void* dx, void* dw_gate, void* dw_up, void* work,
                       int64_t work_bytes, void* stream) {
  if (int rc = check(a)) return rc;
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e = cudaSuccess;
  if ((dw_gate == nullptr) != (dw_up == nullptr)) return fail(SCA2_ERR_ARG, "gated_ffn: dw_gate and dw_up go together");
  if (((uintptr_t)dx | (uintptr_t)dw_gate | (uintptr_t)dw_up | (uintptr_t)dh) & 15u)
    return fail(SCA2_ERR_ARG, "gated_ffn: dh and the gradients must be 16-byte aligned");
  if (a->rows == 0) {
    for (void* p : {dw_gate, dw_up})
      if (p && e == cudaSuccess) e = cudaMemsetAsync(p, 0, (size_t)a->f * a->d * 2, st);
    return e == cudaSuccess ? SCA2_OK : cuda_fail(e, "sca2_gated_ffn_bwd");
  }
  if (!dh) return fail(SCA2_ERR_ARG, "gated_ffn: dh must be non-null");
  if (!work || ((uintptr_t)work & 255u) || work_bytes < sca2_gated_ffn_work_bytes(a->rows, a->d, a->f))
    return fail(SCA2_ERR_ARG, "gated_ffn: workspace null, not 256-byte aligned or too small");
  if (!dx && !dw_gate) return SCA2_OK;
  e = allow_act<BACK>(a->act);
  if (e == cudaSuccess) e = allow<GRADS, SILU>();
  if (e != cudaSuccess) return cuda_fail(e, "sca2_gated_ffn_bwd");
  if (!sca2::tensor_map_encoder()) return fail(SCA2_ERR_CUDA, "gated_ffn: no tensor-map encoder in the driver");
  uint8_t* w = static_cast<uint8_t*>(work);
  void *dg = w, *du = w + up256(a->rows * a->f * 2), *part = w + 2 * up256(a->rows * a->f * 2);
  const int64_t n = a->rows;
  const Geo g = geo_grads(*a, dx != nullptr, dw_gate != nullptr);
  Maps m, x;
  memset(&m, 0, sizeof(m));
  bool ok = map2(&m.a0, a->x, n, a->d, a->ldx, 128) && map2(&m.b0, a->w_gate, a->f, a->d, a->ldg, 128) &&
            map2(&m.b1, a->w_up, a->f, a->d, a->ldu, 128) && map2(&m.o0, dg, n, a->f, a->f, 0) &&
            map2(&m.o1, du, n, a->f, a->f, 0) && map2(&m.dh, dh, n, a->f, a->f, 0);
  memset(&x, 0, sizeof(x));
  if (dx)
    ok = ok && map2(&x.xa0, dg, n, a->f, a->f, 128) && map2(&x.xa1, du, n, a->f, a->f, 128) &&
         map2(&x.xb0, a->w_gate, a->f, a->d, a->ldg, 64) && map2(&x.xb1, a->w_up, a->f, a->d, a->ldu, 64) &&
         map2(&x.xo, dx, n, a->d, a->d, 0);
  if (dw_gate) {
    ok = ok && map2(&x.a0, dg, n, a->f, a->f, 64) && map2(&x.a1, du, n, a->f, a->f, 64) &&
         map2(&x.b0, a->x, n, a->d, a->ldx, 64);
    if (g.splits > 1) ok = ok && map3(&x.o0, part, 2 * g.splits, a->f, a->d);
    else ok = ok && map2(&x.o0, dw_gate, a->f, a->d, a->d, 0) && map2(&x.o1, dw_up, a->f, a->d, a->d, 0);
  }
  if (!ok) return fail(SCA2_ERR_CUDA, "gated_ffn: tensor map refused");
  e = launch_act<BACK>(a->act, m, geo_proj(*a), st);
  if (e == cudaSuccess) e = launch<GRADS, SILU>(x, g, st);
  if (e == cudaSuccess && dw_gate && g.splits > 1) {
    const int64_t n4 = (int64_t)a->f * a->d / 4;
    dw_reduce<<<(unsigned)((2 * n4 + 255) / 256), 256, 0, st>>>(static_cast<const float4*>(part), g.splits, n4,
                                                                static_cast<uint2*>(dw_gate), static_cast<uint2*>(dw_up));
    e = cudaGetLastError();
  }
  return e == cudaSuccess ? SCA2_OK : cuda_fail(e, "sca2_gated_ffn_bwd");
}

}  // extern "C"
