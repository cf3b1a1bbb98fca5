// MXFP4 linear layers: C = epi(A . W^T + bias), A and W in the 4-bit rows and
// scale tiles of jb_mxfp4.cu.
//
//   acc[m, n] = sum over blocks b of 32 columns of
//               2^(Ea[m, b] + Ew[n, b]) * sum over k in b of a[m, k] w[n, k]
//
// on tcgen05.mma kind::mxf4 with block scales (one UE8M0 byte per 32
// elements, scale_vec::2X): the tensor core multiplies the scales in, exact
// products accumulated in f32 in TMEM, four times the bf16 rate.
//
// Persistent CTAs, one per SM, output tiles of 128 x 64 or 128 x 128, or of
// 256 x 192 by pairs of CTAs; K in stages of 256 elements (one 128-byte
// swizzled row of codes):
//   warp 0     TMA producer: codes of A and W, and their scale tiles as rows of
//              128 bytes, by tiled copies (what lies past the end arrives as 0)
//   warp 1     TMEM allocator and MMA issuer: per stage the scale tiles go from
//              shared memory to TMEM (tcgen05.cp 32x128b.warpx4: 128 rows x 4
//              blocks into 4 columns), then four K = 64 products.  Each stage
//              has its own TMEM columns for the scales, so a copy never meets a
//              product that still reads them: the stage's shared memory, and
//              with it its TMEM columns, comes back only after the commit of
//              its products.  In the odd CTA of a pair it passes on that its
//              epilogue has read an accumulator.
//   warps 2..  epilogue, one warp per 32 rows x 64 columns of the tile: the
//              accumulators go to registers at once (tcgen05.ld) and are
//              released before any arithmetic; bias, activation and residual
//              (a TMA-loaded box, issued before the wait for the
//              accumulators) in f32, one rounding, one TMA store of the box.
// The accumulator is double-buffered (2 x BN columns).
//
// What bounds it.  A K = 64 product reads 32 bytes of each of its rows from
// shared memory, at 128 bytes a clock: 128 x 192 by one SM would take 80
// clocks of reading (and more than that to fill) beside 96 of arithmetic, and
// did not get past 217 us at 8192^3.  A pair (cta_group::2) gives each SM half
// of W: 186 us, 5.9 PFLOP/s, 90% of four times the measured bf16 rate.
// BN = 192 is the widest tile whose two accumulators leave TMEM columns for
// the scales (384 + 5 stages x 24).  Its odd tiles start 64 rows into a scale
// tile of W: the scale address of the product starts two columns (2 x 32
// rows) later.
//
// Measured (bf16 in and out unless said, without the quantisation of A; captured
// calls at 1965 MHz):
//   20479 x 4096 x 1024                49.1 us  3.5 PFLOP/s  f32 out 73.2
//     GELU                             55.8 us  3.1 PFLOP/s  f32 out 76.3; quick GELU 61.1
//   20479 x 1024 x 4096                39.8 us  4.3 PFLOP/s
//     residual                         43.8 us  3.9 PFLOP/s  f32 56.5
//   777 x 1024 x 4096                   7.0 us               one tile's latency
//   1777 x 1536 x 384, GELU, f16        6.6 us               launch, one tile's latency
//   12 x 2304 x 768                     3.5 us               launch, one tile's latency
//   12 x 1024 x 4096                    6.3 us               16 CTAs, each 64 rows of W alone
// K = 1024: no pipe is full (GELU: tensor 42%, its memory 49%, XU 43%, issue
// 54%); each epilogue warp's chain of TMEM read, activation, box, store and
// wait for the box is the likely bound.  K = 4096, N = 1024: 64% of tensor cycles; N in
// tiles of 192 is 6 for 5.33, and 480 tiles are 6.5 waves in 7, together 21% of
// them.
#include <cudaTypedefs.h>

#include <algorithm>
#include <atomic>
#include <cstring>
#include <mutex>

#include "jb_common.cuh"
#include "jb_internal.h"

namespace jb {
namespace {

constexpr int kBM = 128;
constexpr int kStageK = 256;       // elements of K per stage: 128 bytes of codes
constexpr int kUnitCols = 64;      // columns of an epilogue warp
constexpr int kUnitBytes = 4096;   // its box: 32 rows of 128 bytes (64 16-bit or 32 f32 columns)
constexpr int kSfTile = 512;       // scale bytes of 128 rows x 128 columns

// CG = 2: a cluster of two CTAs (two SMs of one TPC) shares a tile of 256 x BN
// by tcgen05.mma.cta_group::2.  Each CTA holds 128 rows of A and of the
// accumulator and half of W's rows; both hold the scales of all BN columns.
template <int BN, int CG>
struct MxCfg {
  static constexpr int B_ROWS = BN / CG;
  static constexpr int A_BYTES = kBM * 128;
  static constexpr int B_BYTES = B_ROWS * 128;
  // 128-row scale tiles that BN rows of W may touch (tiles start at multiples of BN)
  static constexpr int SFB_TILES = BN > 128 ? 2 : 1;
  static constexpr int SF_BYTES = 2 * kSfTile * (1 + SFB_TILES);
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES + SF_BYTES;
  static constexpr int STAGES = CG == 2 ? 5 : BN == 128 ? 5 : 6;
  static constexpr int SF_COLS = 8 * (1 + SFB_TILES);  // TMEM columns of a stage's scales
  static constexpr int TMEM_COLS = 512;  // all of it (one CTA per SM): the base is column 0
  static_assert(2 * BN + STAGES * SF_COLS <= TMEM_COLS, "TMEM columns");
  static constexpr int EPI_WARPS = 4 * (BN / kUnitCols);
  static constexpr int THREADS = 64 + 32 * EPI_WARPS;
  static constexpr int BARS = 2 * STAGES + 4 + 1 + EPI_WARPS + 2;
  static constexpr int SMEM = 1024 + STAGES * STAGE_BYTES + EPI_WARPS * (kUnitBytes + kUnitCols * 4) + 8 * BARS + 16;
  static_assert(SMEM <= 232448, "shared memory");
};

struct MxParams {
  const float* bias;
  int M, N, K;
  int* err;
};

// Type of the output and the residual.
enum Out { kBf16, kF16, kF32 };

// D[tmem] (+)= A . B^T over K = 64 e2m1 elements, each block of 32 scaled by
// the UE8M0 bytes at sfa / sfb.
template <int CG>
__device__ __forceinline__ void mma_mxf4(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                         uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
  if constexpr (CG == 1)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(
            d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(
            d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
}
// 32 rows of 16 contiguous bytes -> 4 TMEM columns of lanes 0-31, repeated in
// the other three lane quarters (CG = 2: in both CTAs, each from its own
// shared memory).
template <int CG>
__device__ __forceinline__ void tmem_cp_scales(uint32_t taddr, uint64_t desc) {
  if constexpr (CG == 1)
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
  else
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
// Arrive on `bar` (CG = 2: on both CTAs' barriers at that offset) once every
// tcgen05 operation issued so far by this thread has completed.
template <int CG>
__device__ __forceinline__ void commit(uint32_t bar) {
  if constexpr (CG == 1)
    mma_commit(bar);
  else
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
        "h"(static_cast<uint16_t>(3))
        : "memory");
}
// A box into this CTA's shared memory; its bytes count on `bar` (CG = 2: the
// even CTA's barrier, a shared::cluster address).
template <int CG>
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  if constexpr (CG == 1)
    tma_load_2d(dst, map, x, y, bar);
  else
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
// The address of CTA 0's copy of a shared-memory variable of the cluster.
__device__ __forceinline__ uint32_t of_cta0(uint32_t addr) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
  return r;
}
// What this thread has seen happens before what follows the wait below in
// either CTA.
__device__ __forceinline__ void arrive_cluster(uint32_t addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
__device__ __forceinline__ bool warp_wait_cluster(uint32_t bar, uint32_t parity, volatile int* abort) {
  if (!warp_mbar_wait(bar, parity, abort)) return false;
  uint32_t done;  // the phase is complete: once more, with the cluster's scope
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return __all_sync(0xffffffffu, done != 0);
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Descriptor of a scale tile: 8-row groups of 16-byte rows, 128 bytes apart,
// no swizzle.
__device__ __forceinline__ uint64_t scale_desc(uint32_t smem_addr) {
  return static_cast<uint64_t>((smem_addr & 0x3FFFF) >> 4) | (static_cast<uint64_t>(128 >> 4) << 16) |
         (static_cast<uint64_t>(128 >> 4) << 32) | (static_cast<uint64_t>(1) << 46);
}
// kind::mxf4, dense, K-major: A and B e2m1 (1), UE8M0 scales (bit 23), N >> 3
// at 17, M >> 7 at 27; sf = the byte of the scale column that the product's
// first block uses (0 or 2), for A at 29 and B at 4.
constexpr uint32_t mx_idesc(int M, int N, uint32_t sf) {
  return (sf << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(N >> 3) << 17) | (1u << 23) |
         (static_cast<uint32_t>(M >> 7) << 27) | (sf << 29);
}

// 16-byte slot `q` of row `row` of a 128-byte-swizzled box.
__device__ __forceinline__ uint32_t box_slot(uint32_t buf, int row, int q) {
  return buf + row * 128 + ((q ^ (row & 7)) << 4);
}
template <Out OUT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (OUT == kF16) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&b);
}
template <Out OUT>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (OUT == kF16) return __half22float2(*reinterpret_cast<const __half2*>(&w));
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(a)
               : "memory");
  return v;
}
__device__ __forceinline__ void sts128(uint32_t a, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
               : "memory");
}

// GELU(x) = max(x, 0) - a h(a), a = min(|x|, 8), h(a) = erfc(a / sqrt 2) / 2.
// log2 h is smooth and nearly quadratic: a polynomial of degree 6, fitted here
// to log2(erfc(a / sqrt 2) / 2) on [0, 6] for the least error of a h(a), gives
// h as one 2^x, 13 instructions per pair with the two exponentials.  |error of
// GELU| <= 2e-7 and the result's own rounding in f32: at most 3e-7 on |x| <= 8.
// Relative to the result it is within 2^-10 down to x = -6 and passes 2^-9 at
// -6.16 (2.5% at -7, where GELU is -9e-12); below the clamp it stays at
// -5.7e-15.  At a = 6 the polynomial is -29.9, and falls from there.  NaN stays NaN.
__device__ __forceinline__ float max0_nan(float x) {
  float y;
  asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float2 gelu_pair(float2 x) {
  const float2 a = make_float2(fmaxf(-fabsf(x.x), -8.f), fmaxf(-fabsf(x.y), -8.f));  // -a
  float2 q = __ffma2_rn(a, f2(3.231512164e-05f), f2(7.549100555e-04f));
  q = __ffma2_rn(a, q, f2(8.007442579e-03f));
  q = __ffma2_rn(a, q, f2(5.325423181e-02f));
  q = __ffma2_rn(a, q, f2(-4.589267671e-01f));
  q = __ffma2_rn(a, q, f2(1.151135921f));
  q = __ffma2_rn(a, q, f2(-1.000002146f));
  return __ffma2_rn(a, make_float2(ex2_approx(q.x), ex2_approx(q.y)), make_float2(max0_nan(x.x), max0_nan(x.y)));
}

// 32 accumulators -> f32 outputs before the residual.
template <int EPI>
__device__ __forceinline__ void finish32(const uint32_t (&r)[32], uint32_t bias, float (&v)[32]) {
#pragma unroll
  for (int j = 0; j < 32; j += 4) {
    const uint4 b = lds128(bias + 4 * j);
    float2 lo = __fadd2_rn(make_float2(__uint_as_float(r[j]), __uint_as_float(r[j + 1])),
                           make_float2(__uint_as_float(b.x), __uint_as_float(b.y)));
    float2 hi = __fadd2_rn(make_float2(__uint_as_float(r[j + 2]), __uint_as_float(r[j + 3])),
                           make_float2(__uint_as_float(b.z), __uint_as_float(b.w)));
    if constexpr (EPI == JB_EPI_GELU) {
      lo = gelu_pair(lo);
      hi = gelu_pair(hi);
    } else if constexpr (EPI == JB_EPI_QUICK_GELU) {
      lo = make_float2(quick_gelu_tc(lo.x), quick_gelu_tc(lo.y));
      hi = make_float2(quick_gelu_tc(hi.x), quick_gelu_tc(hi.y));
    }
    v[j] = lo.x; v[j + 1] = lo.y; v[j + 2] = hi.x; v[j + 3] = hi.y;
  }
}

template <int BN, int EPI, Out OUT, int CG>
__global__ void __launch_bounds__(MxCfg<BN, CG>::THREADS, 1)
    gemm_mxfp4_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                      const __grid_constant__ CUtensorMap tmSA, const __grid_constant__ CUtensorMap tmSB,
                      const __grid_constant__ CUtensorMap tmC, const __grid_constant__ CUtensorMap tmR,
                      const MxParams p) {
  using Cfg = MxCfg<BN, CG>;
  constexpr bool kRes = EPI == JB_EPI_RESIDUAL;
  constexpr bool F32 = OUT == kF32;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* gbase = smem_raw + (base - raw);
  // [stages][A | B] | [epilogue boxes] | [stages][scales A | scales B] |
  // [epilogue biases] | barriers | tmem slot | abort flag
  const uint32_t boxes = base + Cfg::STAGES * (Cfg::A_BYTES + Cfg::B_BYTES);
  const uint32_t scales = boxes + Cfg::EPI_WARPS * kUnitBytes;
  const uint32_t biases = scales + Cfg::STAGES * Cfg::SF_BYTES;
  const uint32_t bars = biases + Cfg::EPI_WARPS * kUnitCols * 4;
  // CG = 2: full of the even CTA counts for the pair, and peer says there that
  // the odd CTA's epilogue has read its half of an accumulator
  auto full_bar = [&](int s) { return bars + 8u * s; };
  auto empty_bar = [&](int s) { return bars + 8u * (Cfg::STAGES + s); };
  auto tfull_bar = [&](int i) { return bars + 8u * (2 * Cfg::STAGES + i); };
  auto tempty_bar = [&](int i) { return bars + 8u * (2 * Cfg::STAGES + 2 + i); };
  const uint32_t spare = bars + 8u * (2 * Cfg::STAGES + 4);
  auto res_bar = [&](int w) { return bars + 8u * (2 * Cfg::STAGES + 5 + w); };
  auto peer_bar = [&](int i) { return bars + 8u * (2 * Cfg::STAGES + 5 + Cfg::EPI_WARPS + i); };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(gbase + (bars - base) + 8 * Cfg::BARS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);  // uniform to the compiler too
  const int lane = threadIdx.x & 31;
  int rank = 0;  // this CTA's half of the tile
  if constexpr (CG == 2) asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  const int first = blockIdx.x / CG, step = gridDim.x / CG;
  const int n_tiles = (p.N + BN - 1) / BN;
  const int total = (p.M + CG * kBM - 1) / (CG * kBM) * n_tiles;
  const int kb_count = (p.K + kStageK - 1) / kStageK;
  const int k_tiles = (p.K + 127) / 128;  // scale tiles along K

  if (threadIdx.x == 0) {
    for (int s = 0; s < Cfg::STAGES; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(tfull_bar(i), 1);
      mbar_init(tempty_bar(i), Cfg::EPI_WARPS);
      mbar_init(peer_bar(i), 1);
    }
    mbar_init(spare, 1);
    for (int w = 0; w < Cfg::EPI_WARPS; ++w) mbar_init(res_bar(w), 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    if constexpr (CG == 1) {
      tmem_alloc(smem_u32(tmem_slot), Cfg::TMEM_COLS);
    } else {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                   "r"(Cfg::TMEM_COLS)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
  }
  if (warp == 0 && lane == 0) {
    prefetch_tensormap(&tmA);
    prefetch_tensormap(&tmB);
    prefetch_tensormap(&tmSA);
    prefetch_tensormap(&tmSB);
    prefetch_tensormap(&tmC);
    if (kRes) prefetch_tensormap(&tmR);
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();
  tc_fence_after();
  constexpr uint32_t tmem_base = 0;

  // The producer and the issuer walk their loops as whole warps, without
  // exits (a wait that gives up turns the later ones off), and elect one lane
  // around each stage's group of instructions: every operand is then in a
  // uniform register.  With one lane in `if (lane == 0)` a product of any width
  // takes about 250 clocks to issue; a 192-column product of K = 64 runs in 96.
  if (warp == 0) {  // ── producer
    int st = 0, filled = 0;
    uint32_t ph = 0;
    bool ok = true;
    for (int t = first; t < total; t += step) {
      const int mt = t / n_tiles * CG + rank, nb = t % n_tiles;  // rows in 128s, columns in BNs
      const int wt = nb * BN / 128;
#pragma unroll 1
      for (int kb = 0; kb < kb_count; ++kb) {
        if (ok) ok = warp_mbar_wait(empty_bar(st), ph ^ 1u, abort_flag);
        const uint32_t sa = base + st * (Cfg::A_BYTES + Cfg::B_BYTES);
        const uint32_t sf = scales + st * Cfg::SF_BYTES;
        const uint32_t full = CG == 2 ? of_cta0(full_bar(st)) : full_bar(st);
        if (elect_one() && ok) {
          if (CG == 1 || rank == 0) mbar_arrive_expect_tx(full_bar(st), CG * Cfg::STAGE_BYTES);
          load_box<CG>(sa, &tmA, kb * 128, mt * kBM, full);
          load_box<CG>(sa + Cfg::A_BYTES, &tmB, kb * 128, nb * BN + rank * Cfg::B_ROWS, full);
          // two K tiles of scales; past the last one: the next row's, which no product reads
          load_box<CG>(sf, &tmSA, 0, (mt * k_tiles + 2 * kb) * 4, full);
#pragma unroll
          for (int i = 0; i < Cfg::SFB_TILES; ++i)
            load_box<CG>(sf + 2 * kSfTile * (1 + i), &tmSB, 0, ((wt + i) * k_tiles + 2 * kb) * 4, full);
        }
        __syncwarp();
        filled += ok ? 1 : 0;
        if (++st == Cfg::STAGES) {
          st = 0;
          ph ^= 1u;
        }
      }
    }
    if (*abort_flag && rank == 0) {  // the pair's copies in flight land before a CTA leaves (bounded)
      volatile int no_abort = 0;
      for (int b = max(0, filled - Cfg::STAGES); b < filled; ++b)
        mbar_wait(full_bar(b % Cfg::STAGES), (b / Cfg::STAGES) & 1, &no_abort);
    }
  } else if (warp == 1) {  // ── MMA issuer (of the even CTA), or its odd CTA's relay
    constexpr uint32_t kStageDesc = (Cfg::A_BYTES + Cfg::B_BYTES) >> 4;  // descriptors count 16 bytes
    constexpr uint32_t kTileDesc = kSfTile >> 4;
    const uint64_t da0 = umma_desc_sw128(base), db0 = umma_desc_sw128(base + Cfg::A_BYTES);
    const uint64_t ds0 = scale_desc(scales);
    int acc = 0, st = 0;
    uint32_t acc_ph = 0, ph = 0;
    bool ok = true;
    // The odd CTA's warp passes its epilogue's reads on: a release at the
    // cluster's scope takes about 1000 clocks, which the epilogue warps
    // would all wait for (20479 x 4096 x 1024 GELU 58 us, 80 with theirs).
    for (int t = rank == 0 ? total : first; t < total && ok; t += step) {
      ok = warp_mbar_wait(tempty_bar(acc), acc_ph, abort_flag);
      if (ok && lane == 0) arrive_cluster(of_cta0(peer_bar(acc)));
      __syncwarp();
      acc ^= 1;
      if (acc == 0) acc_ph ^= 1u;
    }
    for (int t = rank == 0 ? first : total; t < total; t += step) {
      const uint32_t sf_shift = static_cast<uint32_t>((t % n_tiles) * BN % 128) / 32;
      if (ok) ok = warp_mbar_wait(tempty_bar(acc), acc_ph ^ 1u, abort_flag);
      if (CG == 2 && ok) ok = warp_wait_cluster(peer_bar(acc), acc_ph ^ 1u, abort_flag);
      tc_fence_after();
      const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(acc * BN);
#pragma unroll 1
      for (int kb = 0; kb < kb_count; ++kb) {
        if (ok) ok = warp_mbar_wait(full_bar(st), ph, abort_flag);
        tc_fence_after();
        const uint64_t da = da0 + static_cast<uint32_t>(st) * kStageDesc;
        const uint64_t db = db0 + static_cast<uint32_t>(st) * kStageDesc;
        const uint64_t ds = ds0 + static_cast<uint32_t>(st) * (Cfg::SF_BYTES >> 4);
        const uint32_t tsa = tmem_base + 2 * BN + st * Cfg::SF_COLS;  // [2 K tiles][4]
        const uint32_t tsb = tsa + 8;                                 // [2 K tiles][SFB_TILES][4]
        auto products = [&](int steps) {  // K = 64 each; constant but in the last stage
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            if (2 * c < steps) {
              tmem_cp_scales<CG>(tsa + 4 * c, ds + c * kTileDesc);
#pragma unroll
              for (int i = 0; i < Cfg::SFB_TILES; ++i)
                tmem_cp_scales<CG>(tsb + 4 * (c * Cfg::SFB_TILES + i), ds + (2 * (1 + i) + c) * kTileDesc);
            }
          }
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (k < steps)
              mma_mxf4<CG>(d_tmem, da + 2u * k, db + 2u * k, mx_idesc(CG * kBM, BN, 2 * (k & 1)), tsa + 4 * (k >> 1),
                           tsb + 4 * Cfg::SFB_TILES * (k >> 1) + sf_shift, (kb | k) != 0);
        };
        const int steps = (p.K - kb * kStageK + 63) / 64;
        if (elect_one() && ok) {
          if (steps >= 4)
            products(4);
          else
            products(steps);
          commit<CG>(empty_bar(st));
          if (kb == kb_count - 1) commit<CG>(tfull_bar(acc));
        }
        __syncwarp();
        if (++st == Cfg::STAGES) {
          st = 0;
          ph ^= 1u;
        }
      }
      acc ^= 1;
      if (acc == 0) acc_ph ^= 1u;
    }
    if (!ok && rank == 0) {  // every MMA issued completes before TMEM is freed (bounded)
      volatile int no_abort = 0;
      if (elect_one()) commit<CG>(spare);
      __syncwarp();
      warp_mbar_wait(spare, 0, &no_abort);
    }
  } else {  // ── epilogue
    const int w = warp - 2;
    const int quarter = warp & 3, part = w >> 2;  // warps 2..5, 6..9, ...: each quarter once
    const uint32_t box = boxes + static_cast<uint32_t>(w) * kUnitBytes;
    const uint32_t bias = biases + static_cast<uint32_t>(w) * kUnitCols * 4;
    auto bias_at = [&](int t, int c) {
      const int col = (t % n_tiles) * BN + part * kUnitCols + c;
      return p.bias && col < p.N ? __ldg(p.bias + col) : 0.f;
    };
    float b0 = 0.f, b1 = 0.f;
    if (first < total) {
      b0 = bias_at(first, lane);
      b1 = bias_at(first, 32 + lane);
    }
    int acc = 0, loads = 0, waited = 0;  // residual boxes issued / seen
    uint32_t acc_ph = 0;
    for (int t = first; t < total; t += step) {
      const int row0 = (t / n_tiles * CG + rank) * kBM + quarter * 32;
      const int col0 = (t % n_tiles) * BN + part * kUnitCols;
      const bool live = col0 < p.N && row0 < p.M;  // warp-uniform
      auto load_res = [&](int c) {
        if (lane == 0) {
          mbar_arrive_expect_tx(res_bar(w), kUnitBytes);
          tma_load_2d(box, &tmR, col0 + c, row0, res_bar(w));
        }
        ++loads;
      };
      if (lane == 0) bulk_wait_read_all();  // the box's last store has read it
      __syncwarp();
      if (kRes && live) load_res(0);
      asm volatile("st.shared.b32 [%0], %1;" ::"r"(bias + 4 * lane), "f"(b0) : "memory");
      asm volatile("st.shared.b32 [%0], %1;" ::"r"(bias + 4 * (32 + lane)), "f"(b1) : "memory");
      if (t + step < total) {
        b0 = bias_at(t + step, lane);
        b1 = bias_at(t + step, 32 + lane);
      }
      __syncwarp();
      if (!warp_mbar_wait(tfull_bar(acc), acc_ph, abort_flag)) break;
      tc_fence_after();
      uint32_t r[2][32];
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) +
                             static_cast<uint32_t>(acc * BN + part * kUnitCols);
      tmem_ld_32x32b_x32(taddr, r[0]);
      tmem_ld_32x32b_x32(taddr + 32, r[1]);
      tmem_wait_ld();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(tempty_bar(acc));
      acc ^= 1;
      if (acc == 0) acc_ph ^= 1u;
      if (!live) continue;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float v[32];
        finish32<EPI>(r[half], bias + 128 * half, v);
        if (F32 && half == 1) {  // the second 32 columns use the box again
          if (col0 + 32 >= p.N) break;
          if (lane == 0) bulk_wait_read_all();
          __syncwarp();
          if (kRes) load_res(32);
        }
        if (kRes && (F32 || half == 0)) {
          if (!warp_mbar_wait(res_bar(w), waited & 1, abort_flag)) break;
          ++waited;
        }
        constexpr int kSlots = F32 ? 8 : 4;  // 16-byte slots of a row for 32 columns
#pragma unroll
        for (int q = 0; q < kSlots; ++q) {
          const uint32_t at = box_slot(box, lane, q + (F32 ? 0 : 4 * half));
          if constexpr (F32) {
            float4 o = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
            if (kRes) {
              const uint4 x = lds128(at);
              o.x += __uint_as_float(x.x); o.y += __uint_as_float(x.y);
              o.z += __uint_as_float(x.z); o.w += __uint_as_float(x.w);
            }
            sts128(at, make_uint4(__float_as_uint(o.x), __float_as_uint(o.y), __float_as_uint(o.z),
                                  __float_as_uint(o.w)));
          } else {
            if (kRes) {
              const uint4 x = lds128(at);
              const uint32_t x4[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float2 f = unpack2<OUT>(x4[e]);
                v[8 * q + 2 * e] += f.x;
                v[8 * q + 2 * e + 1] += f.y;
              }
            }
            sts128(at, make_uint4(pack2<OUT>(v[8 * q], v[8 * q + 1]), pack2<OUT>(v[8 * q + 2], v[8 * q + 3]),
                                  pack2<OUT>(v[8 * q + 4], v[8 * q + 5]), pack2<OUT>(v[8 * q + 6], v[8 * q + 7])));
          }
        }
        if (F32 || half == 1) {
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&tmC, box, col0 + (F32 ? 32 * half : 0), row0);
            bulk_commit();
          }
        }
      }
      if (*abort_flag) break;
    }
    if (kRes && waited < loads) {  // a load in flight lands before the CTA leaves (bounded)
      volatile int no_abort = 0;
      mbar_wait(res_bar(w), waited & 1, &no_abort);
    }
    if (lane == 0) bulk_wait_all();  // this warp's stores are complete
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();  // neither CTA leaves while the other one uses its memory
  if (threadIdx.x == 0 && *abort_flag && p.err) atomicOr(p.err, kErrTimeout);
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    if constexpr (CG == 1)
      tmem_dealloc(*tmem_slot, Cfg::TMEM_COLS);
    else
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(*tmem_slot), "r"(Cfg::TMEM_COLS)
                   : "memory");
  }
}

// ── host ────────────────────────────────────────────────────────────────────
PFN_cuTensorMapEncodeTiled_v12000 encoder() {
  static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      ptr = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
  }();
  return fn;
}

// 2-D map over a dense [rows, cols] buffer with boxes of 128 bytes x box_rows,
// 128-byte swizzle or none.
bool make_map(CUtensorMap* map, CUtensorMapDataType type, int esz, const void* ptr, long long rows, int cols,
              int box_rows, bool swizzled = true) {
  auto enc = encoder();
  if (!enc) return false;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(cols) * esz};
  const cuuint32_t box[2] = {static_cast<cuuint32_t>(128 / esz), static_cast<cuuint32_t>(box_rows)};
  const cuuint32_t estr[2] = {1, 1};
  return enc(map, type, 2, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             swizzled ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// Scale tiles as rows of 128 bytes, four to a tile, in boxes of two tiles.
bool make_scale_map(CUtensorMap* map, const uint8_t* scale, int rows, int cols) {
  return make_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, scale, (rows + 127ll) / 128 * ((cols + 127) / 128) * 4, 128, 8,
                  false);
}

template <int BN, int EPI, Out OUT, int CG>
cudaError_t launch_tile(const MxGemmArgs& g, const MxParams& p, cudaStream_t s, std::string* why) {
  using Cfg = MxCfg<BN, CG>;
  CUtensorMap ma, mb, msa, msb, mc, mr;
  const CUtensorMapDataType ct = OUT == kF32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                 : OUT == kF16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                               : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const int esz = OUT == kF32 ? 4 : 2;
  const CUtensorMapDataType u8 = CU_TENSOR_MAP_DATA_TYPE_UINT8;
  bool ok = make_map(&ma, u8, 1, g.aq, g.M, g.K / 2, kBM) && make_map(&mb, u8, 1, g.wq, g.N, g.K / 2, Cfg::B_ROWS) &&
            make_scale_map(&msa, g.a_scale, g.M, g.K) && make_scale_map(&msb, g.w_scale, g.N, g.K) &&
            make_map(&mc, ct, esz, g.C, g.M, g.N, 32);
  mr = mc;  // unused without a residual
  if (ok && EPI == JB_EPI_RESIDUAL) ok = make_map(&mr, ct, esz, g.resid, g.M, g.N, 32);
  if (!ok) {
    if (why) *why = "linear(mxfp4): cuTensorMapEncodeTiled failed";
    return cudaErrorInvalidValue;
  }
  auto kern = gemm_mxfp4_kernel<BN, EPI, OUT, CG>;
  int dev = 0;
  cudaGetDevice(&dev);
  // the shared-memory opt-in is a property of each device's context
  static std::atomic<uint8_t> attr_set[64];
  if (dev < 0 || dev >= 64 || !attr_set[dev].load(std::memory_order_acquire)) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM);
    if (e != cudaSuccess) return e;
    if (dev >= 0 && dev < 64) attr_set[dev].store(1, std::memory_order_release);
  }
  const long long tiles = ((g.M + CG * kBM - 1ll) / (CG * kBM)) * ((g.N + BN - 1) / BN);
  const int grid = static_cast<int>(std::min<long long>(num_sms(dev) / CG, tiles)) * CG;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(Cfg::THREADS);
  cfg.dynamicSmemBytes = Cfg::SMEM;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = CG;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = CG == 1 ? 0 : 1;
  return cudaLaunchKernelEx(&cfg, kern, ma, mb, msa, msb, mc, mr, p);
}

template <int BN, Out OUT, int CG>
cudaError_t launch_epi(const MxGemmArgs& g, const MxParams& p, cudaStream_t s, std::string* why) {
  switch (g.epi) {
    case JB_EPI_GELU: return launch_tile<BN, JB_EPI_GELU, OUT, CG>(g, p, s, why);
    case JB_EPI_QUICK_GELU: return launch_tile<BN, JB_EPI_QUICK_GELU, OUT, CG>(g, p, s, why);
    case JB_EPI_RESIDUAL: return launch_tile<BN, JB_EPI_RESIDUAL, OUT, CG>(g, p, s, why);
    default: return launch_tile<BN, JB_EPI_NONE, OUT, CG>(g, p, s, why);
  }
}
template <int BN, int CG>
cudaError_t launch_out(const MxGemmArgs& g, const MxParams& p, cudaStream_t s, std::string* why) {
  if (g.c_dtype == JB_DT_F16) return launch_epi<BN, kF16, CG>(g, p, s, why);
  // f32 outputs hold 64 accumulators and 32 results: more than the 448
  // threads of BN = 192 have registers for
  if constexpr (BN < 192)
    if (g.c_dtype == JB_DT_F32) return launch_epi<BN, kF32, CG>(g, p, s, why);
  return launch_epi<BN, kBf16, CG>(g, p, s, why);
}

}  // namespace

cudaError_t launch_linear_mxfp4(const MxGemmArgs& g, cudaStream_t s, std::string* why) {
  if (g.M == 0) return cudaSuccess;
  const long long m_tiles = (g.M + kBM - 1ll) / kBM;
  // tile numbers, and scale rows (four to a scale tile) as TMA coordinates
  const long long k_tiles = (g.K + 127) / 128;
  if (m_tiles * ((g.N + 63) / 64) > INT32_MAX / 2 ||
      (std::max<long long>(m_tiles, (g.N + 127ll) / 128) + 2) * k_tiles * 4 > INT32_MAX) {
    if (why) *why = "linear(mxfp4): more tiles than 32 bits number";
    return cudaErrorInvalidValue;
  }
  MxParams p{g.bias, g.M, g.N, g.K, g.err};
  int dev = 0;
  cudaGetDevice(&dev);
  const long long sms = num_sms(dev);
  // Width of the tile.  One wave of 128 x 64 tiles, when it holds them all, is
  // the shortest way through (12 x 2304 x 768: 3.6 us, 3.9 with 128 columns; 777 x
  // 1024 x 4096: 6.9, 7.8); two waves of it are not (1777 x 1024 x 4096: 10.7, 8.0).
  if (m_tiles * ((g.N + 63) / 64) <= sms) return launch_out<64, 1>(g, p, s, why);
  // Pairs do more per wave, and cost more per wave and to start.  In units of
  // the time of a K column in a 128 x 128 tile, waves measured at K = 384 to
  // 4096 take max(K, 640) + 576 and, by pairs, max(K, 640) + 1024 with 600 once.
  // 128 columns against pairs: 5000 x 768 x 768 5.5 us, 6.7; 3000 x 2304 x 768
  // 6.6, 7.1; 9000 x 2304 x 768 13.8, 13.0; 3000 x 1024 x 4096 12.1, 9.2; 20479 x
  // 4096 x 1024 53.7, 47.1.
  const long long k = std::max<long long>(g.K, 640);
  auto waves = [](long long tiles, long long slots) { return (tiles + slots - 1) / slots; };
  const long long one = waves(m_tiles * ((g.N + 127) / 128), sms) * (k + 576);
  const long long two = waves((m_tiles + 1) / 2 * ((g.N + 191) / 192), sms / 2) * (k + 1024) + 600;
  if (g.c_dtype == JB_DT_F32 || one <= two) return launch_out<128, 1>(g, p, s, why);
  return launch_out<192, 2>(g, p, s, why);
}

}  // namespace jb
