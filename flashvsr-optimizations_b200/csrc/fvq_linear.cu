// fvq_linear.cu -- matrix product with bias, activation, gate and residual in its epilogue.
//
//   z = x W^T  [* sx_m * sw_n]  + b                     fp32 accumulation (tcgen05)
//   h = act(z)   or, gated (W = [Wg; Wu], 2n rows),  act(z_g) * z_u
//   y = bf16(h + r)                                     one rounding
//
// Operands bf16 (kind::f16) or E4M3 with one fp32 scale per row (kind::f8f6f4); both take
// 128 bytes of K per row and tile, so one code serves both and only the instruction
// descriptor differs.  Three kernels:
//
//   linear_pair_kernel   many tokens: tensor-bound.  Persistent clusters of two CTAs
//     (cta_group::2, M = 256 tokens, N = bn columns), W and x tiles by TMA through a ring of
//     stages, two accumulators in TMEM so that the next tile's products run under the
//     epilogue.  Gated: the even CTA loads the tile's Wg rows, the odd one its Wu rows, so
//     both halves of an output column meet in the same TMEM lane and no pass over h is made.
//     Where the tiles are few and K is long, two to four pairs share a tile's K and join their
//     accumulators through distributed shared memory (kSplitK).
//   linear_split_kernel  few tokens: bound by reading W once.  The operands change places:
//     `wr` rows of W are the M side, up to 128 tokens the N side, so that a few tokens cost
//     N = 16 instructions and not a 128-row tile; K is split over a cluster of up to eight
//     CTAs until every SM streams its share of W, and each CTA sends its partial sums to the
//     one that owns their tokens, through distributed shared memory; they are added in rank
//     order (no atomics, no workspace, the same bits on every run).
//   linear_vector_kernel  one or two tokens: W streamed through rings in shared memory by bulk
//     copies, fp32 FMAs, x in registers.  No tensor-core pipeline to set up, fill and
//     drain, which is half of the split kernel's time at this size.
//
// Measured on a B200, launches back to back in a CUDA graph, operands larger than L2 in all
// (a copy moves 6.5 TB/s, torch's bf16 product reaches 1672 TFLOP/s for a moment, 1398 for seconds):
//   pair    (m x k -> n) bf16 15360 x 8960 -> 1536 with residual: 270 to 280 us (1.51 to
//           1.56 PFLOP/s).  E4M3 gated 7680 x 1536 -> 2 * 8960: 165 to 215 us with the clock (2.0
//           to 2.6 PFLOP/s).  At 4096 rows of the same products the tensor pipe is 80% and 72%
//           active; the epilogue's arithmetic shares issue slots and power with it (7680 x 1536
//           -> 2 * 4480: 75 us without an activation, 84 with one).
//   split   24 x 8960 -> 1536: E4M3 7.0 us, with bias and residual 7.5 (13.8 MB of W: 2.1 us at a
//           copy's rate; the rest is the start, the exchange of partial sums and the epilogue),
//           bf16 9.2 and 9.7; 24 x 1536 -> 8960: 6.1 and, bf16, 8.0.
//   vector  bf16 1 x 1536 -> 8960: 7.2 us, 1 x 8960 -> 1536: 6.8 us (27.5 MB, 4.0 TB/s, about
//           2.5 us of it start and end), 1 x 4096 -> 12288: 17.1 us (5.9 TB/s).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstring>

#include "fvq_internal.h"
#include "fvq_launch.h"
#include "fvq_ptx.cuh"

namespace fvq {

namespace {

constexpr int kKB = 128;  // bytes of K per row and tile: one 128B swizzle row

// ---------------------------------------------------------------- activations
enum Act { kActNone = 0, kActRelu = 1, kActGelu = 2, kActGeluTanh = 3, kActSilu = 4 };

// 2^x and 1/x as the hardware approximates them (about 2^-22), results below the smallest normal
// flushed to zero.
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ uint64_t f2_both(float v) { return f2_pack(v, v); }

// z * sigmoid(t) with t and z of one sign, u = t / ln 2, for two values: one exponential and one
// reciprocal each, without the cancellation that 1 + tanh has for negative z.  The exponential
// is of -|t|, so the divisor stays in [1, 2] and the negative tail keeps its digits; it is taken
// 2^8 too large (and z 2^8 too small with it) so that it is not flushed before the product is.
__device__ __forceinline__ uint64_t z_sigmoid2(uint64_t z2, uint64_t u2) {
  float z[2], u[2], e[2], r[2];
  f2_split(z2, z[0], z[1]);
  f2_split(u2, u[0], u[1]);
#pragma unroll
  for (int j = 0; j < 2; ++j) e[j] = ex2(8.0f - fabsf(u[j]));
  const uint64_t e2 = f2_pack(e[0], e[1]);
  float d[2];
  f2_split(f2_fma(e2, f2_both(0x1p-8f), f2_both(1.0f)), d[0], d[1]);
#pragma unroll
  for (int j = 0; j < 2; ++j) r[j] = rcp_approx_ftz(d[j]);
  const uint64_t num = f2_mul(f2_mul(z2, f2_both(0x1p-8f)),
                              f2_pack(z[0] < 0.0f ? e[0] : 256.0f, z[1] < 0.0f ? e[1] : 256.0f));
  return f2_mul(num, f2_pack(r[0], r[1]));
}

// 0.5 z erfc(-z / sqrt 2) for two values.  With x = |z| / sqrt 2 and s = 1 / (1 + x / 2),
// g = 0.5 erfc(x) = s 2^(p(s) - x^2 log2 e), where p is the polynomial of degree 7 that meets
// log2(0.5 erfc(x) e^(x^2) / s) at the Chebyshev nodes of s over 0 <= x <= 9.6.  g is off by
// 1e-6 of itself up to x = 2, and by 1e-5 at x = 9 for the rounding of x^2.  The result is
// z (1 - g) for positive z and z g for the others, which has no cancellation.
__device__ __forceinline__ uint64_t gelu2(uint64_t z2) {
  float z[2], a[2], g[2], s[2];
  f2_split(z2, z[0], z[1]);
#pragma unroll
  for (int j = 0; j < 2; ++j) s[j] = rcp_approx_ftz(fmaf(fabsf(z[j]), 0.353553385f, 1.0f));
  const uint64_t s2 = f2_pack(s[0], s[1]);
  constexpr float kP[8] = {-2.82571697f, 1.44092202f, 0.566950738f, -0.0534122437f,
                           0.498900861f, -1.43910909f, 1.08193898f, -0.270475209f};
  uint64_t p = f2_both(kP[7]);
#pragma unroll
  for (int i = 6; i >= 0; --i) p = f2_fma(p, s2, f2_both(kP[i]));
  f2_split(f2_fma(f2_mul(z2, z2), f2_both(-0.7213475204444817f), p), a[0], a[1]);  // log2(e) / 2
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    g[j] = s[j] * ex2(a[j]);
    g[j] = z[j] > 0.0f ? 1.0f - g[j] : g[j];
  }
  return f2_mul(z2, f2_pack(g[0], g[1]));
}

// act(z) of two values in fp32; silu is z sigmoid(z), the tanh form of gelu z sigmoid(2 sqrt(2 /
// pi) (z + 0.044715 z^3)).  relu keeps NaN.
template <int kAct>
__device__ __forceinline__ uint64_t activate2(uint64_t z2) {
  constexpr float kLog2e = 1.4426950408889634f;
  if constexpr (kAct == kActRelu) {
    float lo, hi;
    f2_split(z2, lo, hi);
    return f2_pack(lo < 0.0f ? 0.0f : lo, hi < 0.0f ? 0.0f : hi);
  } else if constexpr (kAct == kActGelu) {
    return gelu2(z2);
  } else if constexpr (kAct == kActGeluTanh) {
    constexpr float kA = 1.5957691216057308f * kLog2e;
    const uint64_t q = f2_fma(f2_mul(z2, z2), f2_both(kA * 0.044715f), f2_both(kA));
    return z_sigmoid2(z2, f2_mul(z2, q));
  } else if constexpr (kAct == kActSilu) {
    return z_sigmoid2(z2, f2_mul(z2, f2_both(kLog2e)));
  } else {
    return z2;
  }
}

// ---------------------------------------------------------------- MMA
template <bool kF8>
__device__ __forceinline__ void mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                         uint32_t accumulate) {
  if constexpr (kF8)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}

template <bool kF8>
__device__ __forceinline__ void mma_one(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                        uint32_t accumulate) {
  if constexpr (kF8)
    mma_f8(d, a, b, idesc, accumulate);
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}

// fp32 accumulator; both operands BF16 (kind::f16) or both E4M3 (kind::f8f6f4), K-major
template <bool kF8>
__host__ __device__ constexpr uint32_t instr_desc(int m, int n) {
  return (1u << 4) | (kF8 ? 0u : (1u << 7) | (1u << 10)) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(m >> 4) << 24);
}

__device__ __forceinline__ void flag(int* abort_flag, uint32_t* err_word, uint32_t bit) {
  atomicOr(err_word, bit);
  *reinterpret_cast<volatile int*>(abort_flag) = 1;
}

// from one lane of a converged warp
__device__ __forceinline__ void warp_flag(int* abort_flag, uint32_t* err_word, uint32_t bit) {
  if (elect_one()) flag(abort_flag, err_word, bit);
  __syncwarp();
}

__device__ __forceinline__ bool warp_aborted(const int* abort_flag) {
  return __shfl_sync(0xFFFFFFFFu, *reinterpret_cast<const volatile int*>(abort_flag), 0) != 0;
}

// ---------------------------------------------------------------- many tokens
constexpr int kPairTokens = 256;                  // per pair; 128 per CTA
constexpr int kPairABytes = 128 * kKB;            // 16 KB
constexpr int kPairBBytes = 128 * kKB;            // half of the (up to 256) W rows
constexpr int kPairStageBytes = kPairABytes + kPairBBytes;
constexpr int kPairStages = 5;
constexpr int kPairEpiWarps = 8;                  // two per TMEM lane quadrant
constexpr int kPairThreads = 64 + 32 * kPairEpiWarps;
constexpr int kChunk = 32;                        // output columns staged at a time (64 bytes)
constexpr int kChunkBytes = 32 * kChunk * 2;      // of one warp's 32 rows
constexpr int kParamBytes = kChunk * 2 * 8;       // a chunk's scales and biases, both halves of a gate
constexpr int kPairStagingOff = kPairStages * kPairStageBytes;
constexpr int kPairParamOff = kPairStagingOff + kPairEpiWarps * 2 * kChunkBytes;
constexpr int kPairBarrierOff = kPairParamOff + kPairEpiWarps * kParamBytes;
constexpr int kPairSmemBytes = kPairBarrierOff + 512;
constexpr int kAccCols = 256;                     // TMEM columns per accumulator
static_assert(kPairSmemBytes <= 232448, "pair plan exceeds shared memory");

struct PairBars {
  uint64_t full[kPairStages];     // even CTA: both CTAs' loads of the stage landed
  uint64_t empty[kPairStages];    // the pair's MMAs on the stage completed
  uint64_t acc_full[2];
  uint64_t acc_empty[2];          // even CTA: both epilogues drained the accumulator
  uint64_t res_full[kPairEpiWarps][2];  // residual chunk landed in the warp's staging buffer
  uint64_t teardown;
  uint64_t odd_done;              // even CTA: the odd one's producer has ended,
  uint32_t odd_fills;             // after this many fills of its stages
  uint32_t tmem_base;
  int abort_flag;
};
static_assert(sizeof(PairBars) <= 512, "pair barrier area");

struct LinearArgs {
  const float* sx;        // [m] or null
  const float* sw;        // [wn] or null
  const uint16_t* bias;   // [wn] or null
  int m, n, k_tiles;
  int act;
  int bn;                 // accumulator columns per tile (pair kernel)
  int residual;           // 0 / 1
  int split, k_each, k_more;  // pair kernel: pairs per tile; K tiles each, and one more for the first k_more
  uint64_t wait_limit;
  uint32_t* err_word;
};

// Scales and biases of 32 W rows, one per lane, on their way to shared memory: fetched a chunk
// ahead, so that their latency (an L2 miss for every new tile) is off the epilogue's path.
struct ColumnParam {
  float scale, bias;
};

template <bool kF8>
__device__ __forceinline__ ColumnParam column_param(const LinearArgs& a, int row, bool inside) {
  ColumnParam c = {1.0f, 0.0f};
  if (inside) {
    if constexpr (kF8) c.scale = a.sw[row];
    if (a.bias != nullptr) c.bias = __uint_as_float(static_cast<uint32_t>(a.bias[row]) << 16);
  }
  return c;
}

// Shared-memory layout of 32 columns: E4M3 16 bytes per column pair (two scales, two biases),
// bf16 the 32 biases.
template <bool kF8>
__device__ __forceinline__ void put_param(float* at, int lane, ColumnParam c) {
  if constexpr (kF8) {
    at[(lane >> 1) * 4 + (lane & 1)] = c.scale;
    at[(lane >> 1) * 4 + 2 + (lane & 1)] = c.bias;
  } else {
    at[lane] = c.bias;
  }
}

// 32 accumulator columns of one row -> z = acc [* sx * sw] + b, in pairs.
template <bool kF8>
__device__ __forceinline__ void affine32(const uint32_t (&r)[32], uint64_t sx2, const float* param,
                                         uint64_t (&z)[16]) {
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "r"(r[2 * i]), "r"(r[2 * i + 1]));
    if constexpr (kF8) {
      const ulonglong2 c = *reinterpret_cast<const ulonglong2*>(param + 4 * i);
      z[i] = f2_fma(f2_mul(v, sx2), c.x, c.y);
    } else {
      z[i] = f2_add(v, *reinterpret_cast<const uint64_t*>(param + 2 * i));
    }
  }
}

template <int kAct, bool kGated>
__device__ __forceinline__ void act32_t(uint64_t (&z)[16], const uint64_t (&u)[16]) {
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    z[i] = activate2<kAct>(z[i]);
    if constexpr (kGated) z[i] = f2_mul(z[i], u[i]);
  }
}

template <bool kGated>
__device__ __forceinline__ void act32(int act, uint64_t (&z)[16], const uint64_t (&u)[16]) {
  switch (act) {
    case kActRelu: act32_t<kActRelu, kGated>(z, u); break;
    case kActGelu: act32_t<kActGelu, kGated>(z, u); break;
    case kActGeluTanh: act32_t<kActGeluTanh, kGated>(z, u); break;
    case kActSilu: act32_t<kActSilu, kGated>(z, u); break;
    default: act32_t<kActNone, kGated>(z, u); break;
  }
}

__device__ __forceinline__ uint32_t cluster_id() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%clusterid.x;" : "=r"(r));
  return r;
}

__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// kSplitK: one tile per cluster of 2 * split CTAs, each pair taking its share of K.
template <bool kF8, bool kGated, bool kSplitK>
__global__ void __launch_bounds__(kPairThreads, 1)
    linear_pair_kernel(const __grid_constant__ CUtensorMap tmap_x,
                       const __grid_constant__ CUtensorMap tmap_w,
                       const __grid_constant__ CUtensorMap tmap_r,
                       const __grid_constant__ CUtensorMap tmap_y, const LinearArgs a) {
  extern __shared__ __align__(1024) uint8_t smem[];
  if ((smem_u32(smem) & 1023u) != 0) {
    if (threadIdx.x == 0) atomicOr(a.err_word, kErrSmemAlign);
    return;  // both CTAs see the same layout, so both return here
  }
  auto* bars = reinterpret_cast<PairBars*>(smem + kPairBarrierOff);
  int* abort_flag = &bars->abort_flag;
  const int warp = warp_index_uniform();
  const int lane = threadIdx.x & 31;
  const uint32_t cta = cluster_ctarank(), rank = cta & 1u;  // in the cluster, in the pair
  const bool even = rank == 0;
  const int split = kSplitK ? a.split : 1, part = kSplitK ? static_cast<int>(cta >> 1) : 0;
  const int pairs = kSplitK ? static_cast<int>(gridDim.x) / (2 * split) : gridDim.x / 2;
  const int pair = kSplitK ? static_cast<int>(cluster_id()) : blockIdx.x / 2;
  const int kt0 = kSplitK ? part * a.k_each + min(part, a.k_more) : 0;
  const int kt1 = kSplitK ? kt0 + a.k_each + (part < a.k_more ? 1 : 0) : a.k_tiles;
  const int bn = a.bn, out_cols = kGated ? bn / 2 : bn;
  const int n_blocks = (a.n + out_cols - 1) / out_cols;
  const int tiles = ((a.m + kPairTokens - 1) / kPairTokens) * n_blocks;
  const int count = pair < tiles ? (tiles - 1 - pair) / pairs + 1 : 0;  // same in both CTAs
  const uint64_t wait_limit = a.wait_limit;
  const uint64_t teardown_limit = wait_limit > kDefaultWaitLimit ? wait_limit : kDefaultWaitLimit;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kPairStages; ++s) {
      mbar_init(&bars->full[s], 1);
      mbar_init(&bars->empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&bars->acc_full[b], 1);
      mbar_init(&bars->acc_empty[b], 2 * kPairEpiWarps);
      for (int w = 0; w < kPairEpiWarps; ++w) mbar_init(&bars->res_full[w][b], 1);
    }
    mbar_init(&bars->teardown, 1);
    mbar_init(&bars->odd_done, 1);
    bars->abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async_smem();
    prefetch_tmap(&tmap_x);
    prefetch_tmap(&tmap_w);
  }
  if (warp == 1) {
    tmem_alloc_pair(&bars->tmem_base, 2 * kAccCols);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync();  // barriers of both CTAs initialised before any remote arrive
  tc_fence_after();
  grid_dependency_wait();
  const uint32_t tmem = bars->tmem_base;
  const auto even_addr = [&](const void* p) { return mapa_shared(smem_u32(p), cta & ~1u); };
  const auto odd_addr = [&](const void* p) { return mapa_shared(smem_u32(p), cta | 1u); };

  if (warp == 0) {
    // ------------------------------------------------------------ producer (both CTAs)
    uint32_t fills = 0;
    const uint32_t w_bytes = static_cast<uint32_t>(bn / 2) * kKB;
    const int k_step = kF8 ? kKB : kKB / 2;  // elements
    int stage = 0;
    uint32_t phase = 0;
    for (int i = 0; i < count && !warp_aborted(abort_flag); ++i) {
      const int t = pair + i * pairs;
      const int nb = t % n_blocks, mb = t / n_blocks;  // N block fastest: x rows stay in L2
      const int x_row = mb * kPairTokens + static_cast<int>(rank) * 128;
      // gated: Wg rows in the even CTA, the same columns' Wu rows in the odd one
      const int w_row = kGated ? nb * out_cols + static_cast<int>(rank) * a.n
                               : nb * bn + static_cast<int>(rank) * (bn / 2);
      for (int kt = kt0; kt < kt1; ++kt) {
        if (!warp_wait_cluster_bounded(&bars->empty[stage], phase ^ 1u, wait_limit)) {
          warp_flag(abort_flag, a.err_word, kErrWaitProducer);
          break;
        }
        uint8_t* sa = smem + stage * kPairStageBytes;
        const uint32_t bar = even_addr(&bars->full[stage]);
        if (elect_one()) {
          if (even) mbar_arrive_expect_tx(&bars->full[stage], 2 * (kPairABytes + w_bytes));
          tma_load_2d_pair(sa, &tmap_x, bar, kt * k_step, x_row);
          tma_load_2d_pair(sa + kPairABytes, &tmap_w, bar, kt * k_step, w_row);
        }
        __syncwarp();
        ++fills;
        if (++stage == kPairStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    grid_launch_dependents();  // this CTA's last tile is on its way
    if (!pair_drain_loads<kPairStages>(cta, bars->full, &bars->odd_done, &bars->odd_fills, fills,
                                       [&](uint32_t) { return kPairABytes + w_bytes; }, teardown_limit))
      warp_flag(abort_flag, a.err_word, kErrWaitTeardown);
    // the odd CTA: the even one's MMAs, and their arrivals here, are over (its MMA warp may have one
    // wait and its own teardown ahead)
    if (!even && !warp_wait_cluster_bounded(&bars->teardown, 0, limit_times(teardown_limit, 3)))
      warp_flag(abort_flag, a.err_word, kErrWaitTeardown);
    if constexpr (kSplitK) cluster_sync();  // the partial sums are in place
  } else if (warp == 1) {
    if (even) {
      // ---------------------------------------------------------- MMA issuer (even CTA)
      const uint32_t idesc = instr_desc<kF8>(kPairTokens, bn);
      int stage = 0;
      uint32_t phase = 0;
      bool issued_any = false, ok = true;
      for (int i = 0; ok && i < count && !warp_aborted(abort_flag); ++i) {
        const int buf = i & 1;
        if (!warp_wait_cluster_bounded(&bars->acc_empty[buf],
                                       (static_cast<uint32_t>(i >> 1) & 1u) ^ 1u, wait_limit)) {
          warp_flag(abort_flag, a.err_word, kErrWaitMma);
          break;
        }
        tc_fence_after();
        const uint32_t d = tmem + static_cast<uint32_t>(buf * kAccCols);
        for (int kt = kt0; kt < kt1; ++kt) {
          if (!warp_wait_cluster_bounded(&bars->full[stage], phase, wait_limit)) {
            warp_flag(abort_flag, a.err_word, kErrWaitMma);
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + stage * kPairStageBytes);
          const uint64_t adesc = make_smem_desc(sa, 16, 1024, 2);
          const uint64_t bdesc = make_smem_desc(sa + kPairABytes, 16, 1024, 2);
          const uint32_t empty_odd = odd_addr(&bars->empty[stage]);
          if (elect_one()) {
#pragma unroll
            for (int j = 0; j < 4; ++j)  // 32-byte K steps inside the 128B swizzle atom
              mma_pair<kF8>(d, adesc + static_cast<uint64_t>(2 * j),
                            bdesc + static_cast<uint64_t>(2 * j), idesc,
                            (kt > kt0 || j > 0) ? 1u : 0u);
            tc_commit_pair(smem_u32(&bars->empty[stage]));
            tc_commit_pair(empty_odd);
          }
          __syncwarp();
          issued_any = true;
          if (++stage == kPairStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        const uint32_t acc_odd = odd_addr(&bars->acc_full[buf]);
        if (elect_one()) {
          tc_commit_pair(smem_u32(&bars->acc_full[buf]));
          tc_commit_pair(acc_odd);
        }
        __syncwarp();
      }
      // Nothing issued may run on when TMEM and the ring go, whichever warp gives up, and when: so
      // this waits whether or not the flag is up by now.
      pair_commit_teardown(&bars->teardown, cta, issued_any);
      if (!warp_wait_cluster_bounded(&bars->teardown, 0, teardown_limit))
        warp_flag(abort_flag, a.err_word, kErrWaitTeardown);
    }
    if constexpr (kSplitK) cluster_sync();
  } else {
    // ------------------------------------------------------------ epilogue (both CTAs)
    // Warp w: TMEM lanes 32 * (w % 4).., every second 32-column chunk of the tile.  A chunk
    // goes through one of the warp's two staging buffers: the residual chunk is loaded into
    // it, the results take its place and leave by a TMA store (which also clips the edges).
    const int quad = warp & 3, half = (warp - 2) >> 2;
    const int trow = quad * 32 + lane;
    uint8_t* staging = smem + kPairStagingOff + (warp - 2) * 2 * kChunkBytes;
    float* param = reinterpret_cast<float*>(smem + kPairParamOff + (warp - 2) * kParamBytes);
    float* param_u = param + (kF8 ? 2 : 1) * kChunk;
    uint64_t* res_full = bars->res_full[warp - 2];
    const int chunks = out_cols / kChunk;
    const uint32_t swizzle = (lane >> 1) & 3u;  // 64B swizzle of row `lane`
    uint32_t uses = 0;  // chunks through the staging buffers so far
    bool ok = true;
    // Split K: the accumulator goes to shared memory, over the ring (its loads have landed and
    // the MMAs that read it are complete), 16 bytes of columns by row: sums[col / 4][row].
    // After the cluster's barrier CTA `cta` joins every split-th chunk, adding the sums of the
    // CTAs of its parity in rank order.
    float4* sums = reinterpret_cast<float4*>(smem);
    if constexpr (kSplitK) {
      if (!mbar_wait_cluster_bounded(&bars->acc_full[0], 0, wait_limit)) {
        flag(abort_flag, a.err_word, kErrWaitEpilogue);
        ok = false;
      }
      ok = __all_sync(0xFFFFFFFFu, ok);
      tc_fence_after();
      for (int c = half; ok && c < bn / kChunk; c += 2) {
        uint32_t r[32];
        tmem_ld_32x32b_x32(tmem + static_cast<uint32_t>(c * kChunk) + (static_cast<uint32_t>(quad * 32) << 16), r);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 8; ++j)
          sums[(c * 8 + j) * 128 + trow] =
              make_float4(__uint_as_float(r[4 * j]), __uint_as_float(r[4 * j + 1]),
                          __uint_as_float(r[4 * j + 2]), __uint_as_float(r[4 * j + 3]));
      }
      tc_fence_before();
      __syncwarp();
      cluster_sync();
    }
    const auto joined = [&](int c, uint32_t (&r)[32]) {  // 32 columns of this row, all parts
      const uint32_t at = smem_u32(sums + c * 8 * 128 + trow);
#pragma unroll
      for (int j = 0; j < 32; ++j) r[j] = 0;
      for (int q = 0; q < split; ++q) {
        const uint32_t peer = mapa_shared(at, 2u * static_cast<uint32_t>(q) + rank);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float4 v = ld_cluster_f4(peer + static_cast<uint32_t>(j * 128 * 16));
          r[4 * j] = __float_as_uint(__uint_as_float(r[4 * j]) + v.x);
          r[4 * j + 1] = __float_as_uint(__uint_as_float(r[4 * j + 1]) + v.y);
          r[4 * j + 2] = __float_as_uint(__uint_as_float(r[4 * j + 2]) + v.z);
          r[4 * j + 3] = __float_as_uint(__uint_as_float(r[4 * j + 3]) + v.w);
        }
      }
    };
    const int c_first = part + split * half, c_step = 2 * split;  // split 1: every second chunk
    for (int i = 0; ok && i < count; ++i) {
      const int t = pair + i * pairs;
      const int nb = t % n_blocks, mb = t / n_blocks;
      const int row0 = mb * kPairTokens + static_cast<int>(rank) * 128 + quad * 32;
      const int row = mb * kPairTokens + static_cast<int>(rank) * 128 + trow;
      const float sx = kF8 && row < a.m ? a.sx[row] : 0.0f;
      const uint64_t sx2 = f2_pack(sx, sx);
      const int buf = i & 1;
      const int tile_col = nb * out_cols;
      const auto fetch = [&](int c, ColumnParam& g, ColumnParam& u) {
        const int col = tile_col + c * kChunk + lane;
        const bool in = c < chunks && col < a.n;
        g = column_param<kF8>(a, col, in);
        if constexpr (kGated) u = column_param<kF8>(a, a.n + col, in);
      };
      ColumnParam pg, pu;
      fetch(c_first, pg, pu);
      bool waited = kSplitK;
      for (int c = c_first; c < chunks; c += c_step) {
        const int col0 = tile_col + c * kChunk;
        const bool inside = col0 < a.n && row0 < a.m;  // warp-uniform
        uint8_t* stage_buf = staging + (uses & 1u) * kChunkBytes;
        __syncwarp();  // the previous chunk's parameters have been read
        put_param<kF8>(param, lane, pg);
        if constexpr (kGated) put_param<kF8>(param_u, lane, pu);
        fetch(c + c_step, pg, pu);
        if (inside) {
          // at most one committed store (of the other buffer) may still be reading
          if (lane == 0) {
            asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
            if (a.residual) {
              mbar_arrive_expect_tx(&res_full[uses & 1u], kChunkBytes);
              tma_load_2d(stage_buf, &tmap_r, &res_full[uses & 1u], col0, row0);
            }
          }
        }
        __syncwarp();
        if (!waited) {
          if (!mbar_wait_cluster_bounded(&bars->acc_full[buf], static_cast<uint32_t>(i >> 1) & 1u,
                                         wait_limit)) {
            flag(abort_flag, a.err_word, kErrWaitEpilogue);
            ok = false;
          }
          ok = __all_sync(0xFFFFFFFFu, ok);
          tc_fence_after();
          waited = true;
        }
        uint32_t r[32], v[32];
        const uint32_t taddr = tmem + static_cast<uint32_t>(buf * kAccCols + c * kChunk) +
                               (static_cast<uint32_t>(quad * 32) << 16);
        if (ok && inside) {
          if constexpr (kSplitK) {
            joined(c, r);
            if constexpr (kGated) joined(c + chunks, v);
          } else {
            tmem_ld_32x32b_x32(taddr, r);
            if constexpr (kGated) tmem_ld_32x32b_x32(taddr + out_cols, v);
          }
        }
        if (inside && a.residual) {
          // a residual load in flight has to land before its buffer is used or the CTA exits
          if (!mbar_wait_bounded(&res_full[uses & 1u], (uses >> 1) & 1u, teardown_limit)) {
            flag(abort_flag, a.err_word, kErrWaitEpilogue);
            ok = false;
          }
          ok = __all_sync(0xFFFFFFFFu, ok);
        }
        if constexpr (!kSplitK) tmem_ld_wait();
        if (!ok) break;
        if (!inside) continue;
        uint64_t z[16], u[16];
        affine32<kF8>(r, sx2, param, z);
        if constexpr (kGated) affine32<kF8>(v, sx2, param_u, u);
        act32<kGated>(a.act, z, u);
        // 16-byte piece q of row l sits at l * 64 + ((q ^ ((l >> 1) & 3)) * 16)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint4* at = reinterpret_cast<uint4*>(stage_buf + lane * 64 + ((q ^ swizzle) * 16));
          if (a.residual) {
            const uint4 w = *at;
            z[4 * q] = f2_add(z[4 * q], f2_of_bf16x2(w.x));
            z[4 * q + 1] = f2_add(z[4 * q + 1], f2_of_bf16x2(w.y));
            z[4 * q + 2] = f2_add(z[4 * q + 2], f2_of_bf16x2(w.z));
            z[4 * q + 3] = f2_add(z[4 * q + 3], f2_of_bf16x2(w.w));
          }
          *at = make_uint4(f2_to_bf16x2(z[4 * q]), f2_to_bf16x2(z[4 * q + 1]),
                           f2_to_bf16x2(z[4 * q + 2]), f2_to_bf16x2(z[4 * q + 3]));
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          tma_store_2d(&tmap_y, stage_buf, col0, row0);
          bulk_commit_group();
        }
        ++uses;
      }
      if (!ok || kSplitK) break;
      if (!waited) {  // fewer chunks than warps: still wait for and release the accumulator
        ok = mbar_wait_cluster_bounded(&bars->acc_full[buf], static_cast<uint32_t>(i >> 1) & 1u,
                                       wait_limit);
        if (!ok) flag(abort_flag, a.err_word, kErrWaitEpilogue);
        ok = __all_sync(0xFFFFFFFFu, ok);
        if (!ok) break;
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(even_addr(&bars->acc_empty[buf]));
    }
    if (lane == 0) bulk_wait_group0();  // stores complete before the CTA exits
  }

  tc_fence_before();
  __syncwarp();
  cluster_sync();  // no CTA leaves while the MMAs, arrivals or reads of others may touch it
  tc_fence_after();
  if (warp == 1) tmem_dealloc_pair(tmem, 2 * kAccCols);
}

// ---------------------------------------------------------------- few tokens
constexpr int kSplitStagesMax = 16;
constexpr int kSplitMax = 8;                      // CTAs per cluster (the portable limit)
constexpr int kSplitThreads = 320;                // producer, MMA issuer, eight epilogue warps
constexpr int kJoinThreads = 256;                 // a power of two, so that a thread keeps its columns
constexpr int kSplitBarrierBytes = 512;
// Shared memory: the ring of stages, then the partial sums of this CTA's tokens, as the
// cluster's CTAs send them (they may arrive while this CTA still multiplies).
constexpr int kSplitDataBytes = (232448 - kSplitBarrierBytes) / 1024 * 1024;
constexpr int kSplitSmemBytes = kSplitDataBytes + kSplitBarrierBytes;
// Half of the shared memory, where that leaves a ring of 88 KB: a longer one gains nothing, and
// less of it starts sooner (E4M3, back to back, all of it and half: 24 x 8960 -> 1536 7.3 and 7.0
// us, 16 x 128 -> 64 2.7 and 2.4; with 80 KB, bf16 24 x 1536 -> 2 x 8960 lost, 13.0 and 13.3).
// Still one CTA per SM, by its registers: with 96 of them, and so two, the same 24 rows took
// 8.0 us.
constexpr int kSplitHalfBytes = (113 * 1024 - kSplitBarrierBytes) / 1024 * 1024;
constexpr int kSplitHalfRing = 88 * 1024;
static_assert(kSplitSmemBytes <= 232448, "split plan exceeds shared memory");

struct SplitBars {
  uint64_t full[kSplitStagesMax];
  uint64_t empty[kSplitStagesMax];
  uint64_t acc_full;
  uint64_t teardown;
  uint32_t tmem_base;
  int abort_flag;
};
static_assert(sizeof(SplitBars) <= kSplitBarrierBytes, "split barrier area");

struct SplitPlan {
  int wr;         // W rows per CTA: 64 or 128 (gated: half of them Wg rows, half Wu rows)
  int tn;         // tokens per CTA: a multiple of 16, at most 128
  int split;      // CTAs per cluster sharing one tile's K
  int group;      // K tiles per stage
  int stages;
  int m_tiles;
  int k_each, k_more, steps, steps_more;
  int own;        // tokens per rank: rank r joins tokens [r * own, (r + 1) * own) of the tile
  int own_mul;    // t / own = t * own_mul >> 16, exact for t * own < 2^16
  int part_off;   // of the partial sums in shared memory
  int bar_off;    // of the barriers, behind them
};

__device__ __forceinline__ void st_cluster_f32(uint32_t addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}

__device__ __forceinline__ uint64_t activate2_any(int act, uint64_t z) {
  switch (act) {
    case kActRelu: return activate2<kActRelu>(z);
    case kActGelu: return activate2<kActGelu>(z);
    case kActGeluTanh: return activate2<kActGeluTanh>(z);
    case kActSilu: return activate2<kActSilu>(z);
    default: return z;
  }
}

template <bool kF8>
__global__ void __launch_bounds__(kSplitThreads, 1)
    linear_split_kernel(const __grid_constant__ CUtensorMap tmap_x,
                        const __grid_constant__ CUtensorMap tmap_w, const SplitPlan p,
                        const int gated, const uint16_t* residual,
                        uint16_t* y, const LinearArgs a) {
  extern __shared__ __align__(1024) uint8_t smem[];
  if ((smem_u32(smem) & 1023u) != 0) {
    if (threadIdx.x == 0) atomicOr(a.err_word, kErrSmemAlign);
    return;  // every CTA of the cluster sees the same layout
  }
  auto* bars = reinterpret_cast<SplitBars*>(smem + p.bar_off);
  int* abort_flag = &bars->abort_flag;
  const int warp = warp_index_uniform();
  const int lane = threadIdx.x & 31;
  // one cluster of `split` CTAs per tile; a rank's K tiles: k_tiles / split, and one more for
  // the first k_tiles % split ranks (the launcher divides, 32-bit and 64-bit divisions here
  // were most of the time before the first copy)
  const int split = p.split, rank = static_cast<int>(cluster_ctarank());
  const int tile = static_cast<int>(cluster_id());
  const int nb = p.m_tiles == 1 ? tile : tile / p.m_tiles, mb = tile - nb * p.m_tiles;
  const int out_rows = gated ? p.wr / 2 : p.wr;  // output columns of y per tile
  const int kt0 = rank * p.k_each + min(rank, p.k_more);
  const int kt1 = kt0 + p.k_each + (rank < p.k_more ? 1 : 0);
  const int steps = rank < p.k_more ? p.steps_more : p.steps;  // stages filled; >= 1 (split <= k_tiles)
  const uint32_t w_bytes = static_cast<uint32_t>(p.wr) * kKB;
  const uint32_t x_bytes = static_cast<uint32_t>(p.tn) * kKB;
  const uint32_t stage_bytes = (w_bytes + x_bytes) * p.group;
  const uint64_t wait_limit = a.wait_limit;
  const uint64_t teardown_limit = wait_limit > kDefaultWaitLimit ? wait_limit : kDefaultWaitLimit;
  uint32_t cols = 32;
  while (static_cast<int>(cols) < p.tn) cols *= 2;

  const int k_step = kF8 ? kKB : kKB / 2;
  const auto fill = [&](int i, int stage) {  // one lane: the copies of step i into its stage
    const int kt = kt0 + i * p.group;
    const int g = min(p.group, kt1 - kt);
    uint8_t* sw = smem + stage * stage_bytes;
    uint64_t* full = &bars->full[stage];
    mbar_arrive_expect_tx(full, (w_bytes + x_bytes) * g);
    for (int j = 0; j < g; ++j) {
      uint8_t* at = sw + j * w_bytes;
      const int k = (kt + j) * k_step;
      if (gated) {  // boxes of wr / 2 rows: Wg, then the same columns' Wu
        tma_load_2d(at, &tmap_w, full, k, nb * out_rows);
        tma_load_2d(at + w_bytes / 2, &tmap_w, full, k, a.n + nb * out_rows);
      } else {
        tma_load_2d(at, &tmap_w, full, k, nb * out_rows);
      }
      tma_load_2d(sw + p.group * w_bytes + j * x_bytes, &tmap_x, full, k, mb * p.tn);
    }
  };

  // The first copies are under way before the rest of the CTA is set up (two steps of them:
  // a copy takes a hundred cycles to issue, and the first stage should not wait for the rest).
  const int ahead = min(min(steps, p.stages), 2);
  if (warp == 0) {
    if (lane < p.stages) {
      mbar_init(&bars->full[lane], 1);
      mbar_init(&bars->empty[lane], 1);
    }
    if (lane == 31) {
      mbar_init(&bars->acc_full, 1);
      mbar_init(&bars->teardown, 1);
      bars->abort_flag = 0;
    }
    fence_barrier_init();
    fence_proxy_async_smem();
    grid_launch_dependents();
    grid_dependency_wait();
    __syncwarp();
    if (elect_one())
      for (int i = 0; i < ahead; ++i) fill(i, i);
    __syncwarp();
  } else if (warp == 1) {
    tmem_alloc(&bars->tmem_base, cols);
    tmem_relinquish();
  }
  grid_dependency_wait();
  __syncwarp();
  if (split > 1) cluster_arrive();  // this CTA runs: the others may send to it
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;
  uint64_t acc_limit = wait_limit;  // on the wait for the accumulator

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    int stage = ahead == p.stages ? 0 : ahead;
    uint32_t phase = ahead == p.stages ? 1u : 0u;
    uint32_t filled = static_cast<uint32_t>(ahead);
    for (int i = ahead; i < steps; ++i) {
      if (!warp_wait_bounded(&bars->empty[stage], phase ^ 1u, wait_limit)) {
        warp_flag(abort_flag, a.err_word, kErrWaitProducer);
        break;
      }
      if (elect_one()) fill(i, stage);
      __syncwarp();
      filled = i + 1;
      if (++stage == p.stages) {
        stage = 0;
        phase ^= 1u;
      }
    }
    // no load may be in flight when the ring is reused or the CTA exits
    for (int s = 0; s < p.stages; ++s) {
      const uint32_t times = filled > static_cast<uint32_t>(s) ? (filled - 1 - s) / p.stages + 1 : 0;
      if (times > 0 && !warp_wait_bounded(&bars->full[s], (times - 1) & 1u, teardown_limit))
        warp_flag(abort_flag, a.err_word, kErrWaitTeardown);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    const uint32_t idesc = instr_desc<kF8>(p.wr, p.tn);
    int stage = 0;
    uint32_t phase = 0;
    int done = 0;  // steps issued
    for (int i = 0; i < steps; ++i) {
      if (!warp_wait_bounded(&bars->full[stage], phase, wait_limit)) {
        warp_flag(abort_flag, a.err_word, kErrWaitMma);
        break;
      }
      tc_fence_after();
      const int g = min(p.group, kt1 - kt0 - i * p.group);
      const uint32_t sw = smem_u32(smem + stage * stage_bytes);
      if (elect_one()) {
        for (int t = 0; t < g; ++t) {
          const uint64_t wdesc = make_smem_desc(sw + t * w_bytes, 16, 1024, 2);
          const uint64_t xdesc = make_smem_desc(sw + p.group * w_bytes + t * x_bytes, 16, 1024, 2);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            mma_one<kF8>(tmem, wdesc + static_cast<uint64_t>(2 * j),
                         xdesc + static_cast<uint64_t>(2 * j), idesc,
                         (i > 0 || t > 0 || j > 0) ? 1u : 0u);
        }
        tc_commit(&bars->empty[stage]);
        if (i == steps - 1) tc_commit(&bars->acc_full);
      }
      __syncwarp();
      ++done;
      if (++stage == p.stages) {
        stage = 0;
        phase ^= 1u;
      }
    }
    // Nothing issued may run on when TMEM and the ring go, whichever warp gives up, and when: the wait
    // for acc_full below, or where that was not committed, one here.
    if (done == steps) {
      acc_limit = teardown_limit;
    } else if (done > 0) {
      if (elect_one()) tc_commit(&bars->teardown);
      __syncwarp();
      if (!warp_wait_bounded(&bars->teardown, 0, teardown_limit))
        warp_flag(abort_flag, a.err_word, kErrWaitTeardown);
    }
  }
  // ------------------------------------------------------------ partial sums to their owners
  // part[(source rank * own + t - owner's first token) * wr + row] of the owner of token t
  float* part = reinterpret_cast<float*>(smem + p.part_off);
  if (!mbar_wait_bounded(&bars->acc_full, 0, acc_limit) &&
      *reinterpret_cast<volatile int*>(abort_flag) == 0)
    flag(abort_flag, a.err_word, kErrWaitEpilogue);
  __syncwarp();
  if (split > 1) cluster_wait();
  tc_fence_after();
  if (warp >= 2) {
    const int quad = warp & 3, half = (warp - 2) >> 2;
    // 128 rows lie in the accumulator's lanes in order, 64 in the first 16 lanes of each quarter
    const int row = p.wr == 128 ? quad * 32 + lane : quad * 16 + lane;
    {
      const uint32_t mine = smem_u32(part) + static_cast<uint32_t>((rank * p.own * p.wr + row) * 4);
      for (int c = half * 16; c < p.tn; c += 32) {
        uint32_t r[16];
        tmem_ld_32x32b_x16(tmem + (static_cast<uint32_t>(quad * 32) << 16) + c, r);
        tmem_ld_wait();
        if (p.wr == 64 && lane >= 16) continue;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int t = c + j, owner = (t * p.own_mul) >> 16;
          const uint32_t at = mine + static_cast<uint32_t>((t - owner * p.own) * p.wr * 4);
          st_cluster_f32(mapa_shared(at, static_cast<uint32_t>(owner)), __uint_as_float(r[j]));
        }
      }
    }
    tc_fence_before();
  }
  __syncwarp();
  if (split > 1) cluster_arrive();

  // ------------------------------------------------------------ join and epilogue
  // This CTA's share of the tile's tokens: a thread keeps four output columns (whose scales and
  // biases it fetches while the cluster's barrier fills) and takes every so many tokens, the
  // ranks' partial sums added in rank order.
  const int first = rank * p.own, count = min(p.own, p.tn - first);  // may be negative
  const int quad_shift = 31 - __clz(out_rows / 4);  // out_rows is a power of two
  const int id = static_cast<int>(threadIdx.x);
  const int row = (id & ((1 << quad_shift) - 1)) * 4, col = nb * out_rows + row;
  const bool in_columns = id < kJoinThreads && col < a.n;
  uint2 bg = make_uint2(0, 0), bu = make_uint2(0, 0);
  float4 sg = make_float4(1.0f, 1.0f, 1.0f, 1.0f), su = sg;
  if (in_columns) {
    if (a.bias != nullptr) {
      bg = *reinterpret_cast<const uint2*>(a.bias + col);
      if (gated) bu = *reinterpret_cast<const uint2*>(a.bias + a.n + col);
    }
    if constexpr (kF8) {
      sg = *reinterpret_cast<const float4*>(a.sw + col);
      if (gated) su = *reinterpret_cast<const float4*>(a.sw + a.n + col);
    }
  }
  __syncwarp();
  if (split > 1)
    cluster_wait();
  else
    __syncthreads();
  const bool good = *reinterpret_cast<volatile int*>(abort_flag) == 0;
  const auto affine = [&](float4 v, float sx, float4 scale, uint2 bias, uint64_t (&z)[2]) {
    z[0] = f2_pack(v.x, v.y);
    z[1] = f2_pack(v.z, v.w);
    if constexpr (kF8) {
      z[0] = f2_mul(f2_mul(z[0], f2_pack(sx, sx)), f2_pack(scale.x, scale.y));
      z[1] = f2_mul(f2_mul(z[1], f2_pack(sx, sx)), f2_pack(scale.z, scale.w));
    }
    z[0] = f2_add(z[0], f2_of_bf16x2(bias.x));
    z[1] = f2_add(z[1], f2_of_bf16x2(bias.y));
  };
  if (good && in_columns) {
    const auto total = [&](int t, int row) {  // the ranks' sums in rank order, loads first
      float4 v[kSplitMax];
      const float* at = part + t * p.wr + row;
#pragma unroll
      for (int q = 0; q < kSplitMax; ++q)
        if (q < split) v[q] = *reinterpret_cast<const float4*>(at + q * p.own * p.wr);
      float4 z = v[0];
#pragma unroll
      for (int q = 1; q < kSplitMax; ++q)
        if (q < split) z.x += v[q].x, z.y += v[q].y, z.z += v[q].z, z.w += v[q].w;
      return z;
    };
    for (int t = id >> quad_shift; t < count; t += kJoinThreads >> quad_shift) {
      const int token = mb * p.tn + first + t;
      if (token >= a.m) break;
      const int64_t dst = static_cast<int64_t>(token) * a.n + col;
      uint2 res = make_uint2(0, 0);
      if (residual != nullptr) res = *reinterpret_cast<const uint2*>(residual + dst);
      const float sx = kF8 ? a.sx[token] : 1.0f;
      uint64_t z[2], u[2];
      affine(total(t, row), sx, sg, bg, z);
      if (gated) affine(total(t, row + out_rows), sx, su, bu, u);
      z[0] = activate2_any(a.act, z[0]);
      z[1] = activate2_any(a.act, z[1]);
#pragma unroll
      for (int j = 0; j < 2; ++j)
        if (gated) z[j] = f2_mul(z[j], u[j]);
      z[0] = f2_add(z[0], f2_of_bf16x2(res.x));
      z[1] = f2_add(z[1], f2_of_bf16x2(res.y));
      *reinterpret_cast<uint2*>(y + dst) = make_uint2(f2_to_bf16x2(z[0]), f2_to_bf16x2(z[1]));
    }
  }
  // nobody sends to this CTA any more; its warps have read TMEM before the barrier above
  __syncwarp();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, cols);
}

// ---------------------------------------------------------------- one or two tokens
// W is one stream of bytes.  Its rows are taken in pairs (gated: column c's Wg and Wu rows),
// every CTA an equal range of them; the CTA's eight warps are groups of `kw`, a group takes
// every (8 / kw)-th pair, and a warp always the same `kw`-th of K, so that its part of x stays
// in its registers.  A warp's parts of its pairs come through a ring of its own by bulk copies
// and are waited for by it alone; only the sums of a block of pairs meet in shared memory (in
// warp order), where one thread per output applies the epilogue.
constexpr int kVecWarps = 8;
constexpr int kVecThreads = 32 * kVecWarps;
constexpr int kVecTokensMax = 2;
constexpr int kVecSlotsMax = 8;
constexpr int kVecGrid = 2;            // CTAs per SM
constexpr int kVecPieces = 256;        // 16-byte pieces of a row that a warp takes at most
constexpr int kVecRing = 11 * 1024;    // of a warp (two CTAs fit an SM), more where two slots need it
constexpr int kVecHead = 1024;         // barriers
constexpr int kVecPart = 2 * kVecThreads * kVecWarps * 4;
constexpr int kVecSmemMax = kVecHead + kVecPart + kVecWarps * 2 * 2 * kVecPieces * 16;

struct VecPlan {
  int k_bytes;
  int kw_log;             // warps that share a row: 1 << kw_log
  int per;                // 16-byte pieces of a row per warp
  int slots, ring_bytes;  // of a warp
  int each, more;         // pairs of rows per CTA, and one more for the first `more`
};

// 16-byte aligned, bytes a multiple of 16
__device__ __forceinline__ void l2_prefetch(const void* p, uint32_t bytes) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"(bytes) : "memory");
}

// 16 bytes of operand -> pairs of fp32: 4 (bf16) or 8 (E4M3)
template <bool kF8>
__device__ __forceinline__ void unpack16(const uint4& v, uint64_t (&f)[kF8 ? 8 : 4]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (kF8) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t h2;
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"(static_cast<uint16_t>(w[i] >> (16 * h))));
        const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&h2));
        f[2 * i + h] = f2_pack(p.x, p.y);
      }
    } else {
      f[i] = f2_of_bf16x2(w[i]);
    }
  }
}

template <bool kF8, int kM, int kS>
__global__ void __launch_bounds__(kVecThreads, 2)
    linear_vector_kernel(const uint8_t* x, const int64_t x_bytes, const uint8_t* w, const VecPlan p,
                         const int gated, const uint16_t* residual, uint16_t* y, const LinearArgs a) {
  extern __shared__ __align__(1024) uint8_t smem[];
  constexpr int kPairs = kF8 ? 8 : 4;
  constexpr int kValues = 2 * kM;                  // sums of a pair of rows
  constexpr int kBlock = kVecThreads / kValues;    // pairs per block
  auto* lost = reinterpret_cast<volatile int*>(smem + kVecWarps * kVecSlotsMax * 8);
  auto* part = reinterpret_cast<float*>(smem + kVecHead);  // [2][kBlock][kw][kValues]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kw = 1 << p.kw_log, groups = kVecWarps >> p.kw_log;
  const int group = warp >> p.kw_log, slice = warp & (kw - 1);
  auto* bar = reinterpret_cast<uint64_t*>(smem) + warp * kVecSlotsMax;
  uint8_t* ring = smem + kVecHead + kVecPart + warp * p.ring_bytes;
  const int unit0 = static_cast<int>(blockIdx.x) * p.each + min(static_cast<int>(blockIdx.x), p.more);
  const int total = p.each + (static_cast<int>(blockIdx.x) < p.more ? 1 : 0);  // pairs of the CTA
  const int piece0 = slice * p.per, len = min(p.per, p.k_bytes / 16 - piece0);  // of this warp, len > 0
  const int mine = total > group ? ((total - 1 - group) >> (3 - p.kw_log)) + 1 : 0;  // pairs of this warp
  const uint32_t row_bytes = static_cast<uint32_t>(len) * 16u, slot_bytes = static_cast<uint32_t>(p.per) * 32u;
  static_assert(kVecWarps == 8, "3 is its logarithm");

  if (lane == 0) {
    for (int i = 0; i < p.slots; ++i) mbar_init(&bar[i], 1);
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  if (threadIdx.x == 0) *lost = 0;
  grid_launch_dependents();
  const auto row_of = [&](int i, int r) {  // the warp's part of its i-th pair's row r
    const int64_t unit = unit0 + group + i * groups;
    const int64_t row = gated ? unit + (r == 0 ? 0 : a.n) : 2 * unit + r;
    return w + row * p.k_bytes + piece0 * 16;
  };
  // While the kernel before still runs: the first slots' bytes towards L2.  Nothing is read, so
  // W may be what that kernel writes.  (One row of 1536 x 8960 E4M3 behind its like: 6.5 -> 6.0
  // us.  The split kernel, whose CTAs take a whole SM, lost by it: 24 rows 10.3 -> 11.3.)
  if (lane < 2 * p.slots && (lane >> 1) < mine) l2_prefetch(row_of(lane >> 1, lane & 1), row_bytes);
  __syncwarp();
  grid_dependency_wait();
  const auto fetch = [&](int i, int slot) {  // lane 0: the warp's i-th pair
    if (i >= mine) return;
    uint8_t* to = ring + slot * slot_bytes;
    mbar_arrive_expect_tx(&bar[slot], 2 * row_bytes);
    bulk_load(to, row_of(i, 0), row_bytes, &bar[slot]);
    bulk_load(to + p.per * 16, row_of(i, 1), row_bytes, &bar[slot]);
  };
  if (lane == 0)
    for (int i = 0; i < p.slots; ++i) fetch(i, i);
  uint4 xr[kM][kS];
#pragma unroll
  for (int t = 0; t < kM; ++t)
#pragma unroll
    for (int i = 0; i < kS; ++i) {
      const int at = lane + 32 * i;
      xr[t][i] = make_uint4(0, 0, 0, 0);
      if (at < len && t < a.m) xr[t][i] = reinterpret_cast<const uint4*>(x + t * x_bytes)[piece0 + at];
    }
  __syncthreads();  // the barriers and the flag are initialised

  const int outs = gated ? 1 : 2;  // outputs of a pair, for each token
  const int id = static_cast<int>(threadIdx.x);
  const int out_pair = gated ? id / kM : id / kValues, out_row = gated ? 0 : id / kM % 2, out_t = id % kM;
  int slot = 0;
  uint32_t phases = 0;  // bit s: parity of slot s
  int i = 0;            // pairs of this warp so far
  for (int base = 0, buf = 0; base < total; base += kBlock, buf ^= 1) {
    // this thread's output of the block; what its epilogue reads is under way meanwhile
    const int unit = base + out_pair;
    const int col = (unit0 + unit) * outs + out_row;
    const bool output = out_pair < kBlock && unit < total && out_t < a.m;
    const int64_t dst = static_cast<int64_t>(out_t) * a.n + col;
    float sx = 1.0f, sg = 1.0f, su = 1.0f, bg = 0.0f, bu = 0.0f, res = 0.0f;
    if (output) {
      const auto bf16 = [](const uint16_t* at) { return __uint_as_float(static_cast<uint32_t>(*at) << 16); };
      if constexpr (kF8) {
        sx = a.sx[out_t];
        sg = a.sw[col];
        if (gated) su = a.sw[a.n + col];
      }
      if (a.bias != nullptr) {
        bg = bf16(a.bias + col);
        if (gated) bu = bf16(a.bias + a.n + col);
      }
      if (residual != nullptr) res = bf16(residual + dst);
    }
    float* sums = part + buf * (kBlock * kVecWarps * kValues);
    for (int u = group; u < kBlock && base + u < total; u += groups, ++i) {
      // As in the streaming norm: a wait that runs out is reported and waited for once more, so
      // that no copy is in flight when the CTA exits.
      const uint32_t parity = (phases >> slot) & 1u;
      if (*lost == 0 && !mbar_wait_bounded(&bar[slot], parity, a.wait_limit)) {
        atomicOr(a.err_word, kErrWaitProducer);
        if (!mbar_wait_bounded(&bar[slot], parity,
                               a.wait_limit > kDefaultWaitLimit ? a.wait_limit : kDefaultWaitLimit))
          *lost = 1;  // later pairs are not waited for; the output is undefined
      }
      phases ^= 1u << slot;
      const uint4* rows = reinterpret_cast<const uint4*>(ring + slot * slot_bytes);
      uint64_t acc[2][kM];
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int t = 0; t < kM; ++t) acc[r][t] = 0;
#pragma unroll
      for (int j = 0; j < kS; ++j) {
        const int at = lane + 32 * j;
        if (at >= len) continue;
        if constexpr (kM * kS * kPairs > 24) {  // unpacked anew for every pair, or it spills
#pragma unroll
          for (int t = 0; t < kM; ++t)
            asm volatile("" : "+r"(xr[t][j].x), "+r"(xr[t][j].y), "+r"(xr[t][j].z), "+r"(xr[t][j].w));
        }
        uint64_t xf[kM][kPairs];
#pragma unroll
        for (int t = 0; t < kM; ++t) unpack16<kF8>(xr[t][j], xf[t]);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          uint64_t wf[kPairs];
          unpack16<kF8>(rows[r * p.per + at], wf);
#pragma unroll
          for (int t = 0; t < kM; ++t)
#pragma unroll
            for (int e = 0; e < kPairs; ++e) acc[r][t] = f2_fma(wf[e], xf[t][e], acc[r][t]);
        }
      }
      __syncwarp();
      if (lane == 0) fetch(i + p.slots, slot);
      if (++slot == p.slots) slot = 0;
      // Sums over the warp: while a lane holds several values, each step exchanges half of them
      // (the upper lanes keep the upper half), so that the last lanes hold one value each.
      float v[kValues];
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int t = 0; t < kM; ++t) {
          float lo, hi;
          f2_split(acc[r][t], lo, hi);
          v[r * kM + t] = lo + hi;
        }
      int index = 0;
#pragma unroll
      for (int o = 16, have = kValues; o > 0; o >>= 1) {
        if (have > 1) {
          have /= 2;
          const bool upper = (lane & o) != 0;
#pragma unroll
          for (int e = 0; e < kValues / 2; ++e) {
            if (e >= have) break;
            const float give = upper ? v[e] : v[e + have];
            const float keep = upper ? v[e + have] : v[e];
            v[e] = keep + __shfl_xor_sync(0xFFFFFFFFu, give, o);
          }
          if (upper) index += have;
        } else {
          v[0] += __shfl_xor_sync(0xFFFFFFFFu, v[0], o);
        }
      }
      if ((lane & (32 / kValues - 1)) == 0) sums[((u << p.kw_log) + slice) * kValues + index] = v[0];
    }
    __syncthreads();  // (the other half of `part` was read before the block's last barrier)
    if (output) {
      float z = 0.0f, u = 0.0f;
      const float* at = sums + (out_pair << p.kw_log) * kValues + out_row * kM + out_t;
      for (int q = 0; q < kw; ++q) z += at[q * kValues];
      if (gated)
        for (int q = 0; q < kw; ++q) u += at[q * kValues + kM];
      if constexpr (kF8) z = z * sx * sg;
      z += bg;
      float unused;
      f2_split(activate2_any(a.act, f2_pack(z, 0.0f)), z, unused);
      if (gated) {
        if constexpr (kF8) u = u * sx * su;
        z *= u + bu;
      }
      y[dst] = __bfloat16_as_ushort(__float2bfloat16_rn(z + res));
    }
  }
}

// ---------------------------------------------------------------- host side
using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                   const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                   const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                   CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// 2-D map over [rows, cols] elements of 1 or 2 bytes, rows `stride_bytes` apart; the box is
// `box_rows` x `box_bytes` (64 or 128), with the swizzle of that width.  Reads outside give zeros.
bool make_map(CUtensorMap* map, const void* base, int64_t rows, int64_t cols, int64_t stride_bytes,
              int elem, int box_rows, int box_bytes = kKB) {
  auto enc = reinterpret_cast<EncodeTiledFn>(tensor_map_encode_fn());
  if (enc == nullptr) return false;
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(stride_bytes)};
  cuuint32_t box[2] = {static_cast<cuuint32_t>(box_bytes / elem), static_cast<cuuint32_t>(box_rows)};
  cuuint32_t estr[2] = {1, 1};
  return enc(map, elem == 2 ? CU_TENSOR_MAP_DATA_TYPE_UINT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8, 2,
             const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             box_bytes == kKB ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <bool kF8, bool kGated, bool kSplitK>
cudaError_t launch_pair(const LinearProblem& l, const LinearArgs& a, cudaStream_t st,
                        const char** why) {
  const int elem = kF8 ? 1 : 2;
  alignas(64) CUtensorMap mx, mw, mr, my;
  std::memset(&mr, 0, sizeof(mr));
  if (!make_map(&mx, l.x, l.m, l.k, l.x_stride * elem, elem, 128) ||
      !make_map(&mw, l.w, kGated ? 2 * l.n : l.n, l.k, l.k * elem, elem, a.bn / 2) ||
      !make_map(&my, l.y, l.m, l.n, l.n * 2, 2, 32, 2 * kChunk) ||
      (l.residual != nullptr && !make_map(&mr, l.residual, l.m, l.n, l.n * 2, 2, 32, 2 * kChunk))) {
    *why = "cuTensorMapEncodeTiled failed";
    return cudaErrorInvalidValue;
  }
  static ContextCache attr_done;
  auto* kernel = linear_pair_kernel<kF8, kGated, kSplitK>;
  if (cudaError_t e = ensure_max_dynamic_smem(attr_done, reinterpret_cast<const void*>(kernel),
                                              kPairSmemBytes))
    return e;
  const int64_t out_cols = kGated ? a.bn / 2 : a.bn;
  const int64_t tiles = ((l.m + kPairTokens - 1) / kPairTokens) * ((l.n + out_cols - 1) / out_cols);
  if (kSplitK)
    return launch_dependent(kernel, static_cast<unsigned>(2 * a.split * tiles), kPairThreads, kPairSmemBytes, st,
                            2 * a.split, mx, mw, mr, my, a);
  int64_t pairs = sm_count() / 2;
  if (pairs > tiles) pairs = tiles;
  return launch_dependent(kernel, static_cast<unsigned>(2 * pairs), kPairThreads, kPairSmemBytes, st, 2, mx, mw,
                          mr, my, a);
}

template <bool kF8>
cudaError_t launch_split(const LinearProblem& l, const LinearArgs& a, const SplitPlan& p,
                         cudaStream_t st, const char** why) {
  const int elem = kF8 ? 1 : 2;
  alignas(64) CUtensorMap mx, mw;
  if (!make_map(&mx, l.x, l.m, l.k, l.x_stride * elem, elem, p.tn) ||
      !make_map(&mw, l.w, l.gated ? 2 * l.n : l.n, l.k, l.k * elem, elem,
                l.gated ? p.wr / 2 : p.wr)) {
    *why = "cuTensorMapEncodeTiled failed";
    return cudaErrorInvalidValue;
  }
  static ContextCache attr_done;
  auto* kernel = linear_split_kernel<kF8>;
  if (cudaError_t e = ensure_max_dynamic_smem(attr_done, reinterpret_cast<const void*>(kernel),
                                              kSplitSmemBytes))
    return e;
  const int64_t out_rows = l.gated ? p.wr / 2 : p.wr;
  const int64_t tiles = ((l.m + p.tn - 1) / p.tn) * ((l.n + out_rows - 1) / out_rows);
  return launch_dependent(kernel, static_cast<unsigned>(tiles * p.split), kSplitThreads, p.bar_off + kSplitBarrierBytes, st,
                          p.split, mx, mw, p, l.gated ? 1 : 0, l.residual, l.y, a);
}

// The vector kernel's plan; false where a row does not fit the warps that may share it.
bool plan_vector(const LinearProblem& l, VecPlan* p, int* grid) {
  const int64_t k_bytes = l.k * (l.fp8 ? 1 : 2), pieces = k_bytes / 16;
  if (pieces > kVecWarps * kVecPieces) return false;
  const int64_t units = l.gated ? l.n : l.n / 2;
  *grid = static_cast<int>(units < kVecGrid * sm_count() ? units : kVecGrid * sm_count());
  p->each = static_cast<int>(units / *grid);
  p->more = static_cast<int>(units % *grid);
  // Warps that share a row: a warp spends about 450 cycles on a pair beside its share of the
  // bytes (the wait, the refill, the sum over the lanes), so many pairs want whole rows and few
  // pairs all eight warps; two slots should fit the ring.
  const int per_slice = (l.fp8 ? 100 : 50) * (l.m == 1 ? 2 : 3) / 2;
  int64_t best = INT64_MAX;
  for (int log = 3; log >= 0; --log) {
    const int64_t per = (pieces + (1 << log) - 1) >> log;
    if (log < 3 && per > kVecRing / 64) break;
    if (log > 0 && (pieces >> log) < 32) continue;  // every warp has a share
    const int64_t turns = (p->each + (p->more > 0 ? 1 : 0) + (kVecWarps >> log) - 1) / (kVecWarps >> log);
    const int64_t cost = turns * (450 + per_slice * ((per + 31) / 32));
    if (cost < best) {
      best = cost;
      p->kw_log = log;
    }
  }
  p->k_bytes = static_cast<int>(k_bytes);
  p->per = static_cast<int>((pieces + (1 << p->kw_log) - 1) >> p->kw_log);
  const int slot_bytes = p->per * 32;
  p->slots = kVecRing / slot_bytes;
  if (p->slots < 2) p->slots = 2;
  if (p->slots > kVecSlotsMax) p->slots = kVecSlotsMax;
  p->ring_bytes = p->slots * slot_bytes;
  return true;
}

template <bool kF8, int kM, int kS>
cudaError_t launch_vector(const LinearProblem& l, const LinearArgs& a, const VecPlan& p, int grid, cudaStream_t st) {
  static ContextCache attr_done;
  auto* kernel = linear_vector_kernel<kF8, kM, kS>;
  if (cudaError_t e = ensure_max_dynamic_smem(attr_done, reinterpret_cast<const void*>(kernel), kVecSmemMax))
    return e;
  return launch_dependent(kernel, static_cast<unsigned>(grid), kVecThreads,
                          kVecHead + kVecPart + kVecWarps * p.ring_bytes, st, 0, static_cast<const uint8_t*>(l.x),
                          l.x_stride * (kF8 ? 1 : 2), static_cast<const uint8_t*>(l.w), p, l.gated ? 1 : 0,
                          l.residual, l.y, a);
}

template <bool kF8, int kM>
cudaError_t launch_vector_by_width(const LinearProblem& l, const LinearArgs& a, const VecPlan& p, int grid,
                                   cudaStream_t st) {
  if (p.per <= 64) return launch_vector<kF8, kM, 2>(l, a, p, grid, st);
  if (p.per <= 96) return launch_vector<kF8, kM, 3>(l, a, p, grid, st);
  if (p.per <= 128) return launch_vector<kF8, kM, 4>(l, a, p, grid, st);
  if (p.per <= 160) return launch_vector<kF8, kM, 5>(l, a, p, grid, st);
  if (p.per <= 192) return launch_vector<kF8, kM, 6>(l, a, p, grid, st);
  return launch_vector<kF8, kM, kVecPieces / 32>(l, a, p, grid, st);
}

template <bool kF8>
cudaError_t launch_vector_by_tokens(const LinearProblem& l, const LinearArgs& a, const VecPlan& p, int grid,
                                    cudaStream_t st) {
  return l.m == 1 ? launch_vector_by_width<kF8, 1>(l, a, p, grid, st)
                  : launch_vector_by_width<kF8, 2>(l, a, p, grid, st);
}

// How many clusters of `split` of the split kernel's CTAs run at a time: a cluster stays inside
// a GPC, and on a B200 sizes 3 to 8 leave up to a fifth of the SMs unused (74 pairs, 45 triples,
// 33 fours, 26 fives, 22 sixes, 15 sevens and eights).  Asked once per device and size.
template <bool kF8>
int resident_clusters(int split) {
  static std::atomic<int> known[64][kSplitMax + 1];
  if (split == 1) return sm_count();
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return sm_count() / split;
  int n = known[dev][split].load(std::memory_order_relaxed);
  if (n == 0) {
    static ContextCache attr_done;
    auto* kernel = linear_split_kernel<kF8>;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(split * sm_count()));
    cfg.blockDim = dim3(kSplitThreads);
    cfg.dynamicSmemBytes = kSplitSmemBytes;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(split);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (ensure_max_dynamic_smem(attr_done, reinterpret_cast<const void*>(kernel), kSplitSmemBytes) !=
            cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n <= 0) {
      cudaGetLastError();  // the estimate below stands in
      n = sm_count() / split;
    }
    known[dev][split].store(n, std::memory_order_relaxed);
  }
  return n;
}

// Both planners estimate cycles per SM from measured rates and take the cheapest tile.
//
// Split: a K tile costs its four MMAs, or its bytes: W at an SM's share of HBM (24 bytes a
// cycle when all of them read, up to 40 when fewer do), x from L2.  An MMA takes its W rows from
// shared memory at 32 bytes a cycle: 128 of them about 137 cycles whatever the tokens up to 128,
// 64 of them half of that up to 32 tokens and more beyond (24 x 1536 -> 8960: 8.1 us by 64 rows
// and 9.9 by 128 in bf16, 6.2 and 7.6 in E4M3; with 48 tokens 12.6 and 9.8, 9.3 and 8.1).  Setup,
// drain and output take about 5200 cycles, sending and joining the partial sums 0.35 a sum and,
// between CTAs, 1200 more (128 x 400 -> 1000 in bf16: 6.3 us on seven CTAs a tile of 128 rows,
// 4.5 on four of 64).
template <bool kF8>
SplitPlan plan_split(const LinearProblem& l, int k_tiles, double* cost) {
  SplitPlan best = {};
  *cost = 1e30;
  const int64_t wn = l.gated ? 2 * l.n : l.n;
  for (int wr = 64; wr <= 128; wr *= 2) {
    const int64_t n_tiles = (wn + wr - 1) / wr;
    int last_tn = 0;
    for (int tn_max = 64; tn_max <= 128; tn_max *= 2) {
      const int64_t m_tiles = (l.m + tn_max - 1) / tn_max;
      const int tn = static_cast<int>(((l.m + m_tiles - 1) / m_tiles + 15) / 16 * 16);
      if (tn == last_tn) continue;
      last_tn = tn;
      const double mma = wr == 128 ? 550.0 : tn <= 32 ? 290.0 : 470.0 + 2.0 * tn;
      for (int split = 1; split <= kSplitMax && split <= k_tiles; ++split) {
        const int64_t clusters = resident_clusters<kF8>(split);
        const int64_t waves = (n_tiles * m_tiles + clusters - 1) / clusters;
        const double share = 24.0 * sm_count() / static_cast<double>(n_tiles * m_tiles * split);  // of HBM
        const double bytes = wr * kKB / (share < 24.0 ? 24.0 : share > 40.0 ? 40.0 : share) + tn * kKB / 64.0;
        const double c = static_cast<double>(waves) *
                         ((k_tiles + split - 1) / split * (mma > bytes ? mma : bytes) + 5200.0 +
                          (split > 1 ? 1200.0 : 0.0) + 0.35 * wr * tn);
        if (c < *cost) {
          *cost = c;
          best.wr = wr;
          best.tn = tn;
          best.split = split;
        }
      }
    }
  }
  const int tile_bytes = (best.wr + best.tn) * kKB;
  int group = 24576 / tile_bytes;
  group = group < 1 ? 1 : group;
  best.group = group;
  best.own = (best.tn + best.split - 1) / best.split;
  best.own_mul = (65536 + best.own - 1) / best.own;
  const int part_bytes = best.split * best.own * best.wr * 4;
  const int stage_bytes = tile_bytes * group;
  const bool half = (kSplitHalfBytes - part_bytes) / stage_bytes * stage_bytes >= kSplitHalfRing;
  const int budget = half ? kSplitHalfBytes : kSplitDataBytes;
  best.stages = (budget - part_bytes) / stage_bytes;
  if (best.stages > kSplitStagesMax) best.stages = kSplitStagesMax;
  best.part_off = best.stages * stage_bytes;
  best.bar_off = (best.part_off + part_bytes + 1023) / 1024 * 1024;
  best.m_tiles = static_cast<int>((l.m + best.tn - 1) / best.tn);
  best.k_each = k_tiles / best.split;
  best.k_more = k_tiles % best.split;
  best.steps = (best.k_each + group - 1) / group;
  best.steps_more = (best.k_each + group) / group;
  return best;
}

// Pair: a K tile of a 256 x bn tile takes time in proportion to bn + 205 (7680 x 1536 x 8960
// timed at bn 64 to 256: 0.21, 0.26, 0.29, 0.36 us), so narrower tiles pay only where they
// fill a round of the persistent grid better, and splitting K only where the tiles leave most
// of it idle (1024 x 1536 x 8960: 37 us unsplit).
struct PairPlan {
  int bn, split;
};

template <bool kF8>
PairPlan plan_pair(const LinearProblem& l, int k_tiles, double* cost) {
  const int64_t mb = (l.m + kPairTokens - 1) / kPairTokens;
  PairPlan best = {256, 1};
  *cost = 1e30;
  for (int split = 1; split <= kSplitMax / 2 && split <= k_tiles; ++split) {
    // clusters of either kernel fill an SM per CTA, so the same number of them fits
    const int64_t at_once = split == 1 ? sm_count() / 2 : resident_clusters<kF8>(2 * split);
    for (int bn = 256; bn >= 128; bn -= l.gated ? 64 : 32) {
      const int64_t out_cols = l.gated ? bn / 2 : bn;
      const int64_t tiles = mb * ((l.n + out_cols - 1) / out_cols);
      const int64_t rounds = (tiles + at_once - 1) / at_once;
      const double c = static_cast<double>(rounds) * ((k_tiles + split - 1) / split) * (bn + 205) * 1.5 + 9000.0 +
                       (split > 1 ? static_cast<double>(rounds) * 8000.0 : 0.0);
      if (c < *cost) {
        *cost = c;
        best.bn = bn;
        best.split = split;
      }
    }
  }
  return best;
}

template <bool kF8>
cudaError_t launch_pair_by_plan(const LinearProblem& l, const LinearArgs& a, cudaStream_t st, const char** why) {
  if (a.split > 1)
    return l.gated ? launch_pair<kF8, true, true>(l, a, st, why) : launch_pair<kF8, false, true>(l, a, st, why);
  return l.gated ? launch_pair<kF8, true, false>(l, a, st, why) : launch_pair<kF8, false, false>(l, a, st, why);
}

}  // namespace

static std::atomic<int> g_linear_mode{0};
void set_linear_kernel_mode(int mode) { g_linear_mode.store(mode, std::memory_order_relaxed); }
int linear_kernel_mode() { return g_linear_mode.load(std::memory_order_relaxed); }

cudaError_t launch_linear(const LinearProblem& l, uint64_t wait_limit, cudaStream_t st,
                          const char** why) {
  const char* unused = nullptr;
  if (why == nullptr) why = &unused;
  LinearArgs a = {};
  a.sx = l.sx;
  a.sw = l.sw;
  a.bias = l.bias;
  a.m = static_cast<int>(l.m);
  a.n = static_cast<int>(l.n);
  const int per = l.fp8 ? kKB : kKB / 2;
  a.k_tiles = static_cast<int>((l.k + per - 1) / per);
  a.act = l.act;
  a.residual = l.residual != nullptr ? 1 : 0;
  a.wait_limit = wait_limit;
  a.err_word = error_word_ptr();
  if (a.err_word == nullptr) return cudaErrorInvalidSymbol;
  const int mode = linear_kernel_mode();
  VecPlan v;
  int grid;
  if (mode == 0 && l.m <= kVecTokensMax && plan_vector(l, &v, &grid))
    return l.fp8 ? launch_vector_by_tokens<true>(l, a, v, grid, st) : launch_vector_by_tokens<false>(l, a, v, grid, st);
  double split_cost, pair_cost;
  const SplitPlan p = l.fp8 ? plan_split<true>(l, a.k_tiles, &split_cost)
                            : plan_split<false>(l, a.k_tiles, &split_cost);
  const PairPlan pp = l.fp8 ? plan_pair<true>(l, a.k_tiles, &pair_cost) : plan_pair<false>(l, a.k_tiles, &pair_cost);
  a.bn = pp.bn;
  a.split = pp.split;
  a.k_each = a.k_tiles / pp.split;
  a.k_more = a.k_tiles % pp.split;
  if (mode == 1 || (mode == 0 && split_cost < pair_cost))
    return l.fp8 ? launch_split<true>(l, a, p, st, why) : launch_split<false>(l, a, p, st, why);
  return l.fp8 ? launch_pair_by_plan<true>(l, a, st, why) : launch_pair_by_plan<false>(l, a, st, why);
}

}  // namespace fvq
