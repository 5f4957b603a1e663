// fvq_norm.cu -- root-mean-square norm with the residual's addition, in bf16 or E4M3.
//
//   s = x + r                                   fp32; r bf16 or fp32 (optional)
//   v = s * w * rsqrt(mean(s^2) + eps)          fp32; w bf16 (optional)
//   r_out = s in r's type,  y = bf16(v)         and / or
//   scale = max(max|v| / 448, 1e-12),  q = e4m3(s * w * (rsqrt(..) / scale))
//
// Everything up to the outputs is fp32 in registers; each output is rounded once.  q multiplies
// by one factor per row instead of dividing: three roundings of 2^-24 ahead of E4M3's 2^-4, a
// third of the instructions.  A NaN in a row makes the row NaN, an infinity gives what the
// formulas give (0 for the finite values, NaN for the infinite ones).
//
// HBM-bound: x and r are read once, every output is written once; the row stays in registers
// between the two reductions (sum of squares, then max |v| for E4M3).  Three forms:
//   * rows of at most 512 values: a warp or a part of one, several rows a group when they are
//     short and there are many, so that their loads overlap (65317 rows of 271: 26.6 us, 48
//     streamed; 20000 of 768: 31 us, 20.6 streamed);
//   * few rows: a CTA per row with 8 or 16 values a thread, the shortest chain for one token;
//   * many rows: persistent CTAs whose warps stream rows through rings in shared memory
//     filled by bulk copies (rms_norm_stream_kernel), so that loads stay in flight while
//     earlier rows are reduced and written.  A row that starts or ends off 16 bytes is
//     fetched as the 16-byte aligned window around it, and where rows lie end to end its
//     elements are taken in the pairs that are 4-byte aligned and its outputs leave through
//     the row's buffer, by bulk copies (kVec = 2).
// In the first two forms, and with other strides, such rows take element-wise accesses
// (kVec = 1): neighbouring lanes read neighbouring elements, so the sectors fetched are the same.
//
// Measured on a B200, launches back to back in a CUDA graph over operands larger than L2 (a copy
// moves 6.5 TB/s): one row of 1536 in E4M3 1.9 us; 15360 x 1536 with a bf16 residual to E4M3
// 27 us (6.1 TB/s); 92160 rows of 128 8.9 us (5.3 TB/s, 1.7 us of it start and end); 4099 x 2048
// with an fp32 residual 17.7 us (5.7 TB/s), 4099 x 2047 21.3 us (bounds, shifts and copies of
// the ragged ends are instructions that the aligned form does not have).  More warps a row than
// the rings need cost time (15360 x 1536 to bf16: one warp 14.9 us, two 18.8, four 25.0).
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "fvq_internal.h"
#include "fvq_launch.h"
#include "fvq_ptx.cuh"

namespace fvq {

namespace {

constexpr int kNormThreads = 256;      // of the sub-warp form
constexpr int kNormMaxThreads = 1024;  // of the CTA form
constexpr int kNormMaxD = 16384;

// max with a NaN of either side kept
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Row elements are held as pairs (f2_*); a thread's share of a row is kPairs of them.  kVec 8:
// pairs 4i .. 4i+3 are the eight adjacent elements of its i-th 16-byte vector; kVec 1: pair i
// holds its elements 2i and 2i + 1, as many elements apart as the row has lanes; kVec 2 (rows
// in shared memory, in the streaming form): pair i is two adjacent elements whose place is
// 4-byte aligned, so that the first pair of a row may start one element before it, and the
// last one end one after it; what lies there is the slot's slack.  `at(i)` is the index of
// vector (kVec 8), pair (kVec 2) or element (kVec 1) i; elements outside [0, d) are zero, and
// not stored but to the slack.
// Where a thread's vectors (kVec 8), pairs (2) or elements (1) lie in a row.  kVec 2: pairs
// [1, full) of every lane lie inside the row, so only the first and the last ones need bounds
// (with bounds on every pair they were two thirds of the instructions).
template <int kVec, int kLanes = 0>
struct Place {
  int lane, lanes, odd, full;
  __device__ __forceinline__ int operator()(int i) const {
    return (lane + i * (kLanes == 0 ? lanes : kLanes)) * kVec - (kVec == 2 ? odd : 0);
  }
  __device__ __forceinline__ bool inner(int i) const { return i > 0 && i < full; }
};

template <int kPairs, int kVec, class At>
__device__ __forceinline__ void load_bf16(uint32_t (&w)[kPairs], const uint16_t* p, int d, At at) {
  if constexpr (kVec == 8) {
#pragma unroll
    for (int i = 0; i < kPairs / 4; ++i) {
      uint4 v = make_uint4(0, 0, 0, 0);
      if (at(i) < d) v = *reinterpret_cast<const uint4*>(p + at(i));
      w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
    }
  } else if constexpr (kVec == 2) {
    // from a slot in shared memory, whose slack covers the elements on either side of the row;
    // the caller drops them (mask_pairs)
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      w[i] = 0;
      if (at.inner(i) || at(i) < d) w[i] = *reinterpret_cast<const uint32_t*>(p + at(i));
    }
  } else {
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      const uint32_t lo = at(2 * i) < d ? p[at(2 * i)] : 0u;
      const uint32_t hi = at(2 * i + 1) < d ? p[at(2 * i + 1)] : 0u;
      w[i] = lo | (hi << 16);
    }
  }
}

// The weight's share: global memory of any alignment.
template <int kPairs, int kVec, class At>
__device__ __forceinline__ void load_weight(uint32_t (&w)[kPairs], const uint16_t* p, int d, At at) {
  if constexpr (kVec == 2) {
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      const uint32_t lo = at(i) >= 0 && at(i) < d ? p[at(i)] : 0u;
      const uint32_t hi = at(i) + 1 < d ? p[at(i) + 1] : 0u;
      w[i] = lo | (hi << 16);
    }
  } else {
    load_bf16<kPairs, kVec>(w, p, d, at);
  }
}

// s += the fp32 elements at p
template <int kPairs, int kVec, class At>
__device__ __forceinline__ void add_f32(uint64_t (&s)[kPairs], const float* p, int d, At at) {
  if constexpr (kVec == 8) {
#pragma unroll
    for (int i = 0; i < kPairs / 4; ++i) {
      if (at(i) < d) {
        const float4 a = *reinterpret_cast<const float4*>(p + at(i));
        const float4 b = *reinterpret_cast<const float4*>(p + at(i) + 4);
        s[4 * i] = f2_add(s[4 * i], f2_pack(a.x, a.y));
        s[4 * i + 1] = f2_add(s[4 * i + 1], f2_pack(a.z, a.w));
        s[4 * i + 2] = f2_add(s[4 * i + 2], f2_pack(b.x, b.y));
        s[4 * i + 3] = f2_add(s[4 * i + 3], f2_pack(b.z, b.w));
      }
    }
  } else if constexpr (kVec == 2) {
#pragma unroll
    for (int i = 0; i < kPairs; ++i)
      if (at.inner(i) || at(i) < d) s[i] = f2_add(s[i], *reinterpret_cast<const uint64_t*>(p + at(i)));
  } else {
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      const float lo = at(2 * i) < d ? p[at(2 * i)] : 0.0f;
      const float hi = at(2 * i + 1) < d ? p[at(2 * i + 1)] : 0.0f;
      s[i] = f2_add(s[i], f2_pack(lo, hi));
    }
  }
}

template <int kPairs, int kVec, class At>
__device__ __forceinline__ void store_f32(float* p, const uint64_t (&s)[kPairs], int d, At at) {
  if constexpr (kVec == 8) {
#pragma unroll
    for (int i = 0; i < kPairs / 4; ++i) {
      if (at(i) < d) {
        float f[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) f2_split(s[4 * i + e], f[2 * e], f[2 * e + 1]);
        reinterpret_cast<float4*>(p + at(i))[0] = make_float4(f[0], f[1], f[2], f[3]);
        reinterpret_cast<float4*>(p + at(i))[1] = make_float4(f[4], f[5], f[6], f[7]);
      }
    }
  } else if constexpr (kVec == 2) {
#pragma unroll
    for (int i = 0; i < kPairs; ++i)
      if (at.inner(i) || at(i) < d) *reinterpret_cast<uint64_t*>(p + at(i)) = s[i];
  } else {
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      float lo, hi;
      f2_split(s[i], lo, hi);
      if (at(2 * i) < d) p[at(2 * i)] = lo;
      if (at(2 * i + 1) < d) p[at(2 * i + 1)] = hi;
    }
  }
}

// bf16(s * f)
template <int kPairs, int kVec, class At>
__device__ __forceinline__ void store_bf16(uint16_t* p, const uint64_t (&s)[kPairs], uint64_t f, int d,
                                           At at) {
  if constexpr (kVec == 8) {
#pragma unroll
    for (int i = 0; i < kPairs / 4; ++i)
      if (at(i) < d)
        *reinterpret_cast<uint4*>(p + at(i)) =
            make_uint4(f2_to_bf16x2(f2_mul(s[4 * i], f)), f2_to_bf16x2(f2_mul(s[4 * i + 1], f)),
                       f2_to_bf16x2(f2_mul(s[4 * i + 2], f)), f2_to_bf16x2(f2_mul(s[4 * i + 3], f)));
  } else if constexpr (kVec == 2) {
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      const uint32_t w = f2_to_bf16x2(f2_mul(s[i], f));
      if (at.inner(i) || at(i) < d) *reinterpret_cast<uint32_t*>(p + at(i)) = w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      const uint32_t w = f2_to_bf16x2(f2_mul(s[i], f));
      if (at(2 * i) < d) p[at(2 * i)] = static_cast<uint16_t>(w);
      if (at(2 * i + 1) < d) p[at(2 * i + 1)] = static_cast<uint16_t>(w >> 16);
    }
  }
}

// e4m3(s * f)
template <int kPairs, int kVec, class At>
__device__ __forceinline__ void store_e4m3(uint8_t* p, const uint64_t (&s)[kPairs], uint64_t f, int d,
                                           At at) {
  if constexpr (kVec == 8) {
#pragma unroll
    for (int i = 0; i < kPairs / 4; ++i)
      if (at(i) < d)
        *reinterpret_cast<uint2*>(p + at(i)) =
            make_uint2(f2_to_e4m3x2(f2_mul(s[4 * i], f)) | (f2_to_e4m3x2(f2_mul(s[4 * i + 1], f)) << 16),
                       f2_to_e4m3x2(f2_mul(s[4 * i + 2], f)) | (f2_to_e4m3x2(f2_mul(s[4 * i + 3], f)) << 16));
  } else if constexpr (kVec == 2) {
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      const uint32_t w = f2_to_e4m3x2(f2_mul(s[i], f));
      if (at.inner(i) || at(i) < d) *reinterpret_cast<uint16_t*>(p + at(i)) = static_cast<uint16_t>(w);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      const uint32_t w = f2_to_e4m3x2(f2_mul(s[i], f));
      if (at(2 * i) < d) p[at(2 * i)] = static_cast<uint8_t>(w);
      if (at(2 * i + 1) < d) p[at(2 * i + 1)] = static_cast<uint8_t>(w >> 8);
    }
  }
}

// s = x + r, and r_out = s; p at the row's residual (global or shared memory).
template <int kPairs, int kVec, class At>
__device__ __forceinline__ void add_residual(uint64_t (&s)[kPairs], const void* p, bool f32, void* out,
                                             bool store, int d, At at) {
  if (f32) {
    add_f32<kPairs, kVec>(s, static_cast<const float*>(p), d, at);
    if (store) store_f32<kPairs, kVec>(static_cast<float*>(out), s, d, at);
  } else {
    uint32_t w[kPairs];
    load_bf16<kPairs, kVec>(w, static_cast<const uint16_t*>(p), d, at);
#pragma unroll
    for (int i = 0; i < kPairs; ++i) s[i] = f2_add(s[i], f2_of_bf16x2(w[i]));
    if (store)
      store_bf16<kPairs, kVec>(static_cast<uint16_t*>(out), s, f2_pack(1.0f, 1.0f), d, at);
  }
}

// kVec 2: zeros in place of the elements outside the row.
template <int kPairs, class At>
__device__ __forceinline__ void mask_pairs(uint64_t (&s)[kPairs], int d, At at) {
#pragma unroll
  for (int i = 0; i < kPairs; ++i) {
    if (at.inner(i)) continue;
    if (at(i) < 0 || at(i) >= d) s[i] &= 0xFFFFFFFF00000000ull;
    if (at(i) + 1 >= d) s[i] &= 0x00000000FFFFFFFFull;
  }
}

template <int kPairs>
__device__ __forceinline__ float sum_squares(const uint64_t (&s)[kPairs]) {
  uint64_t q[4] = {0, 0, 0, 0};  // four chains: one of 24 dependent steps is longer than the row's loads
#pragma unroll
  for (int i = 0; i < kPairs; ++i) q[i % 4] = f2_fma(s[i], s[i], q[i % 4]);
  float lo, hi;
  f2_split(f2_add(f2_add(q[0], q[1]), f2_add(q[2], q[3])), lo, hi);
  return lo + hi;
}

// s *= w (when there is a weight)
template <int kPairs>
__device__ __forceinline__ void apply_weight(uint64_t (&s)[kPairs], const uint32_t (&w)[kPairs]) {
#pragma unroll
  for (int i = 0; i < kPairs; ++i) s[i] = f2_mul(s[i], f2_of_bf16x2(w[i]));
}

template <int kPairs>
__device__ __forceinline__ float max_abs(const uint64_t (&s)[kPairs]) {
  float m[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int i = 0; i < kPairs; ++i) {
    float lo, hi;
    f2_split(s[i], lo, hi);
    m[2 * (i % 2)] = max_nan(m[2 * (i % 2)], fabsf(lo));
    m[2 * (i % 2) + 1] = max_nan(m[2 * (i % 2) + 1], fabsf(hi));
  }
  return max_nan(max_nan(m[0], m[1]), max_nan(m[2], m[3]));
}

// max(m / 448, 1e-12); NaN stays NaN
__device__ __forceinline__ float scale448(float m) {
  const float by448 = __fdiv_rn(m, 448.0f);
  return by448 < 1e-12f ? 1e-12f : by448;
}

// Sum / maximum over the threads of a row: kLanes (8, 16 or 32) lanes of a warp, or with
// kLanes = 0 the whole CTA.
template <int kLanes, class Op>
__device__ __forceinline__ float row_reduce(float v, float* smem, Op op) {
  constexpr int kWidth = kLanes == 0 ? 32 : kLanes;
#pragma unroll
  for (int o = kWidth / 2; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
  if constexpr (kLanes == 0) {
    const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
    if (warps > 1) {
      if (lane == 0) smem[threadIdx.x >> 5] = v;
      __syncthreads();
      v = lane < warps ? smem[lane] : 0.0f;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
    }
  }
  return v;
}

__device__ __forceinline__ const uint16_t* x_row(const NormArgs& a, int64_t row) {
  if (a.inner == 1) return a.x + row * a.outer_stride;
  // row / inner, exact below 2^31 (Granlund and Montgomery, "Division by invariant integers using
  // multiplication", 1994): (n + umulhi(n, m)) >> l with m, l of the launcher
  const uint32_t n = static_cast<uint32_t>(row);
  const uint32_t outer = (n + __umulhi(n, a.inner_mul)) >> a.inner_shift;
  const uint32_t in = n - outer * static_cast<uint32_t>(a.inner);
  return a.x + outer * a.outer_stride + in * a.inner_stride;
}

// ---------------------------------------------------------------- short rows, few rows
// kPer: elements per thread.  kLanes 0: one CTA per row; otherwise kLanes lanes per row and
// kRows rows per group, whose loads overlap.  A row has at most (threads of the row) * kPer
// elements.
template <int kLanes, int kRows, int kPer, int kVec>
__global__ void __launch_bounds__(kLanes == 0 ? kNormMaxThreads : kNormThreads)
    rms_norm_kernel(const NormArgs a) {
  static_assert(kLanes != 0 || kRows == 1, "one row per CTA");
  grid_launch_dependents();
  grid_dependency_wait();
  __shared__ float sum_smem[32];
  __shared__ float max_smem[32];
  constexpr int kPairs = kPer / 2;
  const int lanes = kLanes == 0 ? static_cast<int>(blockDim.x) : kLanes;
  const int lane = kLanes == 0 ? static_cast<int>(threadIdx.x) : static_cast<int>(threadIdx.x) % lanes;
  const int d = a.d;
  const Place<kVec> at = {lane, lanes, 0, 0};
  // kRows rows, `step` apart, so that neighbouring groups read neighbouring rows
  const int64_t step = kLanes == 0 ? 1 : kNormThreads / lanes;
  const int64_t first = kLanes == 0 ? static_cast<int64_t>(blockIdx.x)
                                    : blockIdx.x * step * kRows + static_cast<int>(threadIdx.x) / lanes;
  uint32_t xw[kRows][kPairs];
#pragma unroll
  for (int k = 0; k < kRows; ++k)  // a row past the last one repeats it: the warp's shuffles stay whole
    load_bf16<kPairs, kVec>(xw[k], x_row(a, min(first + k * step, a.rows - 1)), d, at);
  uint32_t w[kPairs];
  if (a.weight != nullptr) load_weight<kPairs, kVec>(w, a.weight, d, at);
#pragma unroll
  for (int k = 0; k < kRows; ++k) {
    const bool live = first + k * step < a.rows;
    const int64_t row = min(first + k * step, a.rows - 1);
    const int64_t base = row * d;
    uint64_t s[kPairs];
#pragma unroll
    for (int i = 0; i < kPairs; ++i) s[i] = f2_of_bf16x2(xw[k][i]);
    if (a.residual != nullptr) {
      const int64_t bytes = base * (a.residual_f32 ? 4 : 2);
      add_residual<kPairs, kVec>(s, static_cast<const uint8_t*>(a.residual) + bytes, a.residual_f32,
                                 static_cast<uint8_t*>(a.residual_out) + bytes, live, d, at);
    }
    const float sq = row_reduce<kLanes>(sum_squares(s), sum_smem, [](float p, float q) { return p + q; });
    const float rstd = rsqrtf(sq / static_cast<float>(d) + a.eps);
    if (a.weight != nullptr) apply_weight(s, w);
    if (a.y != nullptr && live) store_bf16<kPairs, kVec>(a.y + base, s, f2_pack(rstd, rstd), d, at);
    if (a.q != nullptr) {
      const float m = row_reduce<kLanes>(max_abs(s), max_smem, [](float p, float q) { return max_nan(p, q); });
      const float scale = scale448(m * rstd), f = rstd * __frcp_rn(scale);
      if (!live) continue;
      if (lane == 0) a.scale[row] = scale;
      store_e4m3<kPairs, kVec>(a.q + base, s, f2_pack(f, f), d, at);
    }
  }
}

// ---------------------------------------------------------------- many long rows
// One CTA of 16 warps per SM.  A group of `kGroup` warps walks rows group by group over the
// grid; each group owns a ring of `slots` row buffers (x's row, then the residual's), one
// mbarrier each.  A slot is refilled as soon as the group holds its row in registers.  (No
// grid_launch_dependents here: with the next kernel let in early, 15360 rows of 1536 took
// 29.5 us instead of 28.2.)
constexpr int kStreamWarps = 16;
constexpr int kStreamThreads = 32 * kStreamWarps;
constexpr int kStreamSmem = 216 * 1024;
constexpr int kStreamSlotsMax = 8;
constexpr int kStreamHead = 2048;  // barriers and the reductions' partials

struct StreamPlan {
  int x_bytes;     // bytes of x's window in a slot (a multiple of 16)
  int slot_bytes;
  int slots;
};

// What a bulk copy fetches of a row: the 16-byte pieces around it, less those that are not
// wholly inside the tensor (first and last row).  Both ends of the tensor are given rounded
// inwards.
struct Piece {
  const uint8_t* lo;  // first byte fetched
  uint32_t bytes;
  uint32_t off;       // of the row in its slot
  uint32_t skip;      // of the fetched bytes in the slot
};

__device__ __forceinline__ Piece piece_of(const uint8_t* row, uint32_t bytes, const uint8_t* begin16,
                                          const uint8_t* end16) {
  Piece p;
  const uintptr_t at = reinterpret_cast<uintptr_t>(row);
  p.off = static_cast<uint32_t>(at & 15u);
  const uint8_t* first = row - p.off;
  const uint8_t* last = first + ((p.off + bytes + 15u) & ~15u);
  p.lo = first < begin16 ? begin16 : first;
  p.skip = static_cast<uint32_t>(p.lo - first);
  p.bytes = static_cast<uint32_t>((last > end16 ? end16 : last) - p.lo);
  return p;
}

// The elements of a row that its piece leaves out (at most 15 bytes at either end), by the
// first lanes.  Returns whether there were any.
template <class T>
__device__ __forceinline__ bool patch_row(const uint8_t* row, uint8_t* slot_row, uint32_t bytes, const Piece& p,
                                          int lane) {
  const uint32_t head = p.lo > row ? static_cast<uint32_t>(p.lo - row) : 0u;
  const uint32_t got = static_cast<uint32_t>(p.lo - row) + p.bytes;  // modulo 2^32: the end of the piece
  const uint32_t tail = got < bytes ? bytes - got : 0u;
  if (head == 0 && tail == 0) return false;
  const uint32_t at = lane * static_cast<uint32_t>(sizeof(T));
  if (at < head) *reinterpret_cast<T*>(slot_row + at) = *reinterpret_cast<const T*>(row + at);
  if (at < tail) *reinterpret_cast<T*>(slot_row + got + at) = *reinterpret_cast<const T*>(row + got + at);
  return true;
}

template <int kGroup>
__device__ __forceinline__ void group_sync(int group) {
  if constexpr (kGroup == 1)
    __syncwarp();
  else
    asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(32 * kGroup) : "memory");
}

template <int kGroup, class Op>
__device__ __forceinline__ float group_reduce(float v, float* smem, int group, int warp_in_group, Op op) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
  if constexpr (kGroup > 1) {
    if ((threadIdx.x & 31) == 0) smem[warp_in_group] = v;
    group_sync<kGroup>(group);
    v = smem[0];
#pragma unroll
    for (int k = 1; k < kGroup; ++k) v = op(v, smem[k]);
  }
  return v;
}

// A row of `bytes` (elements of `elem`) from shared to global memory, both at the same offset
// in 16 bytes: the whole 16-byte pieces by one bulk copy (lane 0's; committed by the caller),
// the elements before and after them by the first lanes.
__device__ __forceinline__ void flush_row(uint8_t* to, const uint8_t* from, int bytes, int elem, int lane) {
  const int head = min(bytes, static_cast<int>((16u - (reinterpret_cast<uintptr_t>(to) & 15u)) & 15u));
  const int body = (bytes - head) & ~15;
  if (lane == 0 && body > 0)
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(to + head),
                 "r"(smem_u32(from + head)), "r"(body)
                 : "memory");
  const int tail = bytes - head - body;  // head and tail hold at most 15 elements each
  const int at = lane < 16 ? lane * elem : head + body + (lane - 16) * elem;
  if (lane < 32 && (lane < 16 ? lane * elem < head : (lane - 16) * elem < tail)) {
    if (elem == 4)
      *reinterpret_cast<uint32_t*>(to + at) = *reinterpret_cast<const uint32_t*>(from + at);
    else if (elem == 2)
      *reinterpret_cast<uint16_t*>(to + at) = *reinterpret_cast<const uint16_t*>(from + at);
    else
      to[at] = from[at];
  }
}

template <int kGroup, int kPer, int kVec>
__global__ void __launch_bounds__(kStreamThreads, 1)
    rms_norm_stream_kernel(const NormArgs a, const StreamPlan p, const uint64_t wait_limit,
                           uint32_t* err_word) {
  extern __shared__ __align__(128) uint8_t smem[];
  constexpr int kGroups = kStreamWarps / kGroup;
  constexpr int kLanes = 32 * kGroup;
  constexpr int kPairs = kPer / 2;
  auto* bars = reinterpret_cast<uint64_t*>(smem);                          // [groups][slots]
  auto* sums = reinterpret_cast<float*>(smem + kStreamWarps * kStreamSlotsMax * 8);
  auto* maxima = sums + 2 * kStreamWarps;
  auto* lost = reinterpret_cast<volatile int*>(maxima + kStreamWarps);      // a load never landed
  const int warp = threadIdx.x >> 5;
  const int group = warp / kGroup, in_group = warp % kGroup;
  const int lane = static_cast<int>(threadIdx.x) - group * kLanes;
  const bool leader = lane == 0;
  uint64_t* bar = bars + group * kStreamSlotsMax;
  uint8_t* ring = smem + kStreamHead + group * p.slots * p.slot_bytes;
  const int d = a.d;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * kGroups;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * kGroups + group;
  // kVec 2: rows of odd length start at odd elements every second time; `stride` is even, so
  // all rows of a group start alike
  const int odd = kVec == 2 ? static_cast<int>(row0 * d & 1) : 0;
  const Place<kVec, kLanes> at = {lane, kLanes, odd, (d + odd) / (2 * kLanes)};
  const int res_bytes = a.residual == nullptr ? 0 : a.residual_f32 ? 4 : 2;

  const auto r_row = [&](int64_t row) {
    return static_cast<const uint8_t*>(a.residual) + row * d * res_bytes;
  };
  const uint32_t x_size = 2u * d, r_size = static_cast<uint32_t>(d * res_bytes);
  const auto up16 = [](const void* q) {
    return reinterpret_cast<const uint8_t*>((reinterpret_cast<uintptr_t>(q) + 15u) & ~static_cast<uintptr_t>(15u));
  };
  const auto down16 = [](const void* q) {
    return reinterpret_cast<const uint8_t*>(reinterpret_cast<uintptr_t>(q) & ~static_cast<uintptr_t>(15u));
  };
  const uint8_t* x_begin = up16(a.x);
  const uint8_t* x_end = down16(x_row(a, a.rows - 1) + d);
  const uint8_t* r_begin = up16(a.residual);
  const uint8_t* r_end = res_bytes == 0 ? nullptr : down16(r_row(a.rows));
  const auto x_piece = [&](const uint8_t* row) {
    if constexpr (kVec == 8) return Piece{row, x_size, 0u, 0u};
    return piece_of(row, x_size, x_begin, x_end);
  };
  const auto r_piece = [&](const uint8_t* row) {
    if constexpr (kVec == 8) return Piece{row, r_size, 0u, 0u};
    return piece_of(row, r_size, r_begin, r_end);
  };
  const auto fetch = [&](int64_t row, int slot) {  // the leader
    if (row >= a.rows) return;
    const Piece x = x_piece(reinterpret_cast<const uint8_t*>(x_row(a, row)));
    Piece r = {nullptr, 0u, 0u, 0u};
    if (res_bytes != 0) r = r_piece(r_row(row));
    mbar_arrive_expect_tx(&bar[slot], x.bytes + r.bytes);
    uint8_t* to = ring + slot * p.slot_bytes;
    bulk_load(to + x.skip, x.lo, x.bytes, &bar[slot]);
    if (res_bytes != 0) bulk_load(to + p.x_bytes + r.skip, r.lo, r.bytes, &bar[slot]);
  };

  if (threadIdx.x == 0) *lost = 0;
  if (leader) {
    for (int s = 0; s < p.slots; ++s) mbar_init(&bar[s], 1);
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  grid_dependency_wait();
  if (leader) {
    for (int s = 0; s < p.slots; ++s) fetch(row0 + s * stride, s);
  }
  // the weight stays in registers up to 48 values a lane, and comes from L1 for every row beyond
  constexpr bool kKeepWeight = kPer <= 48;
  uint32_t w[kPairs];
  if (kKeepWeight && a.weight != nullptr) load_weight<kPairs, kVec>(w, a.weight, d, at);
  __syncthreads();  // the barriers are initialised

  int64_t base = row0 * d;
  const int64_t base_step = stride * d;
  int slot = 0;
  int turn = 0;
  uint32_t phases = 0;        // bit s: parity of slot s
  for (int64_t row = row0; row < a.rows; row += stride, base += base_step) {
    uint8_t* xs = ring + slot * p.slot_bytes;
    uint8_t* rs = xs + p.x_bytes;
    // A wait that runs out is reported, and waited for once more: the ring stays in step, and
    // no load is in flight when the CTA exits.
    const uint32_t parity = (phases >> slot) & 1u;
    if (*lost == 0 && !mbar_wait_bounded(&bar[slot], parity, wait_limit)) {
      atomicOr(err_word, kErrWaitProducer);
      if (!mbar_wait_bounded(&bar[slot], parity, wait_limit > kDefaultWaitLimit ? wait_limit : kDefaultWaitLimit))
        *lost = 1;  // later rows are not waited for; their outputs are undefined
    }
    phases ^= 1u << slot;
    if constexpr (kVec != 8) {
      const uint8_t* from = reinterpret_cast<const uint8_t*>(x_row(a, row));
      const Piece x = x_piece(from);
      xs += x.off;
      bool patched = patch_row<uint16_t>(from, xs, x_size, x, lane);
      if (res_bytes != 0) {
        const Piece r = r_piece(r_row(row));
        rs += r.off;
        patched |= res_bytes == 4 ? patch_row<float>(r_row(row), rs, r_size, r, lane)
                                  : patch_row<uint16_t>(r_row(row), rs, r_size, r, lane);
      }
      if (patched) {
        fence_proxy_async_smem();  // the slot's next bulk copy comes after these stores
        group_sync<kGroup>(group);
      }
    }
    uint32_t xw[kPairs];
    load_bf16<kPairs, kVec>(xw, reinterpret_cast<const uint16_t*>(xs), d, at);
    uint64_t s[kPairs];
#pragma unroll
    for (int i = 0; i < kPairs; ++i) s[i] = f2_of_bf16x2(xw[i]);
    if (res_bytes != 0) {
      uint8_t* to = kVec == 2 ? rs : static_cast<uint8_t*>(a.residual_out) + base * res_bytes;
      add_residual<kPairs, kVec>(s, rs, res_bytes == 4, to, true, d, at);
    }
    if constexpr (kVec == 2) mask_pairs(s, d, at);
    // A warp refills its slot as soon as it holds the row.  A larger group does after the sum's
    // barrier, which says the same (the partial sums alternate between two places, so that no
    // other barrier is needed before them).
    if constexpr (kGroup == 1) {
      __syncwarp();
      if (leader && kVec != 2) fetch(row + p.slots * stride, slot);
    }
    const float sq = group_reduce<kGroup>(sum_squares(s), sums + (turn ^= 1) * kStreamWarps + group * kGroup, group,
                                          in_group, [](float x, float y) { return x + y; });
    if constexpr (kVec == 2) {
      // the previous row's slot held its outputs: free once their copies have read it
      if (leader && row != row0) {
        bulk_wait_group_read0();
        fetch(row + (p.slots - 1) * stride, slot == 0 ? p.slots - 1 : slot - 1);
      }
    } else if constexpr (kGroup > 1) {
      if (leader) fetch(row + p.slots * stride, slot);
    }
    const float rstd = rsqrtf(sq / static_cast<float>(d) + a.eps);
    if (!kKeepWeight && a.weight != nullptr) load_weight<kPairs, kVec>(w, a.weight, d, at);
    if (a.weight != nullptr) apply_weight(s, w);
    if (a.y != nullptr)
      store_bf16<kPairs, kVec>(kVec == 2 ? reinterpret_cast<uint16_t*>(xs) : a.y + base, s, f2_pack(rstd, rstd),
                               d, at);
    uint8_t* qs = a.q + base;  // kVec 2: in x's place, at its own offset in 16 bytes
    if constexpr (kVec == 2) qs = ring + slot * p.slot_bytes + (reinterpret_cast<uintptr_t>(a.q + base) & 15u);
    if (a.q != nullptr) {
      const float m = group_reduce<kGroup>(max_abs(s), maxima + group * kGroup, group, in_group,
                                           [](float x, float y) { return max_nan(x, y); });
      const float scale = scale448(m * rstd), f = rstd * __frcp_rn(scale);
      if (leader) a.scale[row] = scale;
      store_e4m3<kPairs, kVec>(qs, s, f2_pack(f, f), d, at);
    }
    if constexpr (kVec == 2) {
      fence_proxy_async_smem();
      group_sync<kGroup>(group);
      if (res_bytes != 0)
        flush_row(static_cast<uint8_t*>(a.residual_out) + base * res_bytes, rs, d * res_bytes, res_bytes, lane);
      if (a.y != nullptr) flush_row(reinterpret_cast<uint8_t*>(a.y + base), xs, 2 * d, 2, lane);
      if (a.q != nullptr) flush_row(a.q + base, qs, d, 1, lane);
      if (leader) bulk_commit_group();
    }
    if (++slot == p.slots) slot = 0;
  }
  if (kVec == 2 && leader) bulk_wait_group0();  // the copies out of shared memory are complete
}

template <int kLanes, int kRows, int kPer>
cudaError_t norm_launch(const NormArgs& a, bool vec, cudaStream_t st) {
  const int threads = kLanes != 0 ? kNormThreads : ((a.d + kPer - 1) / kPer + 31) / 32 * 32;
  const int rows = kLanes != 0 ? kNormThreads / kLanes * kRows : 1;
  const unsigned grid = static_cast<unsigned>((a.rows + rows - 1) / rows);
  if (vec) return launch_dependent(rms_norm_kernel<kLanes, kRows, kPer, 8>, grid, threads, 0, st, 0, a);
  return launch_dependent(rms_norm_kernel<kLanes, kRows, kPer, 1>, grid, threads, 0, st, 0, a);
}

template <int kLanes, int kPer = 8>
cudaError_t norm_short(const NormArgs& a, bool vec, cudaStream_t st) {
  // two rows a group once that still leaves every SM its threads (92160 rows of 128: 10.0 us
  // with one, 9.0 with two, 9.4 with four)
  if (a.rows * kLanes >= static_cast<int64_t>(sm_count()) * 2048 * 2)
    return norm_launch<kLanes, 16 / kPer, kPer>(a, vec, st);
  return norm_launch<kLanes, 1, kPer>(a, vec, st);
}

template <int kGroup, int kPer, int kVec>
cudaError_t stream_launch(const NormArgs& a, const StreamPlan& p, uint64_t wait_limit,
                          uint32_t* err_word, cudaStream_t st) {
  static ContextCache attr_done;
  auto* kernel = rms_norm_stream_kernel<kGroup, kPer, kVec>;
  const int bytes = kStreamHead + kStreamSmem;
  if (cudaError_t e = ensure_max_dynamic_smem(attr_done, reinterpret_cast<const void*>(kernel), bytes))
    return e;
  return launch_dependent(kernel, static_cast<unsigned>(sm_count()), kStreamThreads, bytes, st, 0, a, p,
                          wait_limit, err_word);
}

template <int kGroup, int kVec>
cudaError_t stream_by_width(const NormArgs& a, const StreamPlan& p, uint64_t wait_limit,
                            uint32_t* err_word, cudaStream_t st) {
  const int per = (a.d + (kVec == 2 ? 1 : 0) + 32 * kGroup - 1) / (32 * kGroup);
  // 17 values a lane at the least (rows are longer than 512, and groups grow when they have
  // to); sixteen warps hold the longest row with 32
  if (kGroup == kStreamWarps || per <= 32)
    return stream_launch<kGroup, 32, kVec>(a, p, wait_limit, err_word, st);
  if constexpr (kGroup < kStreamWarps) {
    if (per <= 48) return stream_launch<kGroup, 48, kVec>(a, p, wait_limit, err_word, st);
    return stream_launch<kGroup, 72, kVec>(a, p, wait_limit, err_word, st);
  }
  return cudaErrorInvalidValue;
}

template <int kGroup>
cudaError_t stream_by_form(const NormArgs& a, const StreamPlan& p, int form, uint64_t wait_limit,
                           uint32_t* err_word, cudaStream_t st) {
  if (form == 8) return stream_by_width<kGroup, 8>(a, p, wait_limit, err_word, st);
  if (form == 2) return stream_by_width<kGroup, 2>(a, p, wait_limit, err_word, st);
  return stream_by_width<kGroup, 1>(a, p, wait_limit, err_word, st);
}

}  // namespace

int64_t rms_norm_max_d() { return kNormMaxD; }

cudaError_t launch_rms_norm(const NormArgs& args, uint64_t wait_limit, cudaStream_t st) {
  if (args.rows <= 0) return cudaSuccess;
  NormArgs a = args;
  a.inner_shift = 0;
  while ((int64_t(1) << a.inner_shift) < a.inner) ++a.inner_shift;
  a.inner_mul = static_cast<uint32_t>(
      ((uint64_t(1) << 32) * ((uint64_t(1) << a.inner_shift) - static_cast<uint64_t>(a.inner))) /
          static_cast<uint64_t>(a.inner) + 1);
  const auto at16 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
  const bool vec = a.d % 8 == 0 && a.outer_stride % 8 == 0 && a.inner_stride % 8 == 0 &&
                   at16(a.x) && at16(a.weight) && at16(a.residual) && at16(a.residual_out) &&
                   at16(a.y) && at16(a.q);
  const int d = a.d;
  if (d > kNormMaxD) return cudaErrorInvalidValue;
  if (d <= 64) return norm_short<8>(a, vec, st);
  if (d <= 128) return norm_short<16>(a, vec, st);
  if (d <= 256) return norm_short<32>(a, vec, st);
  if (d <= 512) return norm_short<32, 16>(a, vec, st);
  {
    // warps per row: rings of two rows per group within the shared memory, 72 values a lane
    StreamPlan p;
    const int res = a.residual == nullptr ? 0 : a.residual_f32 ? 4 : 2, slack = vec ? 0 : 16;
    p.x_bytes = (2 * d + slack + 15) / 16 * 16;
    p.slot_bytes = p.x_bytes + (res == 0 ? 0 : (res * d + slack + 15) / 16 * 16);
    int group = 1;
    while (group < 16 && (d + 1 > 32 * group * 72 || kStreamWarps / group * 2 * p.slot_bytes > kStreamSmem))
      group *= 2;
    p.slots = kStreamSmem / (kStreamWarps / group) / p.slot_bytes;
    if (p.slots > kStreamSlotsMax) p.slots = kStreamSlotsMax;
    const auto off = [](const void* q, uintptr_t mask) { return (reinterpret_cast<uintptr_t>(q) & mask) != 0; };
    const bool even = (sm_count() * (kStreamWarps / group)) % 2 == 0;
    // one output, rows end to end from 16-byte aligned starts: every row of every tensor but q
    // then has its x's offset
    const bool pairs = !vec && a.inner == 1 && a.outer_stride == d && even && !off(a.x, 15) && !off(a.y, 15) &&
                       !off(a.q, 15) && !off(a.residual, 15) && !off(a.residual_out, 15) &&
                       (a.y == nullptr || a.q == nullptr);
    if (a.rows >= static_cast<int64_t>(sm_count()) * (kStreamWarps / group) * 2) {
      uint32_t* err_word = error_word_ptr();
      if (err_word == nullptr) return cudaErrorInvalidSymbol;
      const int form = vec ? 8 : pairs ? 2 : 1;
      switch (group) {
        case 1: return stream_by_form<1>(a, p, form, wait_limit, err_word, st);
        case 2: return stream_by_form<2>(a, p, form, wait_limit, err_word, st);
        case 4: return stream_by_form<4>(a, p, form, wait_limit, err_word, st);
        case 8: return stream_by_form<8>(a, p, form, wait_limit, err_word, st);
        default: return stream_by_form<16>(a, p, form, wait_limit, err_word, st);
      }
    }
  }
  if (d <= 8 * kNormMaxThreads) return norm_launch<0, 1, 8>(a, vec, st);
  return norm_launch<0, 1, 16>(a, vec, st);
}

}  // namespace fvq
