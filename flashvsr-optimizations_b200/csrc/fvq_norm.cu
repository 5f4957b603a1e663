// fvq_norm.cu -- root-mean-square norm with the residual's addition, in bf16 or E4M3.
//
//   s = x + r                                   fp32; r bf16 or fp32 (optional)
//   v = s * rsqrt(mean(s^2) + eps) * w          fp32; w bf16 (optional)
//   r_out = s in r's type,  y = bf16(v)         and / or
//   scale = max(max|v| / 448, 1e-12),  q = e4m3(v * (1 / scale))
//
// Everything up to the outputs is fp32 in registers; each output is rounded once.  q multiplies
// by the correctly rounded reciprocal of the scale instead of dividing: two roundings of 2^-24
// ahead of E4M3's 2^-4, a third of the instructions.  A NaN in a row makes the row NaN, an
// infinity gives what the formulas give (0 for the finite values, NaN for the infinite ones).
//
// HBM-bound: x and r are read once, every output is written once; the row stays in registers
// between the two reductions (sum of squares, then max |v| for E4M3).  Short rows go to
// sub-warp groups of lanes so that a warp's 16-byte loads stay dense, rows of at most 2048
// values to one warp (no barrier), longer ones to one CTA.  Row starts or lengths that are no
// multiple of 16 bytes take element-wise loads (kVec = 1): neighbouring lanes read
// neighbouring elements, so the sectors fetched are the same.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "fvq_internal.h"
#include "fvq_ptx.cuh"

namespace fvq {

namespace {

constexpr int kNormThreads = 256;
constexpr int kNormMaxPerThread = 64;  // row elements a thread holds in registers

__device__ __forceinline__ float bf_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf_hi(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }

__device__ __forceinline__ uint32_t bf16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// kVec consecutive bf16 / fp32 elements <-> fp32 registers (kVec 8: 16-byte accesses)
template <int kVec>
__device__ __forceinline__ void load_bf16(const uint16_t* p, float* f) {
  if constexpr (kVec == 8) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f[2 * j] = bf_lo(w[j]);
      f[2 * j + 1] = bf_hi(w[j]);
    }
  } else {
    f[0] = __uint_as_float(static_cast<uint32_t>(__ldg(p)) << 16);
  }
}

template <int kVec>
__device__ __forceinline__ void load_f32(const float* p, float* f) {
  if constexpr (kVec == 8) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(p));
    const float4 b = __ldg(reinterpret_cast<const float4*>(p) + 1);
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w;
    f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
  } else {
    f[0] = __ldg(p);
  }
}

template <int kVec>
__device__ __forceinline__ void store_bf16(uint16_t* p, const float* f) {
  if constexpr (kVec == 8)
    *reinterpret_cast<uint4*>(p) = make_uint4(bf16x2(f[0], f[1]), bf16x2(f[2], f[3]),
                                              bf16x2(f[4], f[5]), bf16x2(f[6], f[7]));
  else
    *p = __bfloat16_as_ushort(__float2bfloat16_rn(f[0]));
}

template <int kVec>
__device__ __forceinline__ void store_f32(float* p, const float* f) {
  if constexpr (kVec == 8) {
    reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
  } else {
    *p = f[0];
  }
}

// kLanes threads share a row: 8, 16 or 32 lanes of a warp, or all kNormThreads of the CTA.
template <int kLanes>
__device__ __forceinline__ float row_sum(float v, float* smem) {
  constexpr int kWidth = kLanes < 32 ? kLanes : 32;
#pragma unroll
  for (int o = kWidth / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  if constexpr (kLanes > 32) {
    if ((threadIdx.x & 31) == 0) smem[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int w = 0; w < kLanes / 32; ++w) v += smem[w];
  }
  return v;
}

// Maximum of magnitude bits: orders like the values, infinities above finite ones, NaN on top.
template <int kLanes>
__device__ __forceinline__ uint32_t row_max(uint32_t v, uint32_t* smem) {
  constexpr int kWidth = kLanes < 32 ? kLanes : 32;
#pragma unroll
  for (int o = kWidth / 2; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
  if constexpr (kLanes > 32) {
    if ((threadIdx.x & 31) == 0) smem[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int w = 0; w < kLanes / 32; ++w) v = max(v, smem[w]);
  }
  return v;
}

// kPer: elements per thread (a multiple of kVec); a row has at most kLanes * kPer.
template <int kLanes, int kPer, int kVec>
__global__ void __launch_bounds__(kNormThreads) rms_norm_kernel(const NormArgs a) {
  __shared__ float sum_smem[kNormThreads / 32];
  __shared__ uint32_t max_smem[kNormThreads / 32];
  constexpr int kIter = kPer / kVec;
  const int lane = threadIdx.x % kLanes;
  int64_t row = static_cast<int64_t>(blockIdx.x) * (kNormThreads / kLanes) + threadIdx.x / kLanes;
  // a group past the last row repeats the last one without storing: the warp's shuffles stay whole
  const bool live = row < a.rows;
  if (!live) row = a.rows - 1;
  const int64_t outer = row / a.inner;
  const uint16_t* x = a.x + outer * a.outer_stride + (row - outer * a.inner) * a.inner_stride;
  const int d = a.d;
  const int64_t base = row * d;

  float s[kPer];
#pragma unroll
  for (int i = 0; i < kIter; ++i) {
    const int j = (lane + i * kLanes) * kVec;
    if (j < d) {
      load_bf16<kVec>(x + j, &s[i * kVec]);
    } else {
#pragma unroll
      for (int e = 0; e < kVec; ++e) s[i * kVec + e] = 0.0f;
    }
  }
  if (a.residual != nullptr) {
    float r[kPer];
    if (a.residual_f32) {
      const float* p = static_cast<const float*>(a.residual) + base;
#pragma unroll
      for (int i = 0; i < kIter; ++i) {
        const int j = (lane + i * kLanes) * kVec;
        if (j < d) load_f32<kVec>(p + j, &r[i * kVec]);
      }
    } else {
      const uint16_t* p = static_cast<const uint16_t*>(a.residual) + base;
#pragma unroll
      for (int i = 0; i < kIter; ++i) {
        const int j = (lane + i * kLanes) * kVec;
        if (j < d) load_bf16<kVec>(p + j, &r[i * kVec]);
      }
    }
#pragma unroll
    for (int i = 0; i < kIter; ++i) {
      const int j = (lane + i * kLanes) * kVec;
      if (j < d) {
#pragma unroll
        for (int e = 0; e < kVec; ++e) s[i * kVec + e] += r[i * kVec + e];
        if (live) {
          if (a.residual_f32)
            store_f32<kVec>(static_cast<float*>(a.residual_out) + base + j, &s[i * kVec]);
          else
            store_bf16<kVec>(static_cast<uint16_t*>(a.residual_out) + base + j, &s[i * kVec]);
        }
      }
    }
  }
  float sq = 0.0f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) sq = fmaf(s[i], s[i], sq);
  sq = row_sum<kLanes>(sq, sum_smem);
  const float rstd = rsqrtf(sq / static_cast<float>(d) + a.eps);

  uint32_t mag = 0;
#pragma unroll
  for (int i = 0; i < kIter; ++i) {
    const int j = (lane + i * kLanes) * kVec;
    if (j < d) {
      float w[kVec];
      if (a.weight != nullptr) {
        load_bf16<kVec>(a.weight + j, w);
      } else {
#pragma unroll
        for (int e = 0; e < kVec; ++e) w[e] = 1.0f;
      }
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        float& v = s[i * kVec + e];
        v = v * rstd * w[e];
        mag = max(mag, __float_as_uint(v) & 0x7FFFFFFFu);
      }
      if (a.y != nullptr && live) store_bf16<kVec>(a.y + base + j, &s[i * kVec]);
    }
  }
  if (a.q != nullptr) {
    mag = row_max<kLanes>(mag, max_smem);
    const float by448 = __fdiv_rn(__uint_as_float(mag), 448.0f);
    const float scale = by448 < 1e-12f ? 1e-12f : by448;  // NaN stays NaN
    const float inv = __frcp_rn(scale);
    if (!live) return;
    if (lane == 0) a.scale[row] = scale;
    uint8_t* q = a.q + base;
#pragma unroll
    for (int i = 0; i < kIter; ++i) {
      const int j = (lane + i * kLanes) * kVec;
      if (j < d) {
        if constexpr (kVec == 8) {
          uint32_t c[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            c[e] = e4m3x2(s[i * kVec + 2 * e] * inv, s[i * kVec + 2 * e + 1] * inv);
          *reinterpret_cast<uint2*>(q + j) = make_uint2(c[0] | (c[1] << 16), c[2] | (c[3] << 16));
        } else {
          q[j] = static_cast<uint8_t>(e4m3x2(s[i] * inv, 0.0f) & 0xFFu);
        }
      }
    }
  }
}

template <int kLanes, int kPer>
void norm_launch(const NormArgs& a, bool vec, cudaStream_t st) {
  constexpr int kRows = kNormThreads / kLanes;
  const unsigned grid = static_cast<unsigned>((a.rows + kRows - 1) / kRows);
  if (vec)
    rms_norm_kernel<kLanes, kPer, 8><<<grid, kNormThreads, 0, st>>>(a);
  else
    rms_norm_kernel<kLanes, kPer, 1><<<grid, kNormThreads, 0, st>>>(a);
}

}  // namespace

int64_t rms_norm_max_d() { return static_cast<int64_t>(kNormThreads) * kNormMaxPerThread; }

cudaError_t launch_rms_norm(const NormArgs& a, cudaStream_t st) {
  if (a.rows <= 0) return cudaSuccess;
  const auto at16 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
  const bool vec = a.d % 8 == 0 && a.outer_stride % 8 == 0 && a.inner_stride % 8 == 0 &&
                   at16(a.x) && at16(a.weight) && at16(a.residual) && at16(a.residual_out) &&
                   at16(a.y) && at16(a.q);
  const int d = a.d;
  if (d <= 64) norm_launch<8, 8>(a, vec, st);
  else if (d <= 128) norm_launch<16, 8>(a, vec, st);
  else if (d <= 256) norm_launch<32, 8>(a, vec, st);
  else if (d <= 512) norm_launch<32, 16>(a, vec, st);
  else if (d <= 1024) norm_launch<32, 32>(a, vec, st);
  else if (d <= 1536) norm_launch<32, 48>(a, vec, st);
  else if (d <= 2048) norm_launch<32, 64>(a, vec, st);
  else if (d <= 4096) norm_launch<256, 16>(a, vec, st);
  else if (d <= 6144) norm_launch<256, 24>(a, vec, st);
  else if (d <= 8192) norm_launch<256, 32>(a, vec, st);
  else if (d <= 10240) norm_launch<256, 40>(a, vec, st);
  else if (d <= 12288) norm_launch<256, 48>(a, vec, st);
  else if (d <= rms_norm_max_d()) norm_launch<256, 64>(a, vec, st);
  else return cudaErrorInvalidValue;
  return cudaGetLastError();
}

}  // namespace fvq
