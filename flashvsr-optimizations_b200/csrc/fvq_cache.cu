// fvq_cache.cu -- paged FP8 store of attention keys and values.
//
// Pages of `page` slots; a slot holds, for each head, d E4M3 codes and one fp32 scale:
//   write: scale = max(max|x| / 448, 1e-12),  q = e4m3(x * (1 / scale))   per token and head
//   read:  bf16(q * scale), rows past a sequence's length zero
//
// Both are HBM-bound copies with a conversion: keys and values go in one launch, a row of
// d <= 512 values to a power-of-two group of lanes (8 values a lane, up to two vectors), so
// that its maximum needs only shuffles.  Slot and page numbers come from the device and are
// checked there: a negative slot is padding and stores nothing, a slot or page past the store
// touches nothing (the rows read are zero) and sets a bit of the device error word.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "fvq_internal.h"
#include "fvq_ptx.cuh"

namespace fvq {

namespace {

constexpr int kCacheThreads = 256;

__device__ __forceinline__ float bf_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf_hi(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }

__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// two E4M3 codes -> two fp32 values (exact)
__device__ __forceinline__ void e4m3x2_to_f32(uint32_t codes, float& lo, float& hi) {
  uint32_t h2;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"(static_cast<uint16_t>(codes)));
  const __half2 h = *reinterpret_cast<const __half2*>(&h2);
  lo = __low2float(h);
  hi = __high2float(h);
}

// kLanes lanes a row; blockIdx.y: 0 keys, 1 values.
template <int kLanes, int kVecs>
__global__ void __launch_bounds__(kCacheThreads) cache_write_kernel(const CacheWriteArgs a,
                                                                   uint32_t* err_word) {
  const CacheRows src = blockIdx.y == 0 ? a.k : a.v;
  const int lane = threadIdx.x % kLanes;
  int64_t row = static_cast<int64_t>(blockIdx.x) * (kCacheThreads / kLanes) + threadIdx.x / kLanes;
  const bool live = row < a.rows;
  if (!live) row = a.rows - 1;  // whole warps at the shuffles; nothing stored
  const int64_t token = row / a.heads;
  const int head = static_cast<int>(row - token * a.heads);
  const int64_t slot = __ldg(a.slots + token);
  const uint16_t* x = src.x + token * src.token_stride + head * src.head_stride;
  const int nvec = a.d / 8;
  uint4 v[kVecs];
  uint32_t m2 = 0;  // max |x|, magnitude bits of the low and high halves (NaN on top)
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int j = lane + i * kLanes;
    v[i] = j < nvec ? __ldg(reinterpret_cast<const uint4*>(x) + j) : make_uint4(0, 0, 0, 0);
    m2 = max_u16x2(m2, max_u16x2(v[i].x & 0x7FFF7FFFu, v[i].y & 0x7FFF7FFFu));
    m2 = max_u16x2(m2, max_u16x2(v[i].z & 0x7FFF7FFFu, v[i].w & 0x7FFF7FFFu));
  }
  uint32_t m = max(m2 & 0xFFFFu, m2 >> 16);
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
  if (!live || slot < 0) return;
  if (slot >= a.num_slots) {
    if (lane == 0 && head == 0 && blockIdx.y == 0) atomicOr(err_word, kErrCacheSlot);
    return;
  }
  const float by448 = __fdiv_rn(__uint_as_float(m << 16), 448.0f);
  const float scale = by448 < 1e-12f ? 1e-12f : by448;  // NaN stays NaN
  const float inv = __frcp_rn(scale);
  const int64_t at = slot * a.heads + head;
  if (lane == 0) src.scale[at] = scale;
  uint2* q = reinterpret_cast<uint2*>(src.codes + at * a.d);
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int j = lane + i * kLanes;
    if (j >= nvec) continue;
    const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
    uint32_t c[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) c[e] = e4m3x2(bf_lo(w[e]) * inv, bf_hi(w[e]) * inv);
    q[j] = make_uint2(c[0] | (c[1] << 16), c[2] | (c[3] << 16));
  }
}

// One thread per 8 codes; blockIdx.y: sequence, blockIdx.z: 0 keys, 1 values; blockIdx.x
// walks the sequence's positions x heads x d / 8.
__global__ void __launch_bounds__(kCacheThreads) cache_read_kernel(const CacheReadArgs a,
                                                                  uint32_t* err_word) {
  const bool values = blockIdx.z != 0;
  const uint8_t* codes = values ? a.v_codes : a.k_codes;
  const float* scales = values ? a.v_scale : a.k_scale;
  uint16_t* out = values ? a.v_out : a.k_out;
  const int64_t b = blockIdx.y;
  const int32_t len_raw = __ldg(a.lengths + b);
  const int64_t most = a.pages_per_seq * a.page < a.max_len ? a.pages_per_seq * a.page : a.max_len;
  const int64_t len = len_raw < most ? len_raw : most;
  if (len_raw > most && blockIdx.x == 0 && threadIdx.x == 0 && !values)
    atomicOr(err_word, kErrCachePage);
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kCacheThreads + threadIdx.x;
  const int dv = a.d / 8;
  const int64_t row = i / dv;  // position x heads + head
  const int64_t pos = row / a.heads;
  if (pos >= a.max_len) return;
  uint4 o = make_uint4(0, 0, 0, 0);
  if (pos < len) {
    const int64_t p = pos / a.page;
    const int64_t page = __ldg(a.table + b * a.pages_per_seq + p);
    if (page >= 0 && page < a.num_pages) {
      const int64_t at = (page * a.page + (pos - p * a.page)) * a.heads + (row - pos * a.heads);
      const uint2 c = __ldg(reinterpret_cast<const uint2*>(codes + at * a.d) + (i - row * dv));
      const float s = __ldg(scales + at);
      const uint32_t cw[4] = {c.x & 0xFFFFu, c.x >> 16, c.y & 0xFFFFu, c.y >> 16};
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float lo, hi;
        e4m3x2_to_f32(cw[e], lo, hi);
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[e]) : "f"(hi * s), "f"(lo * s));
      }
      o = make_uint4(w[0], w[1], w[2], w[3]);
    } else if (!values) {
      atomicOr(err_word, kErrCachePage);
    }
  }
  reinterpret_cast<uint4*>(out)[b * a.max_len * a.heads * dv + i] = o;
}

template <int kLanes, int kVecs>
void write_launch(const CacheWriteArgs& a, uint32_t* err_word, cudaStream_t st) {
  constexpr int kRows = kCacheThreads / kLanes;
  const dim3 grid(static_cast<unsigned>((a.rows + kRows - 1) / kRows), 2);
  cache_write_kernel<kLanes, kVecs><<<grid, kCacheThreads, 0, st>>>(a, err_word);
}

}  // namespace

cudaError_t launch_cache_write(const CacheWriteArgs& a, uint32_t* err_word, cudaStream_t st) {
  if (a.rows <= 0) return cudaSuccess;
  const int nvec = a.d / 8;
  if (nvec <= 8) write_launch<8, 1>(a, err_word, st);
  else if (nvec <= 16) write_launch<16, 1>(a, err_word, st);
  else if (nvec <= 32) write_launch<32, 1>(a, err_word, st);
  else if (nvec <= 64) write_launch<32, 2>(a, err_word, st);
  else return cudaErrorInvalidValue;
  return cudaGetLastError();
}

cudaError_t launch_cache_read(const CacheReadArgs& a, uint32_t* err_word, cudaStream_t st) {
  const int64_t threads = a.max_len * a.heads * (a.d / 8);
  if (threads <= 0 || a.batch <= 0) return cudaSuccess;
  const dim3 grid(static_cast<unsigned>((threads + kCacheThreads - 1) / kCacheThreads),
                  static_cast<unsigned>(a.batch), 2);
  cache_read_kernel<<<grid, kCacheThreads, 0, st>>>(a, err_word);
  return cudaGetLastError();
}

}  // namespace fvq
