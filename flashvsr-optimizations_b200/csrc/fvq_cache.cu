// fvq_cache.cu -- paged FP8 store of attention keys and values.
//
// Pages of `page` slots; a slot holds, for each head, d E4M3 codes and one fp32 scale:
//   write: scale = max(max|x| / 448, 1e-12),  q = e4m3(x * (1 / scale))   per token and head
//   read:  bf16(q * scale), rows past a sequence's length zero
//
// Both are HBM-bound copies with a conversion, keys and values in one launch.  Writing gives
// a row of d <= 512 values to a power-of-two group of lanes (16 values a lane, 8 where
// alignment allows no more), so that its maximum needs only shuffles; reading gives 16 (or 8)
// codes to a thread, four vectors in flight each.  Row and position arithmetic is 32-bit with
// multiplications in place of divisions: with 64-bit divisions both were bound by issue slots
// (reading 4 x 7680 tokens of 12 heads of 128 took 78 us).  Slot and page numbers come from the
// device and are checked there: a negative slot is padding and stores nothing, a slot or page
// past the store touches nothing (the rows read are zero) and sets a bit of the device error
// word.
//
// Measured on a B200, back to back in a CUDA graph (a copy moves 6.5 TB/s), heads of 128, 12 a
// token: writing 64 tokens 1.4 us, 7680 tokens 12.5 us (71 MB, 5.7 TB/s, 1.5 us of it start and
// end); reading 4 x 7680 tokens 40.6 us (247 MB, 6.1 TB/s).
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "fvq_internal.h"
#include "fvq_launch.h"
#include "fvq_ptx.cuh"

namespace fvq {

namespace {

constexpr int kCacheThreads = 256;

__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// Division by a fixed divisor, exact below 2^31 (Granlund and Montgomery, "Division by invariant
// integers using multiplication", 1994).
struct Divider {
  uint32_t d, mul;
  int shift;
};

Divider divider(int64_t d) {
  Divider r;
  r.d = static_cast<uint32_t>(d);
  r.shift = 0;
  while ((int64_t(1) << r.shift) < d) ++r.shift;
  r.mul = static_cast<uint32_t>(((uint64_t(1) << 32) * ((uint64_t(1) << r.shift) - static_cast<uint64_t>(d))) /
                                    static_cast<uint64_t>(d) + 1);
  return r;
}

__device__ __forceinline__ uint32_t divide(uint32_t n, const Divider& by) {
  return (n + __umulhi(n, by.mul)) >> by.shift;
}

// four E4M3 codes * scale -> four bf16 values (one fp32 product and one rounding each)
__device__ __forceinline__ uint2 dequantize4(uint32_t codes, float scale) {
  uint32_t h[2], w[2];
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h[0]) : "h"(static_cast<uint16_t>(codes)));
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h[1]) : "h"(static_cast<uint16_t>(codes >> 16)));
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(f.y * scale), "f"(f.x * scale));
  }
  return make_uint2(w[0], w[1]);
}

// 32-byte accesses: a warp's are whole sectors whichever way they are split up
__device__ __forceinline__ void load32(const void* p, uint32_t (&w)[8]) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]),
                 "=r"(w[7])
               : "l"(p));
}

__device__ __forceinline__ void store32(void* p, const uint2 (&w)[4]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0].x), "r"(w[0].y),
               "r"(w[1].x), "r"(w[1].y), "r"(w[2].x), "r"(w[2].y), "r"(w[3].x), "r"(w[3].y)
               : "memory");
}

// kLanes lanes a row, kElems (8 or 16) values a lane and vector, kRows rows a group, whose
// loads overlap; blockIdx.y: 0 keys, 1 values.
template <int kLanes, int kElems, int kVecs, int kRows>
__global__ void __launch_bounds__(kCacheThreads) cache_write_kernel(const CacheWriteArgs a,
                                                                   const Divider by_heads,
                                                                   uint32_t* err_word) {
  grid_launch_dependents();
  grid_dependency_wait();
  const CacheRows src = blockIdx.y == 0 ? a.k : a.v;
  constexpr uint32_t kStep = kCacheThreads / kLanes;
  const int lane = threadIdx.x % kLanes;
  const uint32_t first = blockIdx.x * (kStep * kRows) + threadIdx.x / kLanes;
  const uint32_t rows = static_cast<uint32_t>(a.rows);
  constexpr int kWords = kElems / 2;
  const int nvec = a.d / kElems;
  uint32_t v[kRows][kVecs][kWords];
  int64_t slot[kRows];
#pragma unroll
  for (int k = 0; k < kRows; ++k) {
    const uint32_t row = min(first + k * kStep, rows - 1);  // whole warps at the shuffles
    const uint32_t token = divide(row, by_heads), head = row - token * by_heads.d;
    slot[k] = first + k * kStep < rows ? a.slots[token] : -1;
    const uint16_t* x = src.x + token * src.token_stride + head * src.head_stride;
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int j = lane + i * kLanes;
#pragma unroll
      for (int e = 0; e < kWords; ++e) v[k][i][e] = 0;
      if (j >= nvec) continue;
      if constexpr (kElems == 16) {
        load32(x + j * 16, v[k][i]);
      } else {
        const uint4 q = *reinterpret_cast<const uint4*>(x + j * 8);
        v[k][i][0] = q.x, v[k][i][1] = q.y, v[k][i][2] = q.z, v[k][i][3] = q.w;
      }
    }
  }
#pragma unroll
  for (int k = 0; k < kRows; ++k) {
    uint32_t m2 = 0;  // max |x|, magnitude bits of the low and high halves (NaN on top)
#pragma unroll
    for (int i = 0; i < kVecs; ++i)
#pragma unroll
      for (int e = 0; e < kWords; ++e) m2 = max_u16x2(m2, v[k][i][e] & 0x7FFF7FFFu);
    uint32_t m = max(m2 & 0xFFFFu, m2 >> 16);
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
    const uint32_t row = min(first + k * kStep, rows - 1);
    const uint32_t head = row - divide(row, by_heads) * by_heads.d;
    if (slot[k] < 0) continue;
    if (slot[k] >= a.num_slots) {
      if (lane == 0 && head == 0 && blockIdx.y == 0) atomicOr(err_word, kErrCacheSlot);
      continue;
    }
    const float by448 = __fdiv_rn(__uint_as_float(m << 16), 448.0f);
    const float scale = by448 < 1e-12f ? 1e-12f : by448;  // NaN stays NaN
    const float inv = __frcp_rn(scale);
    const int64_t at = slot[k] * a.heads + head;
    if (lane == 0) src.scale[at] = scale;
    uint8_t* q = src.codes + at * a.d;
    const uint64_t inv2 = f2_pack(inv, inv);
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int j = lane + i * kLanes;
      if (j >= nvec) continue;
      uint32_t c[kWords / 2];
#pragma unroll
      for (int e = 0; e < kWords / 2; ++e)
        c[e] = f2_to_e4m3x2(f2_mul(f2_of_bf16x2(v[k][i][2 * e]), inv2)) |
               (f2_to_e4m3x2(f2_mul(f2_of_bf16x2(v[k][i][2 * e + 1]), inv2)) << 16);
      if constexpr (kElems == 16)
        *reinterpret_cast<uint4*>(q + j * 16) = make_uint4(c[0], c[1], c[2], c[3]);
      else
        *reinterpret_cast<uint2*>(q + j * 8) = make_uint2(c[0], c[1]);
    }
  }
}

// A CTA reads `span` positions of one sequence: their span * heads * d / kCodes vectors, four
// at a time per thread.  blockIdx.y: sequence, blockIdx.z: 0 keys, 1 values.
constexpr int kReadUnroll = 4;
template <int kCodes>
__global__ void __launch_bounds__(kCacheThreads)
    cache_read_kernel(const CacheReadArgs a, const int span, const Divider by_token,
                      const Divider by_row, const Divider by_page, uint32_t* err_word) {
  grid_launch_dependents();
  grid_dependency_wait();
  const bool values = blockIdx.z != 0;
  const uint8_t* codes = values ? a.v_codes : a.k_codes;
  const float* scales = values ? a.v_scale : a.k_scale;
  const int64_t b = blockIdx.y;
  const int32_t len_raw = a.lengths[b];
  const int64_t most = a.pages_per_seq * a.page < a.max_len ? a.pages_per_seq * a.page : a.max_len;
  const int64_t len = len_raw < most ? len_raw : most;
  if (len_raw > most && blockIdx.x == 0 && threadIdx.x == 0 && !values)
    atomicOr(err_word, kErrCachePage);
  const int64_t pos0 = static_cast<int64_t>(blockIdx.x) * span;
  const int64_t left = a.max_len - pos0;  // > 0
  const uint32_t count = static_cast<uint32_t>(left < span ? left : span) * by_token.d;  // vectors
  uint16_t* out = (values ? a.v_out : a.k_out) + (b * a.max_len + pos0) * a.heads * a.d;
  const int32_t* table = a.table + b * a.pages_per_seq;
  for (uint32_t i0 = threadIdx.x; i0 < count; i0 += kCacheThreads * kReadUnroll) {
    uint32_t c[kReadUnroll][kCodes / 4];
    float s[kReadUnroll];
#pragma unroll
    for (int u = 0; u < kReadUnroll; ++u) {
      const uint32_t i = i0 + u * kCacheThreads;
#pragma unroll
      for (int e = 0; e < kCodes / 4; ++e) c[u][e] = 0;
      s[u] = 0.0f;
      if (i >= count) continue;
      const uint32_t t = divide(i, by_token), vec = i - t * by_token.d;  // vector in the token
      const uint32_t pos = static_cast<uint32_t>(pos0) + t;              // below 2^31
      if (pos >= len) continue;
      const uint32_t p = divide(pos, by_page);
      const int64_t page = table[p];
      if (page < 0 || page >= a.num_pages) {
        if (vec == 0 && !values) atomicOr(err_word, kErrCachePage);
        continue;
      }
      const int64_t slot = page * a.page + (pos - p * by_page.d);
      const uint8_t* at = codes + (slot * a.heads * a.d + static_cast<int64_t>(vec) * kCodes);
      if constexpr (kCodes == 16) {
        const uint4 v = *reinterpret_cast<const uint4*>(at);
        c[u][0] = v.x, c[u][1] = v.y, c[u][2] = v.z, c[u][3] = v.w;
      } else {
        const uint2 v = *reinterpret_cast<const uint2*>(at);
        c[u][0] = v.x, c[u][1] = v.y;
      }
      s[u] = scales[slot * a.heads + divide(vec, by_row)];
    }
#pragma unroll
    for (int u = 0; u < kReadUnroll; ++u) {
      const uint32_t i = i0 + u * kCacheThreads;
      if (i >= count) continue;
      uint16_t* to = out + static_cast<int64_t>(i) * kCodes;
      uint2 w[kCodes / 4];
#pragma unroll
      for (int e = 0; e < kCodes / 4; ++e) w[e] = dequantize4(c[u][e], s[u]);
      if constexpr (kCodes == 16)
        store32(to, w);
      else
        *reinterpret_cast<uint4*>(to) = make_uint4(w[0].x, w[0].y, w[1].x, w[1].y);
    }
  }
}

template <int kLanes, int kElems, int kVecs, int kRows>
cudaError_t write_launch(const CacheWriteArgs& a, uint32_t* err_word, cudaStream_t st) {
  constexpr int kCtaRows = kCacheThreads / kLanes * kRows;
  const dim3 grid(static_cast<unsigned>((a.rows + kCtaRows - 1) / kCtaRows), 2);
  return launch_dependent(cache_write_kernel<kLanes, kElems, kVecs, kRows>, grid, kCacheThreads, 0, st, 0, a,
                          divider(a.heads), err_word);
}

template <int kLanes, int kElems, int kVecs = 1>
cudaError_t write_by_rows(const CacheWriteArgs& a, uint32_t* err_word, cudaStream_t st) {
  // two rows a group once that still leaves every SM two thousand threads
  if (2 * a.rows * kLanes >= static_cast<int64_t>(sm_count()) * 2048 * 2)
    return write_launch<kLanes, kElems, kVecs, 2>(a, err_word, st);
  return write_launch<kLanes, kElems, kVecs, 1>(a, err_word, st);
}

template <int kCodes>
cudaError_t read_launch(const CacheReadArgs& a, uint32_t* err_word, cudaStream_t st) {
  const int64_t per_token = static_cast<int64_t>(a.heads) * a.d / kCodes;
  // whole tokens that one pass of the CTA covers (a long token takes several passes)
  const int64_t fit = kCacheThreads * kReadUnroll / per_token;
  const int64_t span = fit < 1 ? 1 : fit;
  const dim3 grid(static_cast<unsigned>((a.max_len + span - 1) / span), static_cast<unsigned>(a.batch), 2);
  return launch_dependent(cache_read_kernel<kCodes>, grid, kCacheThreads, 0, st, 0, a, static_cast<int>(span),
                          divider(per_token), divider(a.d / kCodes), divider(a.page), err_word);
}

}  // namespace

cudaError_t launch_cache_write(const CacheWriteArgs& a, uint32_t* err_word, cudaStream_t st) {
  if (a.rows <= 0) return cudaSuccess;
  const auto at = [](const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; };
  const bool wide = a.d % 16 == 0 && at(a.k.x, 32) && at(a.v.x, 32) && at(a.k.codes, 16) &&
                    at(a.v.codes, 16) && (a.k.token_stride | a.k.head_stride | a.v.token_stride | a.v.head_stride) % 16 == 0;
  if (wide) {
    if (a.d <= 64) return write_by_rows<4, 16>(a, err_word, st);
    if (a.d <= 128) return write_by_rows<8, 16>(a, err_word, st);
    if (a.d <= 256) return write_by_rows<16, 16>(a, err_word, st);
    return write_by_rows<32, 16>(a, err_word, st);
  }
  if (a.d <= 64) return write_by_rows<8, 8>(a, err_word, st);
  if (a.d <= 128) return write_by_rows<16, 8>(a, err_word, st);
  if (a.d <= 256) return write_by_rows<32, 8>(a, err_word, st);
  return write_by_rows<32, 8, 2>(a, err_word, st);
}

cudaError_t launch_cache_read(const CacheReadArgs& a, uint32_t* err_word, cudaStream_t st) {
  if (a.max_len <= 0 || a.batch <= 0) return cudaSuccess;
  const auto at = [](const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; };
  if (a.d % 16 == 0 && at(a.k_codes, 16) && at(a.v_codes, 16) && at(a.k_out, 32) && at(a.v_out, 32))
    return read_launch<16>(a, err_word, st);
  return read_launch<8>(a, err_word, st);
}

}  // namespace fvq
