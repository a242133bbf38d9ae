// Conversions and scales of the 8-bit paged cache: K and V are held as e4m3 codes with one fp32
// scale per (page, kv head), value = code * scale.
//
// The scales the slot write chooses are powers of two.  An e4m3 code has four significant bits
// whatever its exponent, so a finer scale would not store a value better (only codes below 2^-6
// have fewer bits); a power of two makes every product and quotient with a scale exact, and a
// page whose scale grows keeps its codes' mantissas.
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"

namespace b200 {

constexpr int kFp8HeadDim = 128;           // one row of codes: 128 bytes, one swizzle span
constexpr int kFp8MaxBlockSize = 1024;     // the slot write keeps one word per row of a page in shared memory
constexpr int kFp8MinBlockSize = 16;       // the 16 tokens a warp takes from a tile lie in one page

// Checks shared by the entry points over an 8-bit cache.
int check_fp8_cache(const char* who, const void* key_cache, const void* value_cache, const float* key_scale,
                    const float* value_scale, int num_blocks, int block_size, int num_kv_heads, int head_dim);

// 4-D tiled tensor map over an 8-bit paged cache (num_blocks, block_size, heads, 128): the box is
// box_tokens rows of one head, 128 bytes each, under the 128-byte swizzle.
int get_fp8_cache_tensor_map(const void* cache, int num_blocks, int block_size, int heads, int box_tokens,
                             CUtensorMap* out);

#ifdef __CUDACC__

// Two codes (low, high byte) to two f16: exact, f16 has more exponent and mantissa bits.
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint16_t codes) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(codes));
  return h;
}

// Four floats to four codes (first in the lowest byte), round to nearest even.
__device__ __forceinline__ uint32_t f32x4_to_e4m3x4(float a, float b, float c, float d) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\t"
      "mov.b32 %0, {lo, hi};\n\t}"
      : "=r"(r)
      : "f"(a), "f"(b), "f"(c), "f"(d));
  return r;
}

// Two f16 to two codes (low half in the low byte), round to nearest even.
__device__ __forceinline__ uint16_t f16x2_to_e4m3x2(uint32_t h) {
  uint16_t codes;
  asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(codes) : "r"(h));
  return codes;
}

// Smallest power of two s >= 2^-126 with a <= 448 * s, for a finite a >= 0.  448 = 1.75 * 2^8, so
// with a = m * 2^e, 1 <= m < 2, the exponent is e - 8, or e - 7 when m > 1.75.
__device__ __forceinline__ float fp8_scale_of(float a) {
  const uint32_t bits = __float_as_uint(a);
  int k = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  k = k < -126 ? -126 : k;
  return __uint_as_float((uint32_t)(k + 127) << 23);
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float fast_log2(float x) {
  float y;
  asm("lg2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 4-byte copy to shared memory; zero when `have` is false (nothing is read then).
__device__ __forceinline__ void cp_async_f32(float* dst, const float* src, bool have) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(have ? 4 : 0) : "memory");
}
// Waits for a phase that completes by itself, of copies or matrix products that are under way, whatever the CTA's abort flag
// says: a CTA that gives up must not leave while they write to its memory.  At most 2^20 tries of a microsecond or so.
__device__ __forceinline__ void mbar_wait_landed(uint64_t* bar, uint32_t parity) {
#pragma unroll 1
  for (uint32_t left = 1u << 20; left && !mbar_try_wait(bar, parity); --left) {
  }
}
// One of the barrier's expected arrivals, made when this thread's cp.async copies so far have landed.
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

#endif  // __CUDACC__
}  // namespace b200
