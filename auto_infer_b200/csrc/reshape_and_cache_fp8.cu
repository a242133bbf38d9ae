// Slot write into an 8-bit paged cache: new K / V rows become e4m3 codes under one scale per
// (page, kv head).
//
// Per page p, head h, and K and V apart, with R the rows this call writes to p:
//   a      = max |x| over the finite elements of R
//   s_call = smallest power of two with a <= 448 * s_call (at least 2^-126)
//   s      = s_call                  when the call writes the page's first row (the page starts
//                                    anew) or the old scale is not a positive finite number
//            max(s_old, s_call)      otherwise; when that grows, the page's other rows are
//                                    re-rounded: c' = e4m3(c * s_old / s)
//   row    c = e4m3(x / s), ties to even; infinities and NaN become the NaN code.
// Tokens step through a page in order, so a write of its first row can only mean a new owner; the
// rows the old owner left carry no meaning and are not touched.
//
// A page's scale depends on all rows of the call that fall in it, so each page has one owner in the grid.  The
// slot list may be in any order and may repeat slots (the last row wins): where the page changes from one token to
// the next, token i belongs to CTA i mod gridDim.x, which walks the whole list to collect the rows of that page
// wherever they stand; if the page occurs further up, an earlier token's CTA does.  gridDim.x is odd and pages are
// powers of two, so the page starts of a long prompt (every block_size tokens) and the neighbouring tokens of a
// decode step both spread evenly.  The walk reads 4 bytes a token from L2, eight tokens a thread in flight.
//
// A CTA of 16 warps takes up to 16 such pages at a time: one walk collects the rows of all of them, then each warp
// takes whole (page, head, K / V) units of the pages with at most 16 rows (decode rows: many pages, a row or two
// each; taken one after the other by the whole CTA they cost 5 us a page), and then all warps together the pages
// with more.  For those the CTA has about 128 rows of a head pair whatever the page size, small pages several heads
// at once.  Rows stay in registers between the two passes, magnitudes and codes (read again for the second, from L1:
// 11.4 us instead of 9.7 on a 2048-token chunk).
//
// HBM-bound for prompts (256 bytes read and 128 written per row and head), latency-bound for a decode step.  Measured,
// 8 heads: 4.1 us for 16 decode rows (a launch and five dependent trips to memory), 12.2 us for 60 decode rows and four
// 512-token chunks (13 MB; 2 us of HBM: the walk and its barriers come before any row is loaded, and all CTAs are in it at
// once), 14.8 us for 8191 tokens in pages of 16 (50 MB, 3.4 TB/s), 53 us for 32768 (floor 31: each CTA walks the list once
// per 16 pages).  Re-rounding: 60 rows that raise every scale of pages of 128 take 22.6 us, 4.8 where the scales stay.
#include "fp8.cuh"

namespace b200 {

struct QuantWriteParams {
  const __nv_bfloat16* rows[2];      // key, value: (T, Hkv, 128), heads contiguous
  int64_t stride[2];                 // elements between tokens
  uint8_t* cache[2];
  float* scale[2];
  const int32_t* slot_mapping;
  int num_tokens, num_kv_heads;
  int block_size, block_shift;
  int64_t total_slots;
  int32_t* status;
};

constexpr int kWriteThreads = 512;
constexpr int kShortRows = 16;       // a page with at most this many new rows is one warp's per head and K / V
constexpr int kMaxBatch = 16;        // pages a CTA collects at once,
constexpr int kBatchRows = 2048;     // and at most this many rows of theirs
constexpr int kWalk = 8;             // tokens a thread looks up at a time: their loads are in flight together

// Largest magnitude of 8 bf16 elements as two 16-bit halves, infinities and NaN included (they compare largest).
__device__ __forceinline__ uint32_t top8(const uint4& v, uint32_t top) {
  top = __vmaxu2(top, v.x & 0x7fff7fffu);
  top = __vmaxu2(top, v.y & 0x7fff7fffu);
  top = __vmaxu2(top, v.z & 0x7fff7fffu);
  return __vmaxu2(top, v.w & 0x7fff7fffu);
}
// The same without the elements that are not finite.
__device__ __forceinline__ uint32_t finite_top8(const uint4& v, uint32_t top) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t u = w[i] & 0x7fff7fffu;
    if ((u & 0xffffu) >= 0x7f80u) u &= 0xffff0000u;
    if ((u >> 16) >= 0x7f80u) u &= 0xffffu;
    top = __vmaxu2(top, u);
  }
  return top;
}

// 8 bf16 elements of a row, all finite, to 8 codes under a power-of-two scale with reciprocal inv.
__device__ __forceinline__ uint2 quantise8(const uint4& v, float inv) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  float x[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16) * inv;
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u) * inv;
  }
  return make_uint2(f32x4_to_e4m3x4(x[0], x[1], x[2], x[3]), f32x4_to_e4m3x4(x[4], x[5], x[6], x[7]));
}
// The same for any elements under any scale.
__device__ __forceinline__ uint2 quantise8_any(const uint4& v, float s) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  float x[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16) / s;
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u) / s;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = fmaf(x[i], 0.f, x[i]);    // an infinity becomes NaN, which has a code
  return make_uint2(f32x4_to_e4m3x4(x[0], x[1], x[2], x[3]), f32x4_to_e4m3x4(x[4], x[5], x[6], x[7]));
}

// 8 codes times ratio, rounded to codes again.
__device__ __forceinline__ uint2 rescale8(const uint2& c, float ratio) {
  float y[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t h = e4m3x2_to_f16x2((uint16_t)((i < 2 ? c.x : c.y) >> (16 * (i & 1))));
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    y[2 * i] = f.x * ratio;
    y[2 * i + 1] = f.y * ratio;
  }
  return make_uint2(f32x4_to_e4m3x4(y[0], y[1], y[2], y[3]), f32x4_to_e4m3x4(y[4], y[5], y[6], y[7]));
}

// A page's new scale: what the call asks for when the page starts anew, else the larger of that and the old one.
struct PageScale {
  float s, inv;                // inv: 1 / s if that is exact and all elements are finite, else 0
  float ratio;                 // what the page's other rows are multiplied by (0: too small for fp32), -1 when they stay
  __device__ __forceinline__ PageScale(uint32_t top, float s_old, bool first_row_written, bool all_finite) {
    const float s_call = fp8_scale_of(__uint_as_float(top << 16));
    const bool anew = first_row_written || !(s_old > 0.f && s_old < INFINITY);
    s = anew ? s_call : fmaxf(s_old, s_call);
    inv = all_finite && (__float_as_uint(s) & 0x7fffffu) == 0 ? 1.f / s : 0.f;
    ratio = !anew && s > s_old ? s_old / s : -1.f;
  }
};
__device__ __forceinline__ uint32_t larger_half(uint32_t top) { return max(top & 0xffffu, top >> 16); }

// A CTA holds kHeads heads of a page, K and V: 2 * kHeads units of kWarps warps.
template <int kHeads>
__global__ void __launch_bounds__(kWriteThreads, 2)
reshape_and_cache_fp8_kernel(const QuantWriteParams p) {
  constexpr int kCtaWarps = kWriteThreads / 32;
  constexpr int kWarps = kCtaWarps / (2 * kHeads);
  constexpr int kStep = 2 * kWarps;             // rows a unit covers at a time, half a warp each
  extern __shared__ int page_rows[];            // [batch][block_size]: the token that writes a row of the page, or -1
  __shared__ int owned[kWriteThreads];
  __shared__ int n_owned, page_at[kMaxBatch], start_at[kMaxBatch], first_token[kMaxBatch], row_count[kMaxBatch];
  __shared__ int2 row_list[kMaxBatch][kShortRows];              // (token, row) of a page with few, superseded ones too
  __shared__ uint32_t warp_top[2][kCtaWarps];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int half = lane >> 4, part = lane & 15;                 // half a warp reads one row, 16 bytes a lane
  const int batch = min(kMaxBatch, kBatchRows >> p.block_shift);
  const int row_mask = p.block_size - 1;
  if (tid == 0) n_owned = 0;
  grid_dep_launch();
  grid_dep_wait();
  __syncthreads();

  // page of a slot, or -1 for a padding row or a slot outside the cache
  auto page_of = [&](int slot) -> int { return slot >= 0 && slot < p.total_slots ? slot >> p.block_shift : -1; };

  // this CTA's tokens, 512 at a time: those whose page is not their predecessor's
  for (int64_t base = blockIdx.x; base < p.num_tokens; base += (int64_t)kWriteThreads * gridDim.x) {
    const int64_t mine = base + (int64_t)tid * gridDim.x;
    if (mine < p.num_tokens) {
      const int slot = p.slot_mapping[mine], before = mine > 0 ? p.slot_mapping[mine - 1] : -1;
      const int page = page_of(slot);
      if (page < 0 && slot >= 0 && blockIdx.y == 0 && p.status) atomicOr(p.status, B200_STATUS_BAD_SLOT);
      if (page >= 0 && page != page_of(before)) owned[atomicAdd(&n_owned, 1)] = (int)mine;
    }
    __syncthreads();
    const int n = n_owned;
    for (int e0 = 0; e0 < n; e0 += batch) {
      const int nb = min(batch, n - e0);
      for (int r = tid; r < nb << p.block_shift; r += kWriteThreads) page_rows[r] = -1;
      if (tid < nb) {
        const int start = owned[e0 + tid];
        start_at[tid] = start;
        page_at[tid] = p.slot_mapping[start] >> p.block_shift;
        first_token[tid] = p.num_tokens;
        row_count[tid] = 0;
      }
      __syncthreads();
      // ---- the rows of these pages, wherever they stand in the list; of equal slots the last
      for (int i0 = 0; i0 < p.num_tokens; i0 += kWalk * kWriteThreads) {
        int slot_at[kWalk];
#pragma unroll
        for (int k = 0; k < kWalk; ++k) {
          const int i = i0 + k * kWriteThreads + tid;
          slot_at[k] = i < p.num_tokens ? p.slot_mapping[i] : -1;
        }
        uint32_t found = 0;                        // which of them lie in one of the pages
        for (int e = 0; e < nb; ++e) {
          const uint32_t first_slot = (uint32_t)page_at[e] << p.block_shift;
#pragma unroll
          for (int k = 0; k < kWalk; ++k) found |= ((slot_at[k] ^ first_slot) < (uint32_t)p.block_size ? 1u : 0u) << k;
        }
        uint32_t todo = __reduce_or_sync(0xffffffffu, found);
        while (todo) {
          const int c = __ffs(todo) - 1;
          todo &= todo - 1;
          const int i = i0 + c * kWriteThreads + tid;
          int hit = -1, slot = -1;
          if (found >> c & 1u) {
            slot = p.slot_mapping[i];
            for (int e = 0; e < nb; ++e)           // of two stretches of one page the earlier
              if (slot >> p.block_shift == page_at[e] && (hit < 0 || start_at[e] < start_at[hit])) hit = e;
          }
          const uint32_t hits = __ballot_sync(0xffffffffu, hit >= 0);
          if (hit < 0) continue;
          atomicMax(&page_rows[(hit << p.block_shift) + (slot & row_mask)], i);
          // one counter update for the lanes that share a page
          const uint32_t same = __match_any_sync(hits, hit);
          const int leader = __ffs(same) - 1, rank = __popc(same & ((1u << lane) - 1));
          int entry = 0;
          if (lane == leader) {
            entry = atomicAdd(&row_count[hit], __popc(same));
            atomicMin(&first_token[hit], i);
          }
          entry = __shfl_sync(same, entry, leader) + rank;
          if (entry < kShortRows) row_list[hit][entry] = make_int2(i, slot & row_mask);
        }
      }
      __syncthreads();

      // ---- pages with few rows: a warp each per head and K / V
      for (int u = warp; u < nb * 2 * kHeads; u += kCtaWarps) {
        const int e = u / (2 * kHeads), head = blockIdx.y * kHeads + ((u >> 1) % kHeads);
        const bool is_v = u & 1;
        const int count = row_count[e];
        // a page that occurs before this stretch has its owner there
        if (count > kShortRows || first_token[e] != start_at[e] || head >= p.num_kv_heads) continue;
        const int* const token_of = page_rows + (e << p.block_shift);
        const int page = page_at[e];
        float* const scale_at = (is_v ? p.scale[1] : p.scale[0]) + (int64_t)page * p.num_kv_heads + head;
        const __nv_bfloat16* src = (is_v ? p.rows[1] : p.rows[0]) + (int64_t)head * kFp8HeadDim + part * 8;
        const int64_t stride = is_v ? p.stride[1] : p.stride[0];
        const float s_old = *scale_at;
        uint4 held[kShortRows / 2];                // this half warp's rows, and where they go (-1: none, or superseded)
        int row[kShortRows / 2];
        uint32_t top = 0;
#pragma unroll
        for (int k = 0; k < kShortRows / 2; ++k) {
          held[k] = make_uint4(0u, 0u, 0u, 0u);
          row[k] = -1;
          if (half + 2 * k < count) {
            const int2 at = row_list[e][half + 2 * k];
            if (token_of[at.y] == at.x) {
              row[k] = at.y;
              held[k] = *reinterpret_cast<const uint4*>(src + (int64_t)at.x * stride);
            }
          }
        }
#pragma unroll
        for (int k = 0; k < kShortRows / 2; ++k) top = top8(held[k], top);
        top = __reduce_max_sync(0xffffffffu, larger_half(top));
        const bool plain = top < 0x7f80u;
        if (!plain) {
          top = 0;
#pragma unroll 1
          for (int j = half; j < count; j += 2) {
            const int2 at = row_list[e][j];
            if (token_of[at.y] == at.x)
              top = finite_top8(*reinterpret_cast<const uint4*>(src + (int64_t)at.x * stride), top);
          }
          top = __reduce_max_sync(0xffffffffu, larger_half(top));
        }
        const PageScale ps(top, s_old, token_of[0] >= 0, plain);
        __syncwarp();                              // all lanes have read the old scale: a reduction orders no memory
        if (lane == 0) *scale_at = ps.s;
        uint8_t* const rows_at = (is_v ? p.cache[1] : p.cache[0]) +
                                 ((int64_t)page * p.block_size * p.num_kv_heads + head) * kFp8HeadDim + part * 8;
        const int64_t row_bytes = (int64_t)p.num_kv_heads * kFp8HeadDim;
        if (ps.inv != 0.f) {
#pragma unroll
          for (int k = 0; k < kShortRows / 2; ++k)
            if (row[k] >= 0) *reinterpret_cast<uint2*>(rows_at + row[k] * row_bytes) = quantise8(held[k], ps.inv);
        } else {
#pragma unroll 1
          for (int j = half; j < count; j += 2) {
            const int2 at = row_list[e][j];
            if (token_of[at.y] == at.x)
              *reinterpret_cast<uint2*>(rows_at + at.y * row_bytes) =
                  quantise8_any(*reinterpret_cast<const uint4*>(src + (int64_t)at.x * stride), ps.s);
          }
        }
        if (ps.ratio >= 0.f)                       // a grown scale: round the page's other rows to it
#pragma unroll 1
          for (int r = half; r < p.block_size; r += 2)
            if (token_of[r] < 0) {
              uint2* at = reinterpret_cast<uint2*>(rows_at + r * row_bytes);
              *at = rescale8(*at, ps.ratio);
            }
      }

      // ---- pages with many: all warps
      int turn = 0;
      for (int e = 0; e < nb; ++e) {
        if (row_count[e] <= kShortRows || first_token[e] != start_at[e]) continue;      // the same for all threads
        const int unit = warp / kWarps, unit_warp = warp % kWarps;
        const int head = blockIdx.y * kHeads + (unit >> 1);
        const bool is_v = unit & 1, live = head < p.num_kv_heads;
        const int first = live ? unit_warp * 2 + half : p.block_size;
        const int* const token_of = page_rows + (e << p.block_shift);
        const int page = page_at[e];
        float* const scale_at = (is_v ? p.scale[1] : p.scale[0]) + (int64_t)page * p.num_kv_heads + head;
        const __nv_bfloat16* src = (is_v ? p.rows[1] : p.rows[0]) + (int64_t)head * kFp8HeadDim + part * 8;
        const int64_t stride = is_v ? p.stride[1] : p.stride[0];
        const float s_old = live ? *scale_at : 0.f;
        uint4 held[kShortRows / 2];                // the first rows; those of pages over 128 rows are read again
        uint32_t top = 0;
#pragma unroll
        for (int k = 0; k < kShortRows / 2; ++k) {
          const int r = first + k * kStep, i = r < p.block_size ? token_of[r] : -1;
          held[k] = make_uint4(0u, 0u, 0u, 0u);
          if (i >= 0) held[k] = *reinterpret_cast<const uint4*>(src + (int64_t)i * stride);
        }
#pragma unroll
        for (int k = 0; k < kShortRows / 2; ++k) top = top8(held[k], top);
#pragma unroll 1
        for (int r = first + kShortRows / 2 * kStep; r < p.block_size; r += kStep) {
          const int i = token_of[r];
          if (i >= 0) top = top8(*reinterpret_cast<const uint4*>(src + (int64_t)i * stride), top);
        }
        // The unit's largest, over its warps.  The barrier is also what lets one warp replace the scale that all have
        // read; the two slots keep a page's values apart from the next's.
        auto unit_top = [&](uint32_t t) -> uint32_t {
          t = __reduce_max_sync(0xffffffffu, larger_half(t));
          if (lane == 0) warp_top[turn][warp] = t;
          const bool odd = __syncthreads_or(t >= 0x7f80u);
          for (int w = 0; w < kWarps; ++w) t = max(t, warp_top[turn][unit * kWarps + w]);
          turn ^= 1;
          return odd ? t | 0x80000000u : t;
        };
        top = unit_top(top);
        const bool plain = top < 0x80000000u;      // no element of the CTA's page is infinite or NaN
        if (!plain) {
          top = 0;
#pragma unroll 1
          for (int r = first; r < p.block_size; r += kStep)
            if (token_of[r] >= 0) top = finite_top8(*reinterpret_cast<const uint4*>(src + (int64_t)token_of[r] * stride), top);
          top = unit_top(top);
        }
        const PageScale ps(top, s_old, token_of[0] >= 0, plain);
        if (live && unit_warp == 0 && lane == 0) *scale_at = ps.s;
        uint8_t* const rows_at = (is_v ? p.cache[1] : p.cache[0]) +
                                 ((int64_t)page * p.block_size * p.num_kv_heads + head) * kFp8HeadDim + part * 8;
        const int64_t row_bytes = (int64_t)p.num_kv_heads * kFp8HeadDim;
        if (ps.inv != 0.f) {
#pragma unroll
          for (int k = 0; k < kShortRows / 2; ++k) {
            const int r = first + k * kStep;
            if (r < p.block_size && token_of[r] >= 0)
              *reinterpret_cast<uint2*>(rows_at + r * row_bytes) = quantise8(held[k], ps.inv);
          }
#pragma unroll 1
          for (int r = first + kShortRows / 2 * kStep; r < p.block_size; r += kStep) {
            const int i = token_of[r];
            if (i >= 0)
              *reinterpret_cast<uint2*>(rows_at + r * row_bytes) =
                  quantise8(*reinterpret_cast<const uint4*>(src + (int64_t)i * stride), ps.inv);
          }
        } else {
#pragma unroll 1
          for (int r = first; r < p.block_size; r += kStep)
            if (token_of[r] >= 0)
              *reinterpret_cast<uint2*>(rows_at + r * row_bytes) =
                  quantise8_any(*reinterpret_cast<const uint4*>(src + (int64_t)token_of[r] * stride), ps.s);
        }
        if (ps.ratio >= 0.f)
#pragma unroll 1
          for (int r = first; r < p.block_size; r += kStep)
            if (token_of[r] < 0) {
              uint2* at = reinterpret_cast<uint2*>(rows_at + r * row_bytes);
              *at = rescale8(*at, ps.ratio);
            }
      }
      __syncthreads();                           // the batch's arrays may be written again
    }
    if (tid == 0) n_owned = 0;
    __syncthreads();
  }
}

int check_fp8_cache(const char* who, const void* key_cache, const void* value_cache, const float* key_scale,
                    const float* value_scale, int num_blocks, int block_size, int num_kv_heads, int head_dim) {
  if (!key_cache || !value_cache || !key_scale || !value_scale || num_blocks <= 0 || num_kv_heads <= 0) {
    set_last_error("%s: null cache or scale pointer, or non-positive size", who);
    return B200_EINVAL;
  }
  if (head_dim != kFp8HeadDim) {
    set_last_error("%s: head_dim %d unsupported (kernel is built for 128)", who, head_dim);
    return B200_EUNSUPPORTED;
  }
  if (block_size < kFp8MinBlockSize || block_size > kFp8MaxBlockSize || (block_size & (block_size - 1))) {
    set_last_error("%s: block_size %d must be a power of two from 16 to 1024", who, block_size);
    return B200_EUNSUPPORTED;
  }
  if ((int64_t)num_blocks * block_size > INT32_MAX) {
    set_last_error("%s: %d blocks of %d rows exceed the int32 slots", who, num_blocks, block_size);
    return B200_ETOOLARGE;
  }
  if (reinterpret_cast<uintptr_t>(key_cache) % 16 || reinterpret_cast<uintptr_t>(value_cache) % 16 ||
      reinterpret_cast<uintptr_t>(key_scale) % 4 || reinterpret_cast<uintptr_t>(value_scale) % 4) {
    set_last_error("%s: caches must be 16-byte aligned and scales 4-byte aligned", who);
    return B200_EALIGN;
  }
  return B200_OK;
}

}  // namespace b200

extern "C" int b200_reshape_and_cache_fp8(const void* key, int64_t key_stride, const void* value, int64_t value_stride,
                                          void* key_cache, void* value_cache, float* key_scale, float* value_scale,
                                          const int32_t* slot_mapping, int num_tokens, int num_kv_heads, int head_dim,
                                          int block_size, int num_blocks, int32_t* status, void* stream) {
  using namespace b200;
  const char* who = "reshape_and_cache_fp8";
  int rc = check_fp8_cache(who, key_cache, value_cache, key_scale, value_scale, num_blocks, block_size, num_kv_heads,
                           head_dim);
  if (rc) return rc;
  if (num_tokens == 0) return B200_OK;
  if (!key || !value || !slot_mapping || num_tokens < 0) {
    set_last_error("%s: null pointer or negative token count", who);
    return B200_EINVAL;
  }
  const int64_t row = (int64_t)num_kv_heads * head_dim;
  if (key_stride < row || value_stride < row) {
    set_last_error("%s: token stride smaller than a row", who);
    return B200_EINVAL;
  }
  if (reinterpret_cast<uintptr_t>(key) % 16 || reinterpret_cast<uintptr_t>(value) % 16 || key_stride % 8 ||
      value_stride % 8 || reinterpret_cast<uintptr_t>(slot_mapping) % 4) {
    set_last_error("%s: rows must be 16-byte aligned with token strides that are multiples of 8 elements", who);
    return B200_EALIGN;
  }
  QuantWriteParams p;
  p.rows[0] = static_cast<const __nv_bfloat16*>(key);
  p.rows[1] = static_cast<const __nv_bfloat16*>(value);
  p.stride[0] = key_stride;
  p.stride[1] = value_stride;
  p.cache[0] = static_cast<uint8_t*>(key_cache);
  p.cache[1] = static_cast<uint8_t*>(value_cache);
  p.scale[0] = key_scale;
  p.scale[1] = value_scale;
  p.slot_mapping = slot_mapping;
  p.num_tokens = num_tokens;
  p.num_kv_heads = num_kv_heads;
  p.block_size = block_size;
  p.block_shift = __builtin_ctz(block_size);
  p.total_slots = (int64_t)num_blocks * block_size;
  p.status = status;
  int sms = b200_sm_count();
  if (sms <= 0) sms = 148;
  const size_t smem = sizeof(int) * (size_t)kBatchRows;
  // Heads of a CTA: as many as make about 128 rows of a page, at most the heads there are.  gridDim.x is odd (see
  // above), and all CTAs fit on the device at once, two per SM.
  int heads = 1;
  while (heads < 8 && heads * block_size < 128 && heads < num_kv_heads) heads *= 2;
  const int head_groups = (num_kv_heads + heads - 1) / heads;
  int ctas = (2 * sms / head_groups - 1) | 1;
  ctas = ctas < 1 ? 1 : ctas;
  ctas = num_tokens < ctas ? num_tokens | 1 : ctas;
  auto kernel = heads == 1 ? reshape_and_cache_fp8_kernel<1> : heads == 2 ? reshape_and_cache_fp8_kernel<2>
              : heads == 4 ? reshape_and_cache_fp8_kernel<4> : reshape_and_cache_fp8_kernel<8>;
  return check_cuda(launch_pdl(kernel, dim3(ctas, head_groups), dim3(kWriteThreads), smem,
                               static_cast<cudaStream_t>(stream), p),
                    "reshape_and_cache_fp8 launch");
}
