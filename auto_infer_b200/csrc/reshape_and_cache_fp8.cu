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
// A page's scale depends on all rows of the call that fall in it, so each page has one owner in
// the grid.  The slot list may be in any order and may repeat slots (the last row wins): a CTA
// walks the whole list once to number the stretches of equal pages, takes every gridDim.x-th
// stretch, and walks it again to collect the rows of that page wherever they stand; a stretch
// whose page already occurred further up belongs to an earlier owner.  Both walks read 4 bytes a
// token from L1 / L2 and run once per CTA and page, not per row.
//
// HBM-bound for prompts (256 bytes read and 128 written per row and head), latency-bound for a
// decode step.
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

constexpr int kOwnedBatch = 32;      // stretches a CTA notes per walk
constexpr int kHeldRows = 16;        // rows a half warp keeps in registers between the two passes

// One of 8 bf16 elements of a row to 8 codes; s is the page's scale, inv its reciprocal if that is exact, else 0.
__device__ __forceinline__ uint2 quantise8(const uint4& v, float s, float inv) {
  float x[8];
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float y = inv != 0.f ? x[i] * inv : x[i] / s;
    x[i] = fmaf(y, 0.f, y);          // an infinity becomes NaN, which has a code; finite values pass
  }
  return make_uint2(f32x4_to_e4m3x4(x[0], x[1], x[2], x[3]), f32x4_to_e4m3x4(x[4], x[5], x[6], x[7]));
}

// Largest magnitude among the finite elements, as bf16 bits.
__device__ __forceinline__ uint32_t top8(const uint4& v, uint32_t top) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t lo = w[i] & 0x7fffu, hi = (w[i] >> 16) & 0x7fffu;
    top = max(top, lo < 0x7f80u ? lo : 0u);
    top = max(top, hi < 0x7f80u ? hi : 0u);
  }
  return top;
}

// A CTA holds kHeads heads of a page, K and V: 2 * kHeads units of kWarps warps.
template <int kHeads, int kWarps>
__global__ void __launch_bounds__(64 * kHeads * kWarps)
reshape_and_cache_fp8_kernel(const QuantWriteParams p) {
  constexpr int kThreads = 64 * kHeads * kWarps;
  constexpr int kCtaWarps = kThreads / 32;
  extern __shared__ int page_rows[];            // [block_size] token of each row of the page, [block_size] rows written
  __shared__ int warp_sum[kCtaWarps];
  __shared__ int owned[kOwnedBatch];
  __shared__ int first_token, row_count;
  __shared__ uint32_t warp_top[kCtaWarps];
  int* const token_of = page_rows;
  int* const row_list = page_rows + p.block_size;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int unit = warp / kWarps, unit_warp = warp % kWarps;
  const int head = blockIdx.y * kHeads + (unit >> 1);
  const bool is_v = unit & 1;
  const bool live = head < p.num_kv_heads;
  grid_dep_launch();
  grid_dep_wait();

  // page of token i, or -1 for a padding row or a slot outside the cache
  auto page_of = [&](int i) -> int {
    const int slot = p.slot_mapping[i];
    return slot >= 0 && slot < p.total_slots ? slot >> p.block_shift : -1;
  };
  const int per_thread = (p.num_tokens + kThreads - 1) / kThreads;
  const int seg_lo = min(threadIdx.x * per_thread, p.num_tokens), seg_hi = min(seg_lo + per_thread, p.num_tokens);

  // ---- number the stretches: each thread counts those that start in its segment, then a block scan
  int starts = 0;
  {
    int prev = seg_lo > 0 && seg_lo < seg_hi ? page_of(seg_lo - 1) : -1;
    for (int i = seg_lo; i < seg_hi; ++i) {
      const int page = page_of(i);
      starts += page >= 0 && page != prev;
      prev = page;
      if (page < 0 && blockIdx.x == 0 && blockIdx.y == 0 && p.status && p.slot_mapping[i] >= 0)
        atomicOr(p.status, B200_STATUS_BAD_SLOT);
    }
  }
  int before = starts;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, before, d);
    if (lane >= d) before += o;
  }
  if (lane == 31) warp_sum[warp] = before;
  __syncthreads();
  int total = 0;
  before -= starts;
#pragma unroll
  for (int w = 0; w < kCtaWarps; ++w) {
    if (w < warp) before += warp_sum[w];
    total += warp_sum[w];
  }

  for (int base = blockIdx.x; base < total; base += gridDim.x * kOwnedBatch) {
    // ---- this CTA's stretches base, base + gridDim.x, ..: their first tokens
    {
      int prev = seg_lo > 0 && seg_lo < seg_hi ? page_of(seg_lo - 1) : -1;
      int rank = before;
      if (starts > 0)
        for (int i = seg_lo; i < seg_hi; ++i) {
          const int page = page_of(i);
          if (page >= 0 && page != prev) {
            const int d = rank - base;
            if (d >= 0 && d % gridDim.x == 0 && d / gridDim.x < kOwnedBatch) owned[d / gridDim.x] = i;
            ++rank;
          }
          prev = page;
        }
    }
    const int n_owned = min((total - base + (int)gridDim.x - 1) / (int)gridDim.x, kOwnedBatch);
    for (int e = 0; e < n_owned; ++e) {
      for (int r = threadIdx.x; r < p.block_size; r += kThreads) token_of[r] = -1;
      if (threadIdx.x == 0) {
        first_token = p.num_tokens;
        row_count = 0;
      }
      __syncthreads();                           // also: owned[] is written
      const int start = owned[e];
      const int page = page_of(start);
      // ---- the rows of this page, wherever they stand in the list; of equal slots the last
      for (int i = seg_lo; i < seg_hi; ++i)
        if (page_of(i) == page) {
          atomicMax(&token_of[p.slot_mapping[i] & (p.block_size - 1)], i);
          atomicMin(&first_token, i);
        }
      __syncthreads();
      const bool mine = first_token == start;    // else an earlier stretch owns the page
      if (mine)
        for (int r = threadIdx.x; r < p.block_size; r += kThreads)
          if (token_of[r] >= 0) row_list[atomicAdd(&row_count, 1)] = r;
      __syncthreads();
      if (!mine) continue;                       // the same for all threads

      // ---- pass 1: the largest magnitude; half a warp reads one row, 16 bytes a lane
      const int n_rows = row_count;
      const int half = lane >> 4, part = lane & 15;
      const int first = unit_warp * 2 + half;
      const __nv_bfloat16* src = (is_v ? p.rows[1] : p.rows[0]) + (int64_t)head * kFp8HeadDim + part * 8;
      const int64_t stride = is_v ? p.stride[1] : p.stride[0];
      uint4 held[kHeldRows];
      uint32_t top = 0;
      if (live) {
#pragma unroll
        for (int k = 0; k < kHeldRows; ++k) {
          const int i = first + k * 2 * kWarps;
          if (i < n_rows) held[k] = *reinterpret_cast<const uint4*>(src + (int64_t)token_of[row_list[i]] * stride);
        }
#pragma unroll
        for (int k = 0; k < kHeldRows; ++k)
          if (first + k * 2 * kWarps < n_rows) top = top8(held[k], top);
        for (int i = first + kHeldRows * 2 * kWarps; i < n_rows; i += 2 * kWarps)
          top = top8(*reinterpret_cast<const uint4*>(src + (int64_t)token_of[row_list[i]] * stride), top);
      }
      top = __reduce_max_sync(0xffffffffu, top);
      if (kWarps > 1) {
        if (lane == 0) warp_top[warp] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = max(top, warp_top[unit * kWarps + w]);
      }
      float* const scale_at = (is_v ? p.scale[1] : p.scale[0]) + (int64_t)page * p.num_kv_heads + head;
      float s = 0.f;
      if (live) {
        // ---- the page's scale
        const float s_old = *scale_at;
        const float s_call = fp8_scale_of(__uint_as_float(top << 16));
        const bool anew = token_of[0] >= 0 || !(s_old > 0.f && s_old < INFINITY);
        s = anew ? s_call : fmaxf(s_old, s_call);
        const float inv = (__float_as_uint(s) & 0x7fffffu) == 0 ? 1.f / s : 0.f;
        uint8_t* const rows_at = (is_v ? p.cache[1] : p.cache[0]) +
                                 ((int64_t)page * p.block_size * p.num_kv_heads + head) * kFp8HeadDim;
        const int64_t row_bytes = (int64_t)p.num_kv_heads * kFp8HeadDim;
        // ---- a grown scale: round the page's other rows to it
        if (!anew && s > s_old) {
          const float ratio = s_old / s;
          for (int r = first; r < p.block_size; r += 2 * kWarps) {
            if (token_of[r] >= 0) continue;
            uint2* at = reinterpret_cast<uint2*>(rows_at + r * row_bytes + part * 8);
            const uint2 c = *at;
            float y[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t h = e4m3x2_to_f16x2((uint16_t)((i < 2 ? c.x : c.y) >> (16 * (i & 1))));
              const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
              y[2 * i] = f.x * ratio;
              y[2 * i + 1] = f.y * ratio;
            }
            *at = make_uint2(f32x4_to_e4m3x4(y[0], y[1], y[2], y[3]), f32x4_to_e4m3x4(y[4], y[5], y[6], y[7]));
          }
        }
        // ---- pass 2: the codes
#pragma unroll
        for (int k = 0; k < kHeldRows; ++k) {
          const int i = first + k * 2 * kWarps;
          if (i < n_rows) *reinterpret_cast<uint2*>(rows_at + row_list[i] * row_bytes + part * 8) = quantise8(held[k], s, inv);
        }
        for (int i = first + kHeldRows * 2 * kWarps; i < n_rows; i += 2 * kWarps) {
          const uint4 v = *reinterpret_cast<const uint4*>(src + (int64_t)token_of[row_list[i]] * stride);
          *reinterpret_cast<uint2*>(rows_at + row_list[i] * row_bytes + part * 8) = quantise8(v, s, inv);
        }
      }
      __syncthreads();                           // every warp has read the old scale, and the row lists are done with
      if (live && unit_warp == 0 && lane == 0) *scale_at = s;
    }
    __syncthreads();                             // owned[] may be written again
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
  const size_t smem = 2 * sizeof(int) * (size_t)block_size;
  // A CTA takes about 128 rows of a head pair whatever the page size: small pages share a CTA
  // among heads, so that the walks over the slot list are paid per 64 KB of rows.
  auto run = [&](auto kernel, int heads, int warps) {
    const int head_groups = (num_kv_heads + heads - 1) / heads;
    int ctas = 8 * sms / head_groups;
    ctas = ctas < 1 ? 1 : ctas;
    ctas = num_tokens < ctas ? num_tokens : ctas;
    return check_cuda(launch_pdl(kernel, dim3(ctas, head_groups), dim3(64 * heads * warps), smem,
                                 static_cast<cudaStream_t>(stream), p),
                      "reshape_and_cache_fp8 launch");
  };
  if (block_size >= 128) return run(reshape_and_cache_fp8_kernel<1, 4>, 1, 4);
  if (block_size == 64) return run(reshape_and_cache_fp8_kernel<2, 2>, 2, 2);
  if (block_size == 32) return run(reshape_and_cache_fp8_kernel<4, 1>, 4, 1);
  return run(reshape_and_cache_fp8_kernel<8, 1>, 8, 1);
}
