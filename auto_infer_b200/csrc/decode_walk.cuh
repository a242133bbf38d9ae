// What the split-KV GQA decode kernels (16-bit and 8-bit caches) share: the walk over a CTA's work
// items and the merge of the partial records of the pairs that were cut.
#pragma once
#include "common.cuh"
#include "decode_plan.h"

namespace b200 {

constexpr int kHeadDim = 128;
constexpr int kRecFloats = kMaxRows * kHeadDim + kMaxRows;   // partial record: o (16 x 128), then lse (16)

#ifdef __CUDACC__
// Walks the CTA's (item, tile) sequence; identical in producer and consumers.
struct TileWalker {
  const DecodeItem* items;
  int item, item_end, tile, tile_end;
  DecodeItem cur;
  __device__ __forceinline__ void set(const int4& a, const int4& b, const int4& c) {
    cur.seq = a.x; cur.kv_head = a.y; cur.tile_begin = a.z; cur.tile_end = a.w;
    cur.kv_len = b.x; cur.q_start = b.y; cur.q_len = b.z; cur.causal_base = b.w;
    cur.partial_idx = c.x; cur.direct = c.y; cur.multi_idx = c.z;
    tile = cur.tile_begin;
    tile_end = cur.tile_end;
  }
  __device__ __forceinline__ void load() {
    if (item < item_end) {
      const int4* p = reinterpret_cast<const int4*>(items + item);
      set(__ldg(p), __ldg(p + 1), __ldg(p + 2));
    }
  }
};

// Merge of the partial records of the cut pairs a CTA has noted, by its 256 consumer
// threads: thread -> (row, 8 columns) of the pair's 16 x 128 result.  Records are read
// with L2 loads (other CTAs wrote them) in record order, so the sum does not depend on
// which CTA happens to run the merge.
// `Params` is the launch parameters of the kernel that wrote the records.
template <typename Params>
__device__ __forceinline__ void merge_noted_pairs(const Params& p, const int* list, int count, int off_multi) {
  const int t = threadIdx.x;
  const int row = t >> 4;
  const int col = (t & 15) * 8;
  const int G = p.group;
  for (int e = 0; e < count; ++e) {
    const MultiGroup* mg = reinterpret_cast<const MultiGroup*>(p.plan + off_multi) + list[e];
    const int pb = __ldcg(&mg->part_begin), pe = __ldcg(&mg->part_end);
    const int q_start = __ldcg(&mg->q_start), q_len = __ldcg(&mg->q_len), kv_head = __ldcg(&mg->kv_head);
    if (row >= q_len * G) continue;
    const float* rec = p.part + (int64_t)pb * kRecFloats;
    const int n = pe - pb;
    float mx = -INFINITY;
#pragma unroll 4
    for (int i = 0; i < n; ++i) mx = fmaxf(mx, __ldcg(rec + (int64_t)i * kRecFloats + kMaxRows * kHeadDim + row));
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    float wsum = 0.f;
#pragma unroll 4
    for (int i = 0; i < n; ++i) {
      const float* r = rec + (int64_t)i * kRecFloats;
      const float l = __ldcg(r + kMaxRows * kHeadDim + row);
      const float wgt = (l == -INFINITY) ? 0.f : __expf(l - mx);
      const float4* src = reinterpret_cast<const float4*>(r + row * kHeadDim + col);
      const float4 a = __ldcg(src), b = __ldcg(src + 1);
      wsum += wgt;
      acc[0] += wgt * a.x; acc[1] += wgt * a.y; acc[2] += wgt * a.z; acc[3] += wgt * a.w;
      acc[4] += wgt * b.x; acc[5] += wgt * b.y; acc[6] += wgt * b.z; acc[7] += wgt * b.w;
    }
    const float inv = wsum == 0.f ? 0.f : 1.f / wsum;        // a NaN sum (8-bit cache: a NaN lse) stays one
    const int64_t tok = q_start + row / G;
    const int head = kv_head * G + row % G;
    const int64_t off = (tok * p.num_q_heads + head) * kHeadDim + col;
    if (p.out_is_f32) {
      float* dst = reinterpret_cast<float*>(p.out) + off;
      *reinterpret_cast<float4*>(dst) = make_float4(acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
      *reinterpret_cast<float4*>(dst + 4) = make_float4(acc[4] * inv, acc[5] * inv, acc[6] * inv, acc[7] * inv);
    } else {
      uint4 pk;
      pk.x = pack_bf16(acc[0] * inv, acc[1] * inv); pk.y = pack_bf16(acc[2] * inv, acc[3] * inv);
      pk.z = pack_bf16(acc[4] * inv, acc[5] * inv); pk.w = pack_bf16(acc[6] * inv, acc[7] * inv);
      *reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(p.out) + off) = pk;
    }
    if (p.lse_out && (t & 15) == 0)
      p.lse_out[tok * p.num_q_heads + head] = wsum == 0.f ? -INFINITY : mx + __logf(wsum);
  }
}
#endif  // __CUDACC__
}  // namespace b200
