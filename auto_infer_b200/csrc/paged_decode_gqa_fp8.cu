// Split-KV paged GQA decode / MTP-verify attention over an 8-bit cache, for sm_100a.
//
//   o = sum_j softmax_j(scale * q . (ck_j s_k)) * (cv_j s_v)
//
// with e4m3 codes ck, cv and one scale per (page, kv head), K and V apart.  HBM-bound: a cached
// token costs 2 * 128 bytes per kv head, half of the 16-bit cache, so an SM has half the time per
// token for the same arithmetic.
//
// The plan, the work items, the TMA ring and the merge of cut pairs are those of the 16-bit kernel
// (one persistent CTA per SM, producer warps, eight consumer warps).  What differs:
//   * both products are transposed, S^T = K Q^T and O^T = V^T P^T: the 16 rows of an mma.sync m16n8k16 are
//     tokens (then columns of V), its 8 columns the query rows.  A decode step of most models has at most 8
//     (q_len * group), and the form with the query as A would spend half of every instruction on padding;
//     9 to 16 rows take two column tiles.
//   * codes become f16 on their way from shared memory to the MMA: e4m3 -> f16 is exact and one instruction per
//     pair.  Q (bf16) is scaled per row by a power of two so that it fits f16 exactly, and the weights P are f16
//     too, three bits more than bf16 over the range that counts (below).  (The e4m3 form of mma.sync converts in the same way on this part: 20 cycles a
//     scheduler for 32 x 8 codes, two f16 MMAs take 16.)
//   * no element is multiplied by a scale.  K's scale is uniform over 16 tokens (the least a page holds) and goes
//     into the factor that turns a product into a log2 score.  V's scale goes into the weight,
//     w = 2^(x + log2 s_v - M): M is the running maximum of x + log2 s_v, kept beside the running maximum m of
//     the scores x that the row sum l refers to, and the P of the product is 2^15 w.  So P fits f16 whatever the pages'
//     scales are, the largest contributions have the most bits, and those down to 2^-29 of them lose none: many small
//     weights beside one key that carries the row (and may have a V of zeros) add up to what they should.  O is in units
//     of 2^(M - 15) and is brought to l's 2^m when the row is written.
//   * M only has to be common to the eight lanes that hold a row; a vote finds the tiles that raise it, all others
//     pass without a shuffle.  m is each lane's own until the end.
//   * the order of the 16 dims of a k-step, and which column of V an O^T row stands for, are free as long as both
//     operands and the output use the same, and are taken so that ldmatrix delivers K's codes in place and V's after
//     one byte permute per register.
//   * the scales of a tile's pages ride with the tile: 4-byte cp.async copies that complete on the stage's barrier.
//   * a tile has half the bytes, so a producer has half the time for it: one warp took 1090 cycles a tile, where
//     HBM delivers one in 700.  Each consumer group has a producer warp of its own.
// Measured (8 kv heads): 9.1 us for one row over 777 tokens, 15 us for 16 rows over 512 to 2048, 22 us for 16 x 2 verify rows
// over 512 to 4096, 86 us (5.4 TB/s) for 60 rows over 256 to 8192 in pages of 16, 360 us (6.0 TB/s) for 8 over 131072 each,
// where one kv head instead of eight, rows adjacent instead of 1 KB apart, takes 317.  Short steps pay for the
// plan record, the ramp and the merge of the eight warps.
#include "decode_walk.cuh"
#include "fp8.cuh"

#include <type_traits>

namespace b200 {

constexpr int kF8Groups = 4;                 // consumer groups, which take the tiles in turn
constexpr int kF8GroupWarps = 2;             // 32 tokens of a tile each
// A multiple of the groups: a stage stays with one group for ever.  128 KB in flight; 12 stages (192 KB) leave no L1
// to the block table, the scales and the plan, and took 402 us instead of 366 (360 now) on 8 x 131072 tokens.
constexpr int kF8Stages = 8;
static_assert(kF8Stages % kF8Groups == 0, "each stage must always be consumed by the same warp group");
constexpr int kF8Warps = kF8GroupWarps * kF8Groups;
constexpr int kF8Consumers = kF8Warps * 32;
constexpr int kF8Threads = kF8Consumers + 32 * kF8Groups;        // and a producer warp per group
constexpr int kF8TileBytes = kTileTokens * kFp8HeadDim;          // K or V tile: 64 rows of 128 bytes
constexpr int kF8StageBytes = 2 * kF8TileBytes;
constexpr int kF8MaxBoxes = kTileTokens / kFp8MinBlockSize;      // pages a tile can span
constexpr int kF8SlotFloats = kMaxRows * kHeadDim;
// O's reference lies 2^15 below the largest contribution so far: the largest weight is 2^15, f16 ends at 2^16, and what
// a weight keeps of its bits does not begin to shrink before it is 2^-29 of the largest (2^-14 without).
constexpr float kF8WeightLog2 = 15.f;
static_assert(kF8GroupWarps * 32 == kTileTokens && kF8Warps == 8, "the merge is written for eight warps");
static_assert(kHeadDim == kFp8HeadDim, "one head width");

struct __align__(1024) DecodeFp8Smem {
  uint8_t stage[kF8Stages][kF8StageBytes];                       // [K | V]
  float slots[4][kF8SlotFloats];                                 // merge buffer, 4 warps at a time
  float red_m[kF8Warps][kMaxRows];                               // running maximum of the scores
  float red_o[kF8Warps][kMaxRows];                               // running maximum of score + log2 of V's scale
  float red_l[kF8Warps][kMaxRows];
  float page_scale[kF8Stages][2][kF8MaxBoxes];                   // K, V
  uint64_t full[kF8Stages];
  uint64_t empty[kF8Stages];
  int abort_flag;
  int merge_count;                                               // cut pairs whose last record this CTA wrote
  int merge_list[kMaxDeferred];
};
static_assert(sizeof(DecodeFp8Smem) <= 227 * 1024, "shared memory budget of one CTA");

struct DecodeFp8Params {
  const __nv_bfloat16* q;
  int64_t q_stride;                 // elements between query tokens
  const float* scale_of[2];         // (num_blocks, Hkv), K and V
  const int32_t* block_table;
  int64_t bt_stride;
  int table_rows, table_cols;       // entries the table has: a plan that asks for more finds no page there
  int num_tokens;                   // rows of q and out
  int32_t* plan;                    // the arrival counters of its cut pairs are counted up and put back to zero
  float* part;                      // partial records, kRecFloats each
  void* out;                        // (T, Hq, 128) bf16 or fp32
  float* lse_out;                   // (T, Hq) or null
  int32_t* status;
  int num_q_heads, num_kv_heads, group;
  int block_size, block_shift, num_blocks;
  int box_tokens, boxes_per_tile;
  int out_is_f32;
  int max_partials;                 // records the workspace holds
  float scale_log2;
};

// D(16x8, fp32) += A(16x16, f16, row) * B(16x8, f16, col)
__device__ __forceinline__ void mma_f16_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Transposes an 8 x 8 matrix of f16 pairs that the warp holds row by row.
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v) {
  uint32_t t;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(t) : "r"(v));
  return t;
}

// What a consumer warp carries through the tiles of an item with kN column tiles of 8 query rows.  Lane
// (quad, qlane) belongs to the rows 8 n + 2 qlane + e, e = 0, 1.
template <int kN>
struct RowState {
  float o[8][kN][4];             // O^T, 16 columns of V a step: [step][n][e], columns 2 quad (+1: [2 + e])
  float m[kN][2], l[kN][2];      // this lane's maximum of the scores, and the sum that refers to it
  float mo[kN][2];               // the row's reference of O, the same in its eight lanes
};

// One tile's 32 tokens of this warp, as two halves of 16.
template <int kN>
__device__ __forceinline__ void attend_tile(RowState<kN>& st, const uint32_t (&qf)[kN][8][2], const float (&to_log2)[kN][2],
                                            const int (&lim)[kN][2], uint32_t kbase, uint32_t vbase,
                                            const float (&s_k)[2], const float (&s_v)[2], int tok0, int row_of,
                                            int chunk_of) {
  // ---- S^T = K Q^T: 16 tokens a half, eight k-steps of 16 dims
  float s[2][kN][4];
#pragma unroll
  for (int half = 0; half < 2; ++half)
#pragma unroll
    for (int n = 0; n < kN; ++n) s[half][n][0] = s[half][n][1] = s[half][n][2] = s[half][n][3] = 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t kb[2][4];           // tokens 0-7 and 8-15 of the half in chunk 2j, then in chunk 2j + 1
    ldmatrix_x4(kb[0], kbase + swz128(row_of, j * 2 + chunk_of));
    ldmatrix_x4(kb[1], kbase + swz128(row_of + 16, j * 2 + chunk_of));
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint32_t lo = kb[half][2 * c], hi = kb[half][2 * c + 1];
        const uint32_t a0 = e4m3x2_to_f16x2((uint16_t)lo), a2 = e4m3x2_to_f16x2((uint16_t)(lo >> 16));
        const uint32_t a1 = e4m3x2_to_f16x2((uint16_t)hi), a3 = e4m3x2_to_f16x2((uint16_t)(hi >> 16));
#pragma unroll
        for (int n = 0; n < kN; ++n) mma_f16_16816(s[half][n], a0, a1, a2, a3, qf[n][2 * j + c][0], qf[n][2 * j + c][1]);
      }
  }
  // ---- scores, mask, maxima; element [half][n][2 t + e]: token quad + 8 t of the half, row e
  const float lv[2] = {fast_log2(s_v[0]), fast_log2(s_v[1])};
  float top_o[kN][2];
  bool raised = false;
#pragma unroll
  for (int n = 0; n < kN; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float top[2];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const float f = to_log2[n][e] * s_k[half];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          float& y = s[half][n][2 * t + e];
          y = tok0 + 16 * half + 8 * t > lim[n][e] ? -INFINITY : y * f;
        }
        top[half] = fmaxf(s[half][n][e], s[half][n][2 + e]);
      }
      top_o[n][e] = fmaxf(top[0] + lv[0], top[1] + lv[1]);
      raised |= top_o[n][e] > st.mo[n][e];
      const float m_new = fmaxf(st.m[n][e], fmaxf(top[0], top[1]));
      st.l[n][e] *= fast_exp2(st.m[n][e] - (m_new == -INFINITY ? 0.f : m_new));       // m = -inf -> 0
      st.m[n][e] = m_new;
    }
  if (__any_sync(0xffffffffu, raised)) {
#pragma unroll
    for (int n = 0; n < kN; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float t = top_o[n][e];
        t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 4));
        t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 8));
        t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 16));
        const float mo_new = fmaxf(st.mo[n][e], t);
        const float shrink = fast_exp2(st.mo[n][e] - (mo_new == -INFINITY ? 0.f : mo_new));
        st.mo[n][e] = mo_new;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          st.o[i][n][e] *= shrink;
          st.o[i][n][2 + e] *= shrink;
        }
      }
  }
  // ---- weights: (token, row pair) fragments to the (row, token pair) ones of the second product
  uint32_t pf[2][kN][2];
#pragma unroll
  for (int n = 0; n < kN; ++n) {
    float w[2][2][2];            // [half][t][e]
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float ms = st.m[n][e] == -INFINITY ? 0.f : st.m[n][e];
      const float os = st.mo[n][e] == -INFINITY ? 0.f : st.mo[n][e] - kF8WeightLog2;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        // w = p 2^up with p = 2^(x - m); bounded, so that a weight whose p is 0 does not become 0 * inf
        const float up = st.m[n][e] + lv[half] - os;
        const float c = fast_exp2(up > 126.f ? 126.f : up);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const float pr = fast_exp2(s[half][n][2 * t + e] - ms);
          st.l[n][e] += pr;
          w[half][t][e] = pr * c;
        }
      }
    }
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int t = 0; t < 2; ++t) pf[half][n][t] = transpose_8x8(pack_f16(w[half][t][0], w[half][t][1]));
  }
  // ---- O^T += V^T P^T
#pragma unroll
  for (int j = 0; j < 4; ++j) {                 // two 16-byte chunks of the columns at a time
    uint32_t vb[2][4];                          // chunk 2j: tokens 0-7, 8-15 of the half; then chunk 2j + 1
    ldmatrix_x4_trans(vb[0], vbase + swz128(row_of, j * 2 + chunk_of));
    ldmatrix_x4_trans(vb[1], vbase + swz128(row_of + 16, j * 2 + chunk_of));
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        // bytes (token, column) (t0,d0) (t0,d1) (t1,d0) (t1,d1) -> column d0's tokens, column d1's tokens
        const uint32_t lo = __byte_perm(vb[half][c * 2], 0, 0x3120), hi = __byte_perm(vb[half][c * 2 + 1], 0, 0x3120);
        const uint32_t a0 = e4m3x2_to_f16x2((uint16_t)lo), a1 = e4m3x2_to_f16x2((uint16_t)(lo >> 16));
        const uint32_t a2 = e4m3x2_to_f16x2((uint16_t)hi), a3 = e4m3x2_to_f16x2((uint16_t)(hi >> 16));
#pragma unroll
        for (int n = 0; n < kN; ++n) mma_f16_16816(st.o[2 * j + c][n], a0, a1, a2, a3, pf[half][n][0], pf[half][n][1]);
      }
  }
}

__global__ void __launch_bounds__(kF8Threads, 1)
paged_decode_gqa_fp8_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                            const DecodeFp8Params p) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  DecodeFp8Smem& sm = *reinterpret_cast<DecodeFp8Smem*>(smem_raw);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  if (smem_u32(smem_raw) & 1023u) {       // the swizzled tiles need a 1024-byte aligned base
    if (threadIdx.x == 0 && p.status) atomicOr(p.status, B200_STATUS_BAD_LAUNCH);
    return;
  }

  // The plan is host-built and reaches the device by a copy, never by the kernel in
  // front of this one: its words may be read before the grid dependency is resolved.
  const int32_t* plan = p.plan;
  const int4* rec = reinterpret_cast<const int4*>(plan + kPlanHeaderInts + kCtaInts * blockIdx.x);
  const int4 r0 = __ldg(rec), r1 = __ldg(rec + 1), r2 = __ldg(rec + 2), r3 = __ldg(rec + 3);
  const int4 hdr0 = __ldg(reinterpret_cast<const int4*>(plan));
  const int4 hdr1 = __ldg(reinterpret_cast<const int4*>(plan) + 1);
  const int item_begin = r0.x;
  const int item_end = r0.y;
  const DecodeItem* items = reinterpret_cast<const DecodeItem*>(plan + hdr1.z);   // kHdrOffItems

  if (threadIdx.x == 0) {
    sm.abort_flag = 0;
    sm.merge_count = 0;
    for (int s = 0; s < kF8Stages; ++s) {
      mbar_init(&sm.full[s], 1 + p.boxes_per_tile);   // the TMA bytes, and each box's two scales
      mbar_init(&sm.empty[s], kF8GroupWarps);         // one arrival per warp of the consuming group
    }
    mbar_fence_init();
  }
  __syncthreads();
  // While the kernel in front drains: the first tiles of this CTA's first item are asked into L2 (hints
  // only; the block ids are read past the L1 and used for nothing but the prefetch addresses).
  if (warp == kF8Warps && item_begin < item_end) {
    constexpr int kHintTiles = 4;
    const int nbox = p.boxes_per_tile;
    const int n_hint = min(r1.w - r1.z, kHintTiles) * nbox;          // tile_end - tile_begin of the first item
    if (lane < n_hint && r2.x > 0) {
      const int tile = r1.z + lane / nbox, box = lane % nbox;
      int lb = ((tile * kTileTokens) >> p.block_shift) + box;
      const int last_block = (r2.x - 1) >> p.block_shift;
      lb = lb > last_block ? last_block : lb;
      const bool listed = r1.x < p.table_rows && lb < p.table_cols;
      const int bid = listed ? __ldcg(p.block_table + (int64_t)r1.x * p.bt_stride + lb) : -1;
      if (bid >= 0 && bid < p.num_blocks) {
        const int tok = (tile * kTileTokens + box * p.box_tokens) & (p.block_size - 1);
        tma_prefetch_4d(&k_map, 0, r1.y, tok, bid);
        tma_prefetch_4d(&v_map, 0, r1.y, tok, bid);
      }
    }
  }
  grid_dep_launch();              // the next kernel may be scheduled; it waits for this grid itself
  grid_dep_wait();                // q, the block table and the step's new cache rows come from earlier kernels
  if (hdr0.x != kPlanMagic || hdr0.y != (int)gridDim.x) {      // not a plan for this launch
    if (threadIdx.x == 0 && p.status) atomicOr(p.status, B200_STATUS_BAD_LAUNCH);
    return;
  }
  if (item_begin >= item_end) return;
  volatile int* abort_flag = &sm.abort_flag;

  if (warp >= kF8Warps) {
    // --------------- producer of group warp - kF8Warps: its tiles, its stages ---------------
    const int grp = warp - kF8Warps;
    if (lane == 0) {
      tma_prefetch_desc(&k_map);
      tma_prefetch_desc(&v_map);
    }
    TileWalker w{items, item_begin, item_end, 0, 0, {}};
    w.set(r1, r2, r3);
    uint32_t it = 0;
    const int nbox = p.boxes_per_tile;
    // Block ids come out of a register window: lane l holds the id of logical block win_base + l of the
    // current sequence, and the window after it is already on its way.  A tile's boxes never straddle a
    // window (the box count divides 32).
    int win_seq = -1, win_base = 0, win_ids = 0, nxt_ids = 0;
    // the item after the current one is fetched when the current one starts
    int4 na = r1, nb = r2, nc = r3;
    auto prefetch_item = [&](int idx) {
      if (idx < item_end) {
        const int4* ip = reinterpret_cast<const int4*>(items + idx);
        na = __ldg(ip); nb = __ldg(ip + 1); nc = __ldg(ip + 2);
      }
    };
    prefetch_item(item_begin + 1);
    auto load_window = [&](int seq, int base, int kv_len) -> int {
      const int last_block = (kv_len - 1) >> p.block_shift;
      int lb = base + lane;
      lb = lb > last_block ? last_block : lb;         // past the end: any valid entry of the row
      return seq < p.table_rows && lb < p.table_cols ? p.block_table[(int64_t)seq * p.bt_stride + lb] : -1;
    };
    while (w.item < w.item_end) {
      if (w.tile >= w.tile_end) {                    // item done (or without any tile: an empty key range)
        ++w.item;
        if (w.item < w.item_end) {
          w.set(na, nb, nc);
          prefetch_item(w.item + 1);
        }
        continue;
      }
      {                                              // on to this group's next tile of the item
        const int ahead = (grp - (int)it) & (kF8Groups - 1);
        const int step = min(ahead, w.tile_end - w.tile);
        it += step;
        w.tile += step;
        if (w.tile >= w.tile_end) continue;
      }
      const int first_lb = (w.tile * kTileTokens) >> p.block_shift;
      const int base = first_lb & ~31;
      if (w.cur.seq != win_seq || base != win_base) {
        if (w.cur.seq == win_seq && base == win_base + 32) {
          win_ids = nxt_ids;                          // the prefetched window
        } else {
          win_ids = load_window(w.cur.seq, base, w.cur.kv_len);
        }
        win_seq = w.cur.seq;
        win_base = base;
        nxt_ids = load_window(w.cur.seq, base + 32, w.cur.kv_len);   // used 32 blocks from now, if at all
      }
      // this lane's box of the tile (lanes >= nbox idle); tail boxes re-read the last valid page
      const int last_block = (w.cur.kv_len - 1) >> p.block_shift;
      int lb = first_lb + (lane < nbox ? lane : 0);
      lb = lb > last_block ? last_block : lb;
      int b = __shfl_sync(0xffffffffu, win_ids, lb - win_base);

      const int s = it % kF8Stages;
      const uint32_t ph = (it / kF8Stages) & 1u;
      mbar_wait_bounded(&sm.empty[s], ph ^ 1u, abort_flag, p.status);
      if (__any_sync(0xffffffffu, *abort_flag)) break;      // the stage may still be in use: nothing more is loaded
      if (lane == 0) mbar_arrive_expect_tx(&sm.full[s], kF8StageBytes);
      __syncwarp();
      if (lane < nbox) {
        const bool have = b >= 0 && b < p.num_blocks;
        if (!have) {                                // out-of-pool id: codes and scales are zero, flag it
          if (p.status) atomicOr(p.status, B200_STATUS_BAD_BLOCK);
          b = p.num_blocks;
        }
        const int tok = (w.tile * kTileTokens + lane * p.box_tokens) & (p.block_size - 1);
        uint8_t* dst = sm.stage[s] + lane * p.box_tokens * kFp8HeadDim;
        const int h = w.cur.kv_head;
        tma_load_4d(dst, &k_map, &sm.full[s], 0, h, tok, b);
        tma_load_4d(dst + kF8TileBytes, &v_map, &sm.full[s], 0, h, tok, b);
        const int64_t at = have ? (int64_t)b * p.num_kv_heads + h : 0;
        cp_async_f32(&sm.page_scale[s][0][lane], p.scale_of[0] + at, have);
        cp_async_f32(&sm.page_scale[s][1][lane], p.scale_of[1] + at, have);
        cp_async_arrive(&sm.full[s]);
      }
      __syncwarp();
      ++it;
      ++w.tile;
    }
    // drain: do not leave while copies may still land in this CTA's shared memory.  `it` is past the last tile, or the first
    // tile of this group that was not loaded.
    if (lane == 0) {
      const uint32_t mine = (it + kF8Groups - 1 - grp) / kF8Groups;      // tiles this warp has loaded
      for (uint32_t k = 0; k < (uint32_t)(kF8Stages / kF8Groups) && k < mine; ++k) {
        const uint32_t j = (mine - 1 - k) * kF8Groups + grp;
        mbar_wait_landed(&sm.full[j % kF8Stages], (j / kF8Stages) & 1u);
      }
    }
    return;
  }

  // -------------------------------- consumers --------------------------------
  const int grp = warp / kF8GroupWarps;          // which tiles (running tile counter modulo the groups)
  const int wslice = (warp % kF8GroupWarps) * 32; // 32-token slice of the tile
  const int quad = lane >> 2;         // fragment row (and row + 8)
  const int qlane = lane & 3;
  const int G = p.group;
  const int box[2] = {wslice / p.box_tokens, (wslice + 16) / p.box_tokens};   // the pages of its two halves

  // ldmatrix lane addressing (row of the tile, which of two 16-byte chunks)
  const int row_of = wslice + (((lane >> 3) & 1) << 3) + (lane & 7);     // matrices 1,3 -> tokens +8
  const int chunk_of = lane >> 4;                                        // matrices 2,3 -> next chunk

  TileWalker w{items, item_begin, item_end, 0, 0, {}};
  w.set(r1, r2, r3);
  uint32_t it = 0;

  // Q rows of an item as they lie in memory: lane (quad, qlane) is the source of rows quad and quad + 8 in the
  // B fragments (k = dim, n = row), 8 bytes (4 dims) per 16 dims; rows beyond q_len*group are zero.  They are fetched
  // for the NEXT item right after the tile loop, so the global loads fly while the warps merge and write the current
  // item.
  uint2 qraw[2][8];
  // rows of an item; none if they do not lie within q and out (a plan refilled for a larger step)
  auto rows_of = [&](const DecodeItem& qi) -> int {
    return qi.q_start + qi.q_len <= p.num_tokens ? qi.q_len * G : 0;
  };
  auto load_q = [&](const DecodeItem& qi) {
    const int qrows = rows_of(qi);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = quad + 8 * h;
      const bool have = row < qrows;
      const __nv_bfloat16* src = p.q + (int64_t)(qi.q_start + (have ? row / G : 0)) * p.q_stride +
                                 (int64_t)(qi.kv_head * G + (have ? row % G : 0)) * kHeadDim + qlane * 4;
#pragma unroll
      for (int ks = 0; ks < 8; ++ks)
        qraw[h][ks] = have ? *reinterpret_cast<const uint2*>(src + ks * 16) : make_uint2(0u, 0u);
    }
  };
  load_q(w.cur);

  // A partial record is announced (arrival counter of its pair) one item late, or at the end
  // of the CTA's work: by then its stores have long left the SM and the fence that must
  // precede the announcement costs nothing.
  int pending_multi = -1;
  const int off_multi = hdr1.w;
  auto announce = [&](int multi_idx) {            // thread 0, after a fence by all and a barrier
    MultiGroup* mg = reinterpret_cast<MultiGroup*>(p.plan + off_multi) + multi_idx;
    const int n_parts = mg->part_end - mg->part_begin;
    if (atomicAdd(&mg->arrivals, 1) == n_parts - 1) {
      mg->arrivals = 0;                           // ready for the next launch on this plan
      __threadfence();                            // the other CTAs' records are visible from here on
      if (mg->part_end > p.max_partials) {        // not all of them found room: there is nothing to merge
      } else if (sm.merge_count < kMaxDeferred) {
        sm.merge_list[sm.merge_count] = multi_idx;
        sm.merge_count = sm.merge_count + 1;
      } else if (p.status) {                      // the planner never gives a CTA this many cut pieces
        atomicOr(p.status, B200_STATUS_BAD_LAUNCH);
      }
    }
  };
  // the record of the item after the current one, fetched while the current one streams
  int4 na = r1, nb = r2;
  auto prefetch_item = [&](int idx) {
    if (idx < item_end) {
      const int4* ip = reinterpret_cast<const int4*>(items + idx);
      na = __ldg(ip); nb = __ldg(ip + 1);
    }
  };
  prefetch_item(item_begin + 1);

  while (w.item < w.item_end) {
    const DecodeItem item = w.cur;
    const int rows = rows_of(item);
    // The item's tiles, with one column tile of query rows or two.  What they leave goes to the reduction arrays
    // and, in `o`, to the merge below.
    float row_m[2][2], row_l[2][2], row_o[2][2];       // of rows 8 n + 2 qlane + e
    float o[8][2][4];
    auto attend = [&](auto n_c) {
      constexpr int kN = decltype(n_c)::value;
      // Q to f16: each row times a power of two that brings its largest magnitude to [2^14, 2^15).  bf16 has 8
      // significant bits, f16 11 down to 2^-14: exact for all elements within 2^-28 of the row's largest, and 2^-39 of it
      // off at most below that.
      uint32_t qf[kN][8][2];
      float to_log2[kN][2];              // per row of this lane: a product with K codes to log2 units / s_k
      int lim[kN][2];                    // its last visible key (-1: row unused, everything masked)
#pragma unroll
      for (int n = 0; n < kN; ++n) {
        uint32_t top = 0;
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {
          top = max(top, max(qraw[n][ks].x & 0x7fffu, (qraw[n][ks].x >> 16) & 0x7fffu));
          top = max(top, max(qraw[n][ks].y & 0x7fffu, (qraw[n][ks].y >> 16) & 0x7fffu));
        }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int ex = max((int)(top >> 7), 15);                     // exponent field; at least 15 keeps both factors normal
        // 2^(14 - (ex - 127)); any infinity or NaN makes the row NaN, also where all its scores would be -inf
        const float up = ex == 255 ? NAN : __uint_as_float((uint32_t)(268 - ex) << 23);
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {
          const uint2 v = qraw[n][ks];
          qf[n][ks][0] = pack_f16(__uint_as_float(v.x << 16) * up, __uint_as_float(v.x & 0xffff0000u) * up);
          qf[n][ks][1] = pack_f16(__uint_as_float(v.y << 16) * up, __uint_as_float(v.y & 0xffff0000u) * up);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int row = 2 * qlane + e;                             // its maximum is with the lanes of quad `row`
          const int row_ex = __shfl_sync(0xffffffffu, ex, row * 4);
          to_log2[n][e] = __uint_as_float((uint32_t)(row_ex - 14) << 23) * p.scale_log2;
          lim[n][e] = 8 * n + row < rows ? min(item.causal_base + (8 * n + row) / G, item.kv_len - 1) : -1;
        }
      }
      RowState<kN> st;
#pragma unroll
      for (int n = 0; n < kN; ++n) {
#pragma unroll
        for (int i = 0; i < 8; ++i) st.o[i][n][0] = st.o[i][n][1] = st.o[i][n][2] = st.o[i][n][3] = 0.f;
        st.m[n][0] = st.m[n][1] = st.mo[n][0] = st.mo[n][1] = -INFINITY;
        st.l[n][0] = st.l[n][1] = 0.f;
      }
      const uint32_t first = it + ((grp - it) & (kF8Groups - 1));    // this group's first tile of the item
      const uint32_t last = it + (uint32_t)(item.tile_end - item.tile_begin);
      for (uint32_t k = first; k < last; k += kF8Groups) {
        const int tile = item.tile_begin + (int)(k - it);
        const int s = k % kF8Stages;
        mbar_wait_bounded(&sm.full[s], (k / kF8Stages) & 1u, abort_flag, p.status);
        const float s_k[2] = {sm.page_scale[s][0][box[0]], sm.page_scale[s][0][box[1]]};
        const float s_v[2] = {sm.page_scale[s][1][box[0]], sm.page_scale[s][1][box[1]]};
        // Rows past the sequence's end carry weight 0, but 0 x NaN is NaN: whatever codes an unwritten cache slot
        // holds must not reach the MMA.  Only a pair's last tile has such rows; the warp clears its own.
        const bool ragged = (tile + 1) * kTileTokens > item.kv_len;
        if (ragged) {
          const int first_bad = item.kv_len - tile * kTileTokens;    // first row of the tile past the end
          for (int idx = lane; idx < 32 * 8; idx += 32) {
            const int row = wslice + (idx >> 3);
            if (row >= first_bad)
              *reinterpret_cast<uint4*>(sm.stage[s] + kF8TileBytes + swz128(row, idx & 7)) = make_uint4(0u, 0u, 0u, 0u);
          }
          __syncwarp();
        }
        const uint32_t kbase = smem_u32(sm.stage[s]);
        attend_tile<kN>(st, qf, to_log2, lim, kbase, kbase + kF8TileBytes, s_k, s_v, tile * kTileTokens + wslice + quad,
                        row_of, chunk_of);
        // the stage goes back to TMA: order this warp's stores into it before TMA's writes
        if (ragged) fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.empty[s]);
      }
      it = last;
      // the eight lanes' own maxima and sums to the row's
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float top = -INFINITY, sum = 0.f, ref = -INFINITY;
          if (n < kN) {
            const int nn = n < kN ? n : 0;
            const float own = st.m[nn][e];
            top = own;
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
            sum = top == -INFINITY ? st.l[nn][e] : st.l[nn][e] * fast_exp2(own - top);
            sum += __shfl_xor_sync(0xffffffffu, sum, 4);
            sum += __shfl_xor_sync(0xffffffffu, sum, 8);
            sum += __shfl_xor_sync(0xffffffffu, sum, 16);
            ref = st.mo[nn][e];
          }
          row_m[n][e] = top;
          row_l[n][e] = sum;
          row_o[n][e] = ref;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            o[i][n][e] = n < kN ? st.o[i][n < kN ? n : 0][e] : 0.f;
            o[i][n][2 + e] = n < kN ? st.o[i][n < kN ? n : 0][2 + e] : 0.f;
          }
        }
    };
    if (rows <= 8)
      attend(std::integral_constant<int, 1>{});
    else
      attend(std::integral_constant<int, 2>{});

    // ---- next item's Q on its way, then merge the warps (fixed order) and write the result
    ++w.item;
    if (w.item < w.item_end) {
      w.set(na, nb, __ldg(reinterpret_cast<const int4*>(items + w.item) + 2));
      prefetch_item(w.item + 1);
      load_q(w.cur);
    }
    if (pending_multi >= 0) __threadfence();      // stores of the PREVIOUS partial record (long done)
    if (quad == 0) {
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          sm.red_m[warp][8 * n + 2 * qlane + e] = row_m[n][e];
          sm.red_o[warp][8 * n + 2 * qlane + e] = row_o[n][e];
        }
    }
    named_bar_sync(1, kF8Consumers);                           // (1) every warp's row maxima are in place
    if (pending_multi >= 0) {
      if (threadIdx.x == 0) announce(pending_multi);
      pending_multi = -1;
    }
    // bring this warp's sums and accumulators to the rows' common maxima
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = 8 * n + 2 * qlane + e;
        float g = -INFINITY, go = -INFINITY;
#pragma unroll
        for (int ww = 0; ww < kF8Warps; ++ww) {
          g = fmaxf(g, sm.red_m[ww][row]);
          go = fmaxf(go, sm.red_o[ww][row]);
        }
        // a row whose scores are all NaN has no maximum but a sum that says so
        const float f = row_m[n][e] == -INFINITY ? 1.f : fast_exp2(row_m[n][e] - g);
        const float fo = row_o[n][e] == -INFINITY ? 1.f : fast_exp2(row_o[n][e] - go);
        if (quad == 0) sm.red_l[warp][row] = row_l[n][e] * f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          o[i][n][e] *= fo;
          o[i][n][2 + e] *= fo;
        }
      }
    // A lane holds two neighbouring columns of a row: 8-byte accesses, of which the 16 lanes of a phase belong to four
    // rows of four quads each.  Rows are a multiple of the 32 banks apart: the column is XOR-ed with 8 times the
    // row's lane, which spreads them over all banks.
    const int swz = qlane << 3;
    const int n_cols = rows > 8 ? 2 : 1;          // column tiles that hold rows
    if (warp >= 4) {
      float* slot = sm.slots[warp - 4];
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        if (n >= n_cols) break;
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
          for (int i = 0; i < 8; ++i)
            *reinterpret_cast<float2*>(slot + (8 * n + 2 * qlane + e) * kHeadDim + ((16 * i + 2 * quad) ^ swz)) =
                make_float2(o[i][n][e], o[i][n][2 + e]);
      }
    }
    named_bar_sync(1, kF8Consumers);                           // (2) warps 4-7 have parked their sums
    if (warp < 4) {
      // Add the partner warp's sums in place: a thread rewrites exactly the words it read.  The loads of a row
      // are issued together before any of their stores (the compiler must assume they alias).
      float* slot = sm.slots[warp];
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        if (n >= n_cols) break;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float* row_at = slot + (8 * n + 2 * qlane + e) * kHeadDim;
          float2 a[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) a[i] = *reinterpret_cast<const float2*>(row_at + ((16 * i + 2 * quad) ^ swz));
#pragma unroll
          for (int i = 0; i < 8; ++i)
            *reinterpret_cast<float2*>(row_at + ((16 * i + 2 * quad) ^ swz)) =
                make_float2(a[i].x + o[i][n][e], a[i].y + o[i][n][2 + e]);
        }
      }
    }
    // 256 threads: thread -> rows (t / 32) and (t / 32 + 8), 4 columns each, so a warp reads and
    // writes whole rows.  The rows' maxima and scaled sums are taken BEFORE barrier (3): no warp
    // writes those arrays again (next item) until every thread has passed (3).
    const int t = threadIdx.x;
    const int col = (t & 31) * 4;
    float inv_r[2], unit_r[2], lse_r[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = (t >> 5) + h * 8;
      float g = -INFINITY, go = -INFINITY, lsum = 0.f;
#pragma unroll
      for (int ww = 0; ww < kF8Warps; ++ww) {
        g = fmaxf(g, sm.red_m[ww][row]);
        go = fmaxf(go, sm.red_o[ww][row]);
        lsum += sm.red_l[ww][row];
      }
      // O is in units of 2^(go - 15), the sum in units of 2^g; the factor between them in two halves, each of
      // which fp32 holds however far apart they are
      inv_r[h] = lsum == 0.f ? 0.f : 1.f / lsum;          // a NaN sum stays one
      unit_r[h] = go == -INFINITY ? 0.f : fast_exp2((go - kF8WeightLog2 - g) * 0.5f);
      lse_r[h] = lsum == 0.f ? -INFINITY : g * 0.6931471805599453f + __logf(lsum);
    }
    named_bar_sync(1, kF8Consumers);                           // (3) the four slots hold the warp-pair sums
    const bool record_fits = (item.direct || item.partial_idx < p.max_partials) && rows > 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = (t >> 5) + h * 8;
      if (row >= rows || !record_fits) continue;
      const int pcol = col ^ (((row >> 1) & 3) << 3);
      float4 acc = *reinterpret_cast<const float4*>(&sm.slots[0][row * kHeadDim + pcol]);
#pragma unroll
      for (int sl = 1; sl < 4; ++sl) {
        const float4 y = *reinterpret_cast<const float4*>(&sm.slots[sl][row * kHeadDim + pcol]);
        acc.x += y.x; acc.y += y.y; acc.z += y.z; acc.w += y.w;
      }
      const float u = unit_r[h], inv = inv_r[h];
      const float4 v = make_float4(acc.x * inv * u * u, acc.y * inv * u * u, acc.z * inv * u * u, acc.w * inv * u * u);
      if (item.direct) {
        const int64_t tok = item.q_start + row / G;
        const int head = item.kv_head * G + row % G;
        const int64_t off = (tok * p.num_q_heads + head) * kHeadDim + col;
        if (p.out_is_f32) {
          *reinterpret_cast<float4*>(reinterpret_cast<float*>(p.out) + off) = v;
        } else {
          uint2 pk;
          pk.x = pack_bf16(v.x, v.y);
          pk.y = pack_bf16(v.z, v.w);
          *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(p.out) + off) = pk;
        }
        if (p.lse_out && (t & 31) == 0) p.lse_out[tok * p.num_q_heads + head] = lse_r[h];
      } else {
        float* rec = p.part + (int64_t)item.partial_idx * kRecFloats;
        *reinterpret_cast<float4*>(rec + row * kHeadDim + col) = v;
        if ((t & 31) == 0) rec[kMaxRows * kHeadDim + row] = lse_r[h];
      }
    }
    if (!record_fits && t == 0 && p.status) atomicOr(p.status, B200_STATUS_BAD_LAUNCH);   // workspace, q or out too small
    // Also a record that found no room is counted, or the pair's counter would be off for the next launch on this plan.
    // (Rows outside q leave out all pieces of a pair, and nothing is to be merged then.)
    if (!item.direct && rows > 0) pending_multi = item.multi_idx;
    // The next item's first write to red_m / red_o comes after barrier (3) above, and its first write
    // to red_l and to the slots after its own barrier (1), which no thread passes before it has
    // finished the reads of this item.
  }

  // ---- the last record's announcement, then the merges this CTA owes: the cut pairs
  // whose last record it wrote
  if (pending_multi >= 0) {
    __threadfence();
    named_bar_sync(1, kF8Consumers);
    if (threadIdx.x == 0) announce(pending_multi);
  }
  named_bar_sync(1, kF8Consumers);
  if (sm.merge_count > 0) merge_noted_pairs(p, sm.merge_list, sm.merge_count, off_multi);
}

}  // namespace b200

extern "C" int b200_paged_decode_gqa_fp8(const void* q, int64_t q_stride, const void* key_cache,
                                         const void* value_cache, const float* key_scale,
                                         const float* value_scale, int num_blocks, int block_size,
                                         const int32_t* block_table, int64_t bt_stride, int table_rows,
                                         int table_cols, int32_t* plan_dev, const b200_decode_plan_info* info,
                                         int num_ctas, int num_tokens, int num_q_heads, int num_kv_heads, int head_dim, float scale, void* workspace,
                                         size_t workspace_bytes, void* out, int out_is_f32, float* lse_out,
                                         int32_t* status, void* stream) {
  using namespace b200;
  const char* who = "paged_decode_gqa_fp8";
  int rc = check_fp8_cache(who, key_cache, value_cache, key_scale, value_scale, num_blocks, block_size, num_kv_heads,
                           head_dim);
  if (rc) return rc;
  if (info) num_ctas = info->num_ctas;
  if (info && info->num_items == 0) return B200_OK;
  if (!q || !block_table || !plan_dev || !out || !workspace || num_q_heads <= 0 || num_q_heads % num_kv_heads ||
      num_ctas <= 0 || num_tokens < 0 || table_rows <= 0 || table_cols <= 0) {
    set_last_error("%s: null pointer, bad head counts, no CTAs or an empty block table", who);
    return B200_EINVAL;
  }
  if (reinterpret_cast<uintptr_t>(q) % 8 || q_stride % 4 || q_stride < (int64_t)num_q_heads * head_dim) {
    set_last_error("%s: q must be 8-byte aligned with a token stride >= Hq*D that is a multiple of 4 elements", who);
    return B200_EALIGN;
  }
  if (reinterpret_cast<uintptr_t>(out) % 16 || reinterpret_cast<uintptr_t>(workspace) % 16 ||
      reinterpret_cast<uintptr_t>(plan_dev) % 16) {
    set_last_error("%s: out, workspace and plan must be 16-byte aligned", who);
    return B200_EALIGN;
  }
  const size_t max_partials = workspace_bytes / (kRecFloats * sizeof(float));
  if (info && (size_t)info->num_partials > max_partials) {
    set_last_error("%s: workspace %zu bytes < %zu needed", who, workspace_bytes,
                   (size_t)info->num_partials * kRecFloats * sizeof(float));
    return B200_EPLAN;
  }
  const int box_tokens = block_size < kTileTokens ? block_size : kTileTokens;
  CUtensorMap k_map, v_map;
  rc = get_fp8_cache_tensor_map(key_cache, num_blocks, block_size, num_kv_heads, box_tokens, &k_map);
  if (rc) return rc;
  rc = get_fp8_cache_tensor_map(value_cache, num_blocks, block_size, num_kv_heads, box_tokens, &v_map);
  if (rc) return rc;

  DecodeFp8Params p;
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.q_stride = q_stride;
  p.scale_of[0] = key_scale;
  p.scale_of[1] = value_scale;
  p.block_table = block_table;
  p.bt_stride = bt_stride;
  p.table_rows = table_rows;
  p.table_cols = table_cols;
  p.num_tokens = num_tokens;
  p.plan = plan_dev;
  p.part = static_cast<float*>(workspace);
  p.max_partials = max_partials > (size_t)INT32_MAX ? INT32_MAX : (int)max_partials;
  p.out = out;
  p.lse_out = lse_out;
  p.status = status;
  p.num_q_heads = num_q_heads;
  p.num_kv_heads = num_kv_heads;
  p.group = num_q_heads / num_kv_heads;
  p.block_size = block_size;
  p.block_shift = __builtin_ctz(block_size);
  p.num_blocks = num_blocks;
  p.box_tokens = box_tokens;
  p.boxes_per_tile = kTileTokens / box_tokens;
  p.out_is_f32 = out_is_f32;
  p.scale_log2 = scale * 1.4426950408889634f;

  const size_t smem = sizeof(DecodeFp8Smem);
  static bool attr_set[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 64 || !attr_set[dev]) {
    rc = check_cuda(cudaFuncSetAttribute(paged_decode_gqa_fp8_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)smem),
                    "paged_decode_gqa_fp8 smem attribute");
    if (rc) return rc;
    if (dev < 64) attr_set[dev] = true;
  }
  return check_cuda(launch_pdl(paged_decode_gqa_fp8_kernel, dim3(num_ctas), dim3(kF8Threads), smem,
                               static_cast<cudaStream_t>(stream), k_map, v_map, p),
                    "paged_decode_gqa_fp8 launch");
}
