// Paged GQA attention for wide query blocks over an 8-bit cache (chunked prefill, multi-token
// verify): any q_len, bottom-right causal, on tcgen05 with accumulators in tensor memory.
//
//   o = sum_j softmax_j(scale * q . (ck_j s_k)) * (cv_j s_v)
//
// Work items, queue, warp roles and the two softmax groups over one O are those of the 16-bit kernel:
// 128 packed query rows of a (sequence, kv head) pair per item, one persistent CTA per SM.  What
// the 8-bit cache changes:
//
// * S = Q K^T runs as kind::f8f6f4 on the codes as TMA brings them, without converting K.  Q is split
//   into two e4m3 terms, q = 2^-u (hi + lo) with a power of two per row that brings the row's largest
//   magnitude to [2^7, 2^8): hi = e4m3(2^u q) leaves a rest of at most 4 significant bits of a
//   bf16 q, which lo holds exactly (elements below 2^-10 of the row's largest: to 2^-18 of it).  Two
//   K = 32 MMAs read the bytes that two K = 16 MMAs of the 16-bit kernel read, so S costs the same tensor
//   and shared-memory time and K half of the loads.
// * V is converted to f16 (exact) by the warpgroup that also writes O: splitting P like Q would cost the
//   softmax threads, which set the pace, five instructions per pair of weights, while that warpgroup idles
//   between items.  P is f16, three more bits than bf16 over the range that counts (below).
// * No element is multiplied by a scale.  K's scale and the row's 2^-u are in the factor that
//   turns a product into a log2 score; V's scale is in the weight, w = 2^(x + log2 s_v - M) with M 7 below the running
//   maximum of x + log2 s_v (handed between the groups with O; taken late, so that w stays under 2^15), while each group's
//   row sum refers to its own running maximum m of x.  Weights lose no bits of f16 down to 2^-21 of the largest and are not
//   dropped down to 2^-32: many small ones beside a key that carries the row (and may have a V of zeros) add up to
//   what they should.  A page is at least 16 tokens: a tile has 8 column groups of 16, each with its
//   scales, or one pair for the whole tile when pages hold 128 tokens or more.
//
// Tensor-bound: flops = 4 * 128 * sum over rows of visible keys; 1024 tensor cycles and 1024 cycles of exponentials for a
// tile of 128 x 128.  A tile takes about 1850 cycles: each group's chain scores -> maximum -> weights -> P is about 3700
// long, two of them run, and a softmax warp issues an instruction in about three cycles.  Where an item ends, O has
// to be read before the next item's first P V.  Measured (32 query heads, 8 kv heads; replayed graphs): 527 us on an
// 8192-token prompt (1043 TFLOP/s; about 590 in a long loop of calls, where the clock falls), 105 to 110 us on four 512-token
// chunks over cached prefixes, 37 us on 16 drafts of 5 tokens over 512 to 4096 tokens (42 uncut); a 4096-token prompt takes
// 158 us over pages of 128, 194 over pages of 64 or 32 and 212 over pages of 16 (eight pairs of scales a tile, and
// spills).  The kernel over a 16-bit cache is faster on prompts (518, 93 and 134 to 162 us): the 8-bit one is for the
// cache's size, not for these.  Where few items meet many SMs the plan cuts them along the keys (b200_prefill_split) and a
// second kernel joins the pieces: 83 us instead of 982 on 16 rows over 131072 tokens, 89 instead of 265 on 2 x 64 rows over
// 32768, 62 instead of 73 on 16 drafts over 2048 to 8192.  What else was tried: both groups on row tiles of their own with
// one K / V stream (620 us: the instruction footprint of two O rescales), the groups' exponential sections kept apart by a
// barrier (799 us against 742 at the time).  All roles' loops share the SM's instruction cache, so each piece of code is
// instantiated once and outer loops are not unrolled: from 85 KB of code to 64 KB, with the waits in line, took 742 us to
// 581; the four variants have 53 to 57 KB now.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <exception>
#include <vector>

#include "fp8.cuh"
#include "prefill_plan.cuh"
#include "tc05.cuh"

namespace b200 {

constexpr int kP8TileBytes = kPfTile * kFp8HeadDim;             // K or V codes of a tile: 16 KB
constexpr int kP8KStages = 3;
constexpr int kP8VStages = 2;                                   // codes; two more tiles wait as f16
constexpr int kP8KLead = 2;                                     // K loads run this many tiles ahead of the V loads
constexpr int kP8ScaleSlots = 8;
constexpr int kP8Groups = kPfTile / kFp8MinBlockSize;           // column groups of a tile: 8
constexpr int kMaxGroups = 1024;                                // cut items of a plan (one per SM at most)
constexpr int kP8SoftmaxThreads = 256;
constexpr int kP8ConvertThreads = 128;
constexpr int kP8Threads = kP8SoftmaxThreads + 128 + kP8ConvertThreads;   // whole warpgroups: 512 = 4 x 128
// Registers per thread after the hand-over, softmax, producer and issuers, convert: 256 * 184 + 128 * 56 + 128 * 88 =
// 256 * 192 + 128 * 48 + 128 * 80 = 512 * 128.  Spills inside a loop are dear where shared memory leaves little L1.
// With one page per tile the first split has none (106 us on four 512-token chunks, 111 with the second); the eight
// pairs of scales of smaller pages need the second's softmax registers (97 us on three sequences over pages of 32 tokens,
// 103 with the first).
template <bool kOnePage>
struct P8Regs {
  static constexpr int kSoftmax = kOnePage ? 184 : 192, kOther = kOnePage ? 56 : 48, kConvert = kOnePage ? 88 : 80;
};
constexpr int kP8TmemCols = 512;          // S0 [0,128) S1 [128,256) O [256,384) P_A [384,448) P_B [448,512)
// O is rescaled when a row's largest contribution outgrows what it was when the reference was taken by 2^kP8Lazy, and the
// reference is taken 2^kP8Lift below it: the largest weight is 2^15, f16 ends at 2^16, and a weight loses none of its bits
// down to 2^-21 of the largest contribution.  More lift for less laziness costs rescales: an 8192-token prompt takes 522 us
// with 8 and 7, 535 with 6 and 9, 549 with 4 and 11.
constexpr float kP8Lazy = 8.f, kP8Lift = 15.f - kP8Lazy;
constexpr int kP8OCol = 256;
constexpr int kP8PCol = 384;

struct __align__(1024) Prefill8Smem {
  uint8_t q[2][2][kPfRows * kFp8HeadDim];  // per item parity: hi, lo; [128 rows][128 B], swizzled
  uint8_t k[kP8KStages][kP8TileBytes];     // [128 tokens][128 B], swizzled
  uint8_t v[kP8VStages][kP8TileBytes];
  uint8_t v16[2][2 * kP8TileBytes];        // f16: [dims 0-63 | dims 64-127], 128 tokens x 128 B each, swizzled
  float row_factor[2][kPfRows];            // per item parity: |softmax scale| * log2(e) * 2^-u of the row
  float row_l[2][kPfRows];                 // end of item: the groups' row sums
  float row_m[2][kPfRows];                 // and the maxima they refer to
  float row_mfin[kPfRows];                 // end of item: the reference of O
  float row_ms[2][kPfRows];                // running reference of O after tile j, slot j & 1
  float tile_scale[kP8ScaleSlots][2][kP8Groups];   // K, V scales of a tile's column groups
  uint64_t k_full[kP8KStages];
  uint64_t k_empty[kP8KStages];
  uint64_t v_full[kP8VStages];
  uint64_t v_empty[kP8VStages];
  uint64_t v16_full[2];                    // freed by pv_done
  uint64_t scale_full[kP8ScaleSlots];      // a slot is reused 8 tiles on, when its readers are long through
  uint64_t s_full[2];
  uint64_t s_empty[2];                     // softmax threads: the tile's scores and scales are in registers
  uint64_t p_full[2];                      // per group
  uint64_t pv_done[2];                     // per tile parity
  uint64_t m_ready[2];                     // per tile parity: row_ms[parity] is written
  uint64_t o_done;                         // P V issuer -> convert warps: the item's O is complete
  uint64_t o_free;                         // convert warps -> P V issuer: O is in registers
  uint64_t l_full;                         // softmax threads -> convert warps: row_l / row_m / row_mfin written
  uint64_t l_empty;                        // and read
  uint64_t q_full[2];                      // per item parity: the Q terms and row factors are staged
  uint64_t q_empty[2];                     // all S MMAs of the item have run
  uint64_t mma_idle[2];                    // end of the CTA: all MMAs of the S and the P V issuer have run
  uint64_t item_full[2];                   // work-queue hand-off: producer warp -> the other roles
  uint64_t item_empty[2];
  alignas(16) PrefillPiece next_rec[2];    // the mailbox carries the whole record (read as int4)
  int next_item[2];
  uint32_t tmem_base;
  int abort_flag;
};
static_assert(sizeof(Prefill8Smem) <= 227 * 1024, "shared memory budget of one CTA");

struct Prefill8Params {
  const __nv_bfloat16* q;
  int64_t q_stride;
  const float* scale_of[2];         // (num_blocks, Hkv), K and V
  const int32_t* block_table;
  int64_t bt_stride;
  int table_rows, table_cols;
  int num_tokens;
  int32_t* plan;                    // header, items or pieces, groups
  float* part;                      // partial records of cut items, kPieceRecFloats each
  int max_partials;                 // records the workspace holds
  int* work_counter;                // two plan words: next item to hand out, CTAs that have left
                                    // (the word before them is the number of items)
  void* out;
  float* lse_out;
  int32_t* status;
  int num_q_heads, num_kv_heads, group;
  int block_size, block_shift, num_blocks, box_tokens, boxes_per_tile;
  int out_is_f32;
  float scale_log2;
};

// Instruction descriptor with fp32 accumulation and operand type 0: f16 in kind::f16, e4m3 in kind::f8f6f4.
__host__ __device__ constexpr uint32_t umma_idesc_type0(int m, int n, bool b_mn_major) {
  return (1u << 4) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// Waits for a phase of an mbarrier, at most 2^20 tries of up to about 1.5 us each, which is how long the unit suspends a
// thread by default (a longer hint wakes it later: 582 us instead of 568 on an 8192-token prompt).  Then the CTA's abort
// flag goes up: every later wait returns at once, so control flow stays uniform, nothing more is loaded, the copies and matrix
// products under way are waited for (mbar_wait_landed) and the kernel reports B200_STATUS_WAIT_TIMEOUT at its end.  A dozen
// instructions: it stands at every wait of loops that together have to stay in the instruction cache.  Returns whether the
// phase has completed.  (The producer goes by that: its reading the flag for each load took 547 us instead of 527.)
__device__ __forceinline__ bool mbar_wait_limited(uint64_t* bar, uint32_t parity, uint32_t abort_at) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .u32 left, gone;\n\t"
      "mov.u32 left, 0x100000;\n"
      "again:\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 q, [%1], %2;\n\t"
      "@q bra through;\n\t"
      "ld.volatile.shared.u32 gone, [%3];\n\t"
      "setp.ne.u32 p, gone, 0;\n\t"
      "@p bra through;\n\t"
      "sub.u32 left, left, 1;\n\t"
      "setp.ne.u32 p, left, 0;\n\t"
      "@p bra again;\n\t"
      "st.volatile.shared.u32 [%3], 1;\n"
      "through:\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity), "r"(abort_at)
      : "memory");
  return ok != 0;
}

// Shared-memory matrix descriptor (128-byte swizzle) in two parts: the word with the address, and the rest.
__device__ __forceinline__ uint32_t umma_desc_lo(uint32_t smem_addr, uint32_t lbo_bytes) {
  return ((smem_addr & 0x3FFFFu) >> 4) | ((lbo_bytes >> 4) & 0x3FFFu) << 16;
}
__host__ __device__ constexpr uint64_t umma_desc_rest(uint32_t sbo_bytes) {
  return (uint64_t)((sbo_bytes >> 4) & 0x3FFFu) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// D[tmem] (+)= A[smem] * B[smem] on 8-bit codes, K = 32.
template <bool kAccumulate>
__device__ __forceinline__ void umma_f8_ss_lo(uint32_t tmem_d, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo,
                                              uint32_t b_hi, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .b64 da, db;\n\t.reg .pred p;\n\t"
      "mov.b64 da, {%1, %2};\n\tmov.b64 db, {%3, %4};\n\t"
      "setp.ne.u32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, db, %5, p;\n\t}"
      ::"r"(tmem_d), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "n"(kAccumulate ? 1 : 0));
}
// kOnePage: pages of 128 tokens or more, one pair of scales per tile.  kCut: a plan that has pieces, or that a recorded
// launch may find them in (4 % slower on an 8192-token prompt without any: the roles that walk tiles have no
// register left for where a piece begins).
template <bool kOnePage, bool kCut>
__global__ void __launch_bounds__(kP8Threads, 1)
paged_prefill_fp8_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                         const Prefill8Params p) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  Prefill8Smem& sm = *reinterpret_cast<Prefill8Smem*>(smem_raw);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  if (smem_u32(smem_raw) & 1023u) {       // the swizzled tiles need a 1024-byte aligned base
    if (threadIdx.x == 0 && p.status) atomicOr(p.status, B200_STATUS_BAD_LAUNCH);
    return;
  }

  if (threadIdx.x == 0) {
    sm.abort_flag = 0;
    for (int s = 0; s < kP8KStages; ++s) {
      mbar_init(&sm.k_full[s], 1);
      mbar_init(&sm.k_empty[s], 1);
    }
    for (int s = 0; s < kP8VStages; ++s) {
      mbar_init(&sm.v_full[s], 1);
      mbar_init(&sm.v_empty[s], kP8ConvertThreads);
    }
    for (int s = 0; s < kP8ScaleSlots; ++s) mbar_init(&sm.scale_full[s], 32);
    for (int b = 0; b < 2; ++b) {
      mbar_init(&sm.v16_full[b], kP8ConvertThreads);
      mbar_init(&sm.s_full[b], 1);
      mbar_init(&sm.s_empty[b], 128);
      mbar_init(&sm.p_full[b], 128);
      mbar_init(&sm.pv_done[b], 1);
      mbar_init(&sm.m_ready[b], 128);
      mbar_init(&sm.q_full[b], kP8ConvertThreads);
      mbar_init(&sm.q_empty[b], 1);
      mbar_init(&sm.mma_idle[b], 1);
      mbar_init(&sm.item_full[b], 1);
      mbar_init(&sm.item_empty[b], kP8SoftmaxThreads + 2 + kP8ConvertThreads);   // all consumers of the mailbox
    }
    mbar_init(&sm.o_done, 1);
    mbar_init(&sm.o_free, kP8ConvertThreads);
    mbar_init(&sm.l_full, kP8SoftmaxThreads);
    mbar_init(&sm.l_empty, kP8ConvertThreads);
    mbar_fence_init();
  }
  if (warp == 9) {
    tmem_alloc(&sm.tmem_base, kP8TmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  grid_dep_wait();                // q and the step's new cache rows come from earlier kernels
  const uint32_t tmem = sm.tmem_base;
  volatile int* abort_flag = &sm.abort_flag;
  const uint32_t abort_at = smem_u32(&sm.abort_flag);
  // Items are handed out dynamically, longest first: the producer warp draws the next index from a
  // global counter and passes it to the other roles through a two-slot mailbox.  -1 ends the CTA.
  auto first_of = [](const PrefillPiece& x) -> int { return kCut ? x.tile_begin : 0; };   // first tile
  auto take_item = [&](uint32_t k, PrefillPiece& rec) -> int {
    mbar_wait_limited(&sm.item_full[k & 1u], (k >> 1) & 1u, abort_at);
    const int idx = *reinterpret_cast<volatile int*>(&sm.next_item[k & 1u]);
    const int4* src = reinterpret_cast<const int4*>(&sm.next_rec[k & 1u]);
    const int4 lo = src[0], hi = src[1];
    int2 cut = make_int2(0, -1);
    if constexpr (kCut) cut = *reinterpret_cast<const int2*>(src + 2);
    rec = PrefillPiece{lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w, cut.x, cut.y, {0, 0}};
    mbar_arrive(&sm.item_empty[k & 1u]);
    return (*abort_flag || idx < 0) ? -1 : idx;
  };

  if (warp >= 8 && warp < 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(P8Regs<kOnePage>::kOther));
    if (warp == 8) {
      // ------------------------------ TMA producer ------------------------------
      if (lane == 0) {
        tma_prefetch_desc(&k_map);
        tma_prefetch_desc(&v_map);
      }
      uint32_t it = 0, k_loaded = 0, v_loaded = 0;       // K (and scales), V: tiles whose copies have been issued
      const int nbox = p.boxes_per_tile;
      auto draw = [&](uint32_t k) -> int {
        int idx = -1;
        if (lane == 0) {
          // the first item of a CTA is its own index; the rest of the list is handed out dynamically
          idx = (k == 0) ? (int)blockIdx.x : (int)gridDim.x + atomicAdd(p.work_counter, 1);
          const int pieces = kCut ? __ldg(p.plan + kHdrPieces) : 0;    // 0: nothing is cut
          if (idx >= (pieces ? pieces : __ldg(p.plan + 1)) || *abort_flag) idx = -1;
          mbar_wait_limited(&sm.item_empty[k & 1u], ((k >> 1) & 1u) ^ 1u, abort_at);
          if (idx >= 0) {
            const int4* src = reinterpret_cast<const int4*>(
                p.plan + (pieces ? __ldg(p.plan + kHdrOffPieces) + kPieceInts * idx : kPlanHeaderInts + kPfItemInts * idx));
            int4* dst = reinterpret_cast<int4*>(&sm.next_rec[k & 1u]);
            dst[0] = __ldg(src);
            dst[1] = __ldg(src + 1);
            if constexpr (kCut) dst[2] = pieces ? __ldg(src + 2) : make_int4(0, -1, 0, 0);
          }
          sm.next_item[k & 1u] = idx;
          mbar_arrive(&sm.item_full[k & 1u]);     // release semantics: index and record are visible to waiters
        }
        idx = __shfl_sync(0xffffffffu, idx, 0);
        return idx;
      };
      const int groups_per_box = p.box_tokens / kFp8MinBlockSize;
      // Each piece of code below is instantiated once: the kernel's loops share one instruction cache.  The walk
      // starts with an item without tiles, whose only step draws item 0.
      PrefillPiece item{};
      int idx = 0;
#pragma unroll 1
      for (uint32_t k = 0; idx >= 0; ++k) {          // `item` is item k - 1; item k is drawn on the way
        const int n = item.n_tiles;
        const int32_t* const table = p.block_table + (int64_t)item.seq * p.bt_stride;
        const int last_block = (item.kv_len - 1) >> p.block_shift;
        const int cols = item.seq < p.table_rows ? p.table_cols : 0;
        // The next item is drawn eight tiles before this one's last load: the convert warps stage its Q
        // while this item's last tiles are worked on.
        const int draw_at = n > 8 ? n - 8 : 0;
        // K and V travel through separate rings (a K stage is free again as soon as S = Q K^T has run), the K loads
        // kP8KLead tiles ahead of the V loads, which take the page ids from the K loads' look-up.
        int ids[kP8KLead + 1];                       // of tiles step, step - 1, ..: lane g < 8 has the page of column group g
#pragma unroll 1
        for (int step = 0; step < n + (n > 0 ? kP8KLead : 1); ++step) {
          if (step == draw_at) idx = draw(k);
#pragma unroll
          for (int i = kP8KLead; i > 0; --i) ids[i] = ids[i - 1];
          const int box_row = lane * p.box_tokens;   // first row of this lane's box in the tile
          if (step < n) {
            const uint32_t itx = it + step;
            int bid = -1;
            if (lane < kP8Groups) {
              int lb = ((first_of(item) + step) * kPfTile + lane * kFp8MinBlockSize) >> p.block_shift;
              lb = lb > last_block ? last_block : lb;                  // the tail re-reads the last valid page
              if (lb < cols) bid = table[lb];
              if (bid >= p.num_blocks) bid = -1;
              if (bid < 0 && p.status) atomicOr(p.status, B200_STATUS_BAD_BLOCK);
            }
            ids[0] = bid;
            const int b = __shfl_sync(0xffffffffu, bid, (lane * groups_per_box) & 31);
            const int sk = itx % kP8KStages;
            const bool stage_free = mbar_wait_limited(&sm.k_empty[sk], ((itx / kP8KStages) & 1u) ^ 1u, abort_at);
            if (lane == 0 && stage_free) mbar_arrive_expect_tx(&sm.k_full[sk], kP8TileBytes);
            if (!__all_sync(0xffffffffu, stage_free)) break;       // a wait has run out: nothing more is loaded
            if (lane < nbox)                         // a page outside the pool: TMA fills zeros
              tma_load_4d(sm.k[sk] + box_row * kFp8HeadDim, &k_map, &sm.k_full[sk], 0, item.kv_head,
                          ((first_of(item) + step) * kPfTile + box_row) & (p.block_size - 1), b < 0 ? p.num_blocks : b);
            // The tile's scales, through a ring of their own: the K stage is handed back before the softmax
            // threads read them.  Slot itx - 8 is free: the K stage this tile takes was freed by S of tile
            // itx - 3, whose score buffer was handed back by the readers of tile itx - 5.
            const uint32_t sl = itx % kP8ScaleSlots;
            if (lane < kP8Groups) {
              const int64_t at = bid < 0 ? 0 : (int64_t)bid * p.num_kv_heads + item.kv_head;
              cp_async_f32(&sm.tile_scale[sl][0][lane], p.scale_of[0] + at, bid >= 0);
              cp_async_f32(&sm.tile_scale[sl][1][lane], p.scale_of[1] + at, bid >= 0);
            }
            cp_async_arrive(&sm.scale_full[sl]);
            ++k_loaded;
          }
          if (step >= kP8KLead && n > 0) {
            const int tile = step - kP8KLead;
            const uint32_t itx = it + tile;
            const int b = __shfl_sync(0xffffffffu, ids[kP8KLead], (lane * groups_per_box) & 31);
            const int sv = itx % kP8VStages;
            const bool stage_free = mbar_wait_limited(&sm.v_empty[sv], ((itx / kP8VStages) & 1u) ^ 1u, abort_at);
            if (lane == 0 && stage_free) mbar_arrive_expect_tx(&sm.v_full[sv], kP8TileBytes);
            if (!__all_sync(0xffffffffu, stage_free)) break;
            if (lane < nbox)
              tma_load_4d(sm.v[sv] + box_row * kFp8HeadDim, &v_map, &sm.v_full[sv], 0, item.kv_head,
                          ((first_of(item) + tile) * kPfTile + box_row) & (p.block_size - 1), b < 0 ? p.num_blocks : b);
            ++v_loaded;
          }
          __syncwarp();
        }
        if (__any_sync(0xffffffffu, *abort_flag)) break;
        it += n;
        item = sm.next_rec[k & 1u];                  // not overwritten before this warp draws item k + 2
      }
      // drain: nothing may still be landing when the CTA leaves
      if (lane == 0) {
        for (uint32_t k = 0; k < (uint32_t)kP8KStages && k < k_loaded; ++k) {
          const uint32_t j = k_loaded - 1 - k;
          mbar_wait_landed(&sm.k_full[j % kP8KStages], (j / kP8KStages) & 1u);
        }
        for (uint32_t k = 0; k < (uint32_t)kP8VStages && k < v_loaded; ++k) {
          const uint32_t j = v_loaded - 1 - k;
          mbar_wait_landed(&sm.v_full[j % kP8VStages], (j / kP8VStages) & 1u);
        }
        for (uint32_t k = 0; k < (uint32_t)kP8ScaleSlots && k < k_loaded; ++k) {
          const uint32_t j = k_loaded - 1 - k;
          mbar_wait_landed(&sm.scale_full[j % kP8ScaleSlots], (j / kP8ScaleSlots) & 1u);
        }
      }
    } else if (warp == 9) {
      // ------------------------- MMA issuer: S = Q K^T -------------------------
      if (lane == 0) {
        constexpr uint32_t idesc = umma_idesc_type0(kPfRows, kPfTile, false);
        constexpr uint32_t dq_hi = (uint32_t)(umma_desc_rest(1024) >> 32), dk_hi = dq_hi;
        const uint32_t dq_lo = umma_desc_lo(smem_u32(sm.q[0][0]), 16), dk_lo = umma_desc_lo(smem_u32(sm.k[0]), 16);
        constexpr uint32_t kTerm = (kPfRows * kFp8HeadDim) >> 4;   // one Q term, in descriptor units
        uint32_t it = 0;
#pragma unroll 1
        for (uint32_t item_no = 0;; ++item_no) {
          PrefillPiece rec;
          if (take_item(item_no, rec) < 0) break;
          const int n_tiles = rec.n_tiles;
          const uint32_t qb = item_no & 1u;
          mbar_wait_limited(&sm.q_full[qb], (item_no >> 1) & 1u, abort_at);
          const uint32_t q_lo = dq_lo + qb * 2 * kTerm;
          if (n_tiles == 0) umma_commit(&sm.q_empty[qb]);
#pragma unroll 1
          for (int tile = 0; tile < n_tiles; ++tile, ++it) {
            const int s = it % kP8KStages;
            const int b = it & 1u;
            mbar_wait_limited(&sm.k_full[s], (it / kP8KStages) & 1u, abort_at);
            mbar_wait_limited(&sm.s_empty[b], ((it >> 1) & 1u) ^ 1u, abort_at);
            tc_fence_after();
            const uint32_t k_lo = dk_lo + (uint32_t)((s * kP8TileBytes) >> 4);
            const uint32_t d_tmem = tmem + b * 128;
            umma_f8_ss_lo<false>(d_tmem, q_lo, dq_hi, k_lo, dk_hi, idesc);
#pragma unroll
            for (int i = 1; i < 8; ++i)             // four K = 32 steps of hi, four of lo
              umma_f8_ss_lo<true>(d_tmem, q_lo + (i >> 2) * kTerm + (i & 3) * 2, dq_hi, k_lo + (i & 3) * 2, dk_hi, idesc);
            umma_commit(&sm.s_full[b]);
            umma_commit(&sm.k_empty[s]);
            if (tile == n_tiles - 1) umma_commit(&sm.q_empty[qb]);   // the Q terms may be overwritten
          }
        }
        umma_commit(&sm.mma_idle[0]);
        mbar_wait_landed(&sm.mma_idle[0], 0);
      }
      __syncwarp();
    } else if (warp == 10) {
      // ------------------------- MMA issuer: O += P V --------------------------
      if (lane == 0) {
        constexpr uint32_t idesc = umma_idesc_type0(kPfRows, kPfHeadDim, true);
        constexpr uint32_t dv_hi = (uint32_t)(umma_desc_rest(1024) >> 32);
        const uint32_t dv_lo = umma_desc_lo(smem_u32(sm.v16[0]), kP8TileBytes);
        uint32_t it = 0;
#pragma unroll 1
        for (uint32_t item_no = 0;; ++item_no) {
          PrefillPiece rec;
          if (take_item(item_no, rec) < 0) break;
          const int n_tiles = rec.n_tiles;
          // The previous item's O has been read.  Also an item without tiles waits: o_done and o_free go item by item.
          if (item_no > 0) mbar_wait_limited(&sm.o_free, (item_no - 1) & 1u, abort_at);
#pragma unroll 1
          for (int tile = 0; tile < n_tiles; ++tile, ++it) {
            const int g = it & 1u;                            // the group that owns this tile, and its V buffer
            mbar_wait_limited(&sm.v16_full[g], (it >> 1) & 1u, abort_at);
            mbar_wait_limited(&sm.p_full[g], (it >> 1) & 1u, abort_at);
            tc_fence_after();
            const uint32_t v_lo = dv_lo + (uint32_t)((g * 2 * kP8TileBytes) >> 4);
            const uint32_t p_tmem = tmem + kP8PCol + g * 64;  // P of the tile: 128 tokens as f16 pairs
            const uint32_t d_tmem = tmem + kP8OCol;
            if (tile == 0)                                    // the first tile of the item overwrites
              umma_bf16_ts_lo<false>(d_tmem, p_tmem, v_lo, dv_hi, idesc);
            else
              umma_bf16_ts_lo<true>(d_tmem, p_tmem, v_lo, dv_hi, idesc);
#pragma unroll
            for (int ks = 1; ks < kPfTile / 16; ++ks)
              umma_bf16_ts_lo<true>(d_tmem, p_tmem + ks * 8, v_lo + (uint32_t)((ks * 2048) >> 4), dv_hi, idesc);
            umma_commit(&sm.pv_done[g]);
          }
          umma_commit(&sm.o_done);
        }
        umma_commit(&sm.mma_idle[1]);
        mbar_wait_landed(&sm.mma_idle[1], 0);
      }
      __syncwarp();
    }
  } else if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(P8Regs<kOnePage>::kSoftmax));
    // -------------------------------- softmax --------------------------------
    const int g = warp >> 2;                         // group: KV tiles whose running index & 1 == g
    const int r = threadIdx.x & 127;                 // query row of the tile == TMEM lane
    const uint32_t lane_base = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t o_col = lane_base + kP8OCol;
    const uint32_t p_col = lane_base + kP8PCol + g * 64;
    const int G = p.group;
    uint32_t it = 0;
#pragma unroll 1
    for (uint32_t item_no = 0;; ++item_no) {
      PrefillPiece item;
      if (take_item(item_no, item) < 0) break;
      const int rg = item.row0 + r;
      const bool valid = rg < item.q_len * G;
      // rows past the item's see whatever there is: nobody reads their O
      const int lim = (valid ? min(item.causal_base + rg / G, item.kv_len - 1) : INT_MAX) - first_of(item) * kPfTile;
      const bool idle = !__any_sync(0xffffffffu, valid);
      mbar_wait_limited(&sm.q_full[item_no & 1u], (item_no >> 1) & 1u, abort_at);
      const float row_factor = sm.row_factor[item_no & 1u][r];
      float m = -INFINITY;           // running maximum of this group's scores: what its row sum is scaled to
      float l = 0.f;
#pragma unroll 1
      for (int tile = 0; tile < item.n_tiles; ++tile, ++it) {
        if ((int)(it & 1u) != g) continue;             // the other group's tile
        const uint32_t sb = it & 1u;
        const uint32_t s_col = lane_base + sb * 128;
        constexpr int kN = kOnePage ? 1 : kP8Groups;   // pairs of scales of a tile
        const uint32_t sl = it % kP8ScaleSlots;
        mbar_wait_limited(&sm.s_full[sb], (it >> 1) & 1u, abort_at);
        tc_fence_after();
        if (idle) {                                    // no row of this warp counts: keep the barriers going
          mbar_arrive(&sm.s_empty[sb]);
          // Never ahead of the group: a phase of m_ready and p_full gets one arrival a thread.  The first wait is for an item
          // before in which the others had work to do, the second for one behind where this warp has and does not look back.
          if (it >= 2) mbar_wait_limited(&sm.p_full[g], ((it - 2) >> 1) & 1u, abort_at);
          mbar_arrive(&sm.m_ready[it & 1u]);
          mbar_arrive(&sm.p_full[g]);
          mbar_wait_limited(&sm.p_full[g], (it >> 1) & 1u, abort_at);
          continue;
        }
        // Columns past the row's limit become -inf in place, a quarter of the row at a time: few tiles need it, and code
        // that runs rarely is fetched from far away each time (unrolled over the row it cost 3000 cycles a tile).
        const int last_col = lim - tile * kPfTile;
        if (__builtin_expect(__any_sync(0xffffffffu, last_col < kPfTile - 1), 0)) {
#pragma unroll 1
          for (int c0 = 0; c0 < kPfTile; c0 += 32) {
            uint32_t x[32];
            tmem_ld32(s_col + c0, x);
            tmem_wait_ld();
#pragma unroll
            for (int c = 0; c < 32; ++c) x[c] = c0 + c > last_col ? 0xff800000u : x[c];
            tmem_st32(s_col + c0, x);
          }
          tmem_wait_st();
        }
        // The whole score row goes to registers in one go and the S buffer straight back to
        // the MMA issuer.
        uint32_t sv[4][32];
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4) tmem_ld32(s_col + q4 * 32, sv[q4]);
        mbar_wait_limited(&sm.scale_full[sl], (it / kP8ScaleSlots) & 1u, abort_at);
        float f[kN], lv[kN];                           // product -> log2 score; log2 of V's scale
#pragma unroll
        for (int i = 0; i < kN; ++i) {
          f[i] = row_factor * sm.tile_scale[sl][0][i];
          // not 0, which would make NaN of the -inf that masks (a NaN scale stays NaN)
          f[i] = f[i] < 1.17549435e-38f ? 1.17549435e-38f : f[i];
          lv[i] = fast_log2(sm.tile_scale[sl][1][i]);
        }
        // the reference O is scaled to after the previous tile (owned by the other group)
        float m_in = -INFINITY;
        if (tile > 0) {
          mbar_wait_limited(&sm.m_ready[(it - 1) & 1u], ((it - 1) >> 1) & 1u, abort_at);
          m_in = sm.row_ms[(it - 1) & 1u][r];
        }
        tmem_wait_ld();
        tc_fence_before();
        mbar_arrive(&sm.s_empty[sb]);
        // maximum of the scores, and of the scores plus log2 of V's scale
        float mx = -INFINITY, my = -INFINITY;
        {
          float mq[8];                      // one chain per column group
#pragma unroll
          for (int u = 0; u < 8; ++u)
            mq[u] = fmaxf(__uint_as_float(sv[u >> 1][(u & 1) * 16]), __uint_as_float(sv[u >> 1][(u & 1) * 16 + 1]));
#pragma unroll
          for (int c = 2; c < 16; c += 2)
#pragma unroll
            for (int u = 0; u < 8; ++u)
              mq[u] = fmax3(mq[u], __uint_as_float(sv[u >> 1][(u & 1) * 16 + c]),
                            __uint_as_float(sv[u >> 1][(u & 1) * 16 + c + 1]));
          if constexpr (kOnePage) {
            mx = fmaxf(fmax3(mq[0], mq[1], mq[2]), fmax3(fmax3(mq[3], mq[4], mq[5]), mq[6], mq[7])) * f[0];
            my = mx + (lv[0] - kP8Lift);
          } else {
#pragma unroll
            for (int u = 0; u < 8; ++u) {
              const float x = mq[u] * f[u];
              mx = fmaxf(mx, x);
              my = fmaxf(my, x + lv[u]);
            }
            my -= kP8Lift;
          }
        }
        // lazy rescale: only when some row of the warp outgrew the stale reference
        const bool grow = my - m_in > kP8Lazy || (m_in == -INFINITY && my > -INFINITY);
        const bool rescale = __any_sync(0xffffffffu, grow);
        const float m_used = rescale ? fmaxf(m_in, my) : m_in;
        sm.row_ms[it & 1u][r] = m_used;
        mbar_arrive(&sm.m_ready[it & 1u]);             // release: the next tile's owner may go on
        const float m_new = fmaxf(m, mx);
        const float m_sub = m_new == -INFINITY ? 0.f : m_new;
        l *= fast_exp2(m - m_sub);                     // m = -inf: l is 0
        m = m_new;
        const float o_sub = m_used == -INFINITY ? 0.f : m_used;
        // w = 2^(x + lv - o_sub) = p 2^e with p = 2^(x - m) and e uniform over a column group; the row sum
        // takes 2^-e sum w.  Below 2^-60 a weight is 0 in f16 whatever it is: e stops there so that p
        // itself is not lost from the sum.
        float shift[kN], undo[kN];
#pragma unroll
        for (int i = 0; i < kN; ++i) {
          float e = m_sub + lv[i] - o_sub;
          e = e < -60.f ? -60.f : e > 120.f ? 120.f : e;
          shift[i] = e - m_sub;
          undo[i] = fast_exp2(-e);
        }
        // The group's P buffer is free once the P V of its previous tile (of this item or the
        // one before) has run.  The group waited for the one before that two tiles ago, so
        // the parity wait cannot be off by a phase.
        if (it >= 2) {
          mbar_wait_limited(&sm.pv_done[g], ((it - 2) >> 1) & 1u, abort_at);
          tc_fence_after();
        }
        // O may be touched once the previous tile's P V (the other group's) has run: rare path
        if (rescale && tile > 0) {
          const float corr = (m_in == -INFINITY) ? 0.f : fast_exp2(m_in - m_used);
          mbar_wait_limited(&sm.pv_done[g ^ 1], ((it - 1) >> 1) & 1u, abort_at);
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            uint32_t orow[32];
            tmem_ld32(o_col + c * 32, orow);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) orow[i] = __float_as_uint(__uint_as_float(orow[i]) * corr);
            tmem_st32(o_col + c * 32, orow);
          }
        }
        // Weights, software-pipelined by a quarter of the row: the exponentials of quarter q are issued while
        // quarter q - 1 is summed and packed.  P (f16 pairs) goes to the group's buffer 64 columns at a time.
        float2 ls[4] = {{0.f, 0.f}, {0.f, 0.f}, {0.f, 0.f}, {0.f, 0.f}};
        uint32_t pk[32];
#pragma unroll
        for (int q4 = 0; q4 <= 4; ++q4) {
#pragma unroll
          for (int c = 0; c < 32; c += 2) {
            if (q4 < 4) {
              const int u = kOnePage ? 0 : q4 * 2 + (c >> 4);
              const float2 x = __ffma2_rn(make_float2(__uint_as_float(sv[q4][c]), __uint_as_float(sv[q4][c + 1])),
                                          make_float2(f[u], f[u]), make_float2(shift[u], shift[u]));
              sv[q4][c] = __float_as_uint(fast_exp2(x.x));
              sv[q4][c + 1] = __float_as_uint(fast_exp2(x.y));
            }
            if (q4 > 0) {
              const float2 pp = make_float2(__uint_as_float(sv[q4 - 1][c]), __uint_as_float(sv[q4 - 1][c + 1]));
              if constexpr (kOnePage) {
                ls[(c >> 1) & 3] = __fadd2_rn(ls[(c >> 1) & 3], pp);
              } else {
                const int u = (q4 - 1) * 2 + (c >> 4);
                ls[(c >> 1) & 3] = __ffma2_rn(pp, make_float2(undo[u], undo[u]), ls[(c >> 1) & 3]);
              }
              pk[((q4 - 1) & 1) * 16 + (c >> 1)] = pack_f16(pp.x, pp.y);
            }
          }
          if (q4 == 2) tmem_st32(p_col, pk);
          if (q4 == 4) tmem_st32(p_col + 32, pk);
        }
        {
          const float2 a = __fadd2_rn(ls[0], ls[1]), b = __fadd2_rn(ls[2], ls[3]);
          const float sum = (a.x + a.y) + (b.x + b.y);
          l += kOnePage ? sum * undo[0] : sum;
        }
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&sm.p_full[g]);
      }
      // ---- hand the row sums to the convert warps and go on with the next item
      // the references only grow along the tiles: the last tile's is what O is scaled to
      float mm = -INFINITY;
      if (item.n_tiles > 0) {
        mbar_wait_limited(&sm.m_ready[(it - 1) & 1u], ((it - 1) >> 1) & 1u, abort_at);
        mm = sm.row_ms[(it - 1) & 1u][r];
      }
      if (item_no > 0) mbar_wait_limited(&sm.l_empty, (item_no - 1) & 1u, abort_at);
      sm.row_l[g][r] = l;
      sm.row_m[g][r] = m;
      if (g == 0) sm.row_mfin[r] = mm;
      mbar_arrive(&sm.l_full);
    }
  } else {
    // ------------------- convert: Q terms, V to f16, epilogue -------------------
    // Thread e owns query row e: it stages the row's two e4m3 terms while the item before is worked on, and takes row e
    // of O out of tensor memory at the end.  In between the 128 threads turn each V tile's codes into f16, one tile
    // ahead of its P V or more.
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(P8Regs<kOnePage>::kConvert));
    const int r = threadIdx.x - (kP8Threads - kP8ConvertThreads);
    const uint32_t o_col = tmem + ((uint32_t)((warp & 3) * 32) << 16) + kP8OCol;
    const int G = p.group;
    uint32_t it = 0;                                 // next V tile to convert, over all items
    // Q of the next item: thread e quantises row e.  Its largest magnitude is looked for first, then eight steps convert 16
    // elements each behind the item's last V tiles; what a step loads arrives while a tile is converted.  (All at once
    // before the last V tile it took 10000 cycles, and that tile's P V and the next item's first S waited for it.)
    constexpr int kSteps = 8;
    const uint4* q_row = nullptr;                    // null: a row past the item's, zeros
    int step = kSteps;                               // next step of the item; kSteps: none
    float up = 0.f, row_factor = 0.f;
    uint4 raw[2];
    auto load_step = [&]() {
#pragma unroll
      for (int i = 0; i < 2; ++i) raw[i] = q_row ? q_row[2 * step + i] : make_uint4(0u, 0u, 0u, 0u);
    };
    struct Row {                                     // what this thread keeps of an item
      int n_tiles, kv_len;                           // keys from the item's first tile on
      int partial;                                   // record of a piece of a cut item, or -1
      int64_t out;                                   // its row e among the rows of `out`, or -1
    };
    auto begin_q = [&](const PrefillPiece& x) -> Row {
      const bool fits = x.q_start + x.q_len <= p.num_tokens;
      const int rg = x.row0 + r;
      if (r == 0 && !fits && p.status) atomicOr(p.status, B200_STATUS_BAD_LAUNCH);
      const bool valid = fits && rg < x.q_len * G;
      const int64_t tok = x.q_start + rg / G;
      const int head = x.kv_head * G + rg % G;
      q_row = valid ? reinterpret_cast<const uint4*>(p.q + tok * p.q_stride + (int64_t)head * kPfHeadDim) : nullptr;
      step = 0;
      uint32_t top = 0;                              // maxima of the even and the odd elements
#pragma unroll 1
      for (int c0 = 0; c0 < 16 && valid; c0 += 8) {
        uint4 v[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) v[c] = q_row[c0 + c];
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const uint32_t a = __vmaxu2(v[c].x & 0x7fff7fffu, v[c].y & 0x7fff7fffu);
          const uint32_t b = __vmaxu2(v[c].z & 0x7fff7fffu, v[c].w & 0x7fff7fffu);
          top = __vmaxu2(top, __vmaxu2(a, b));
        }
      }
      // exponent field of the largest; 8 and more: both factors are normal
      const int e = max((int)(max(top & 0xffffu, top >> 16) >> 7), 8);
      // 2^(7 - (e - 127)) with the sign of the softmax scale, so that the factor behind the product is not negative: the
      // softmax threads take the maximum of a row, and mask it, before they multiply.  Any inf or NaN: the row is NaN.
      up = e == 255 ? NAN : copysignf(__uint_as_float((uint32_t)(261 - e) << 23), p.scale_log2);
      row_factor = __uint_as_float((uint32_t)(e - 7) << 23) * fabsf(p.scale_log2);
      return Row{x.n_tiles, x.kv_len - first_of(x) * kPfTile, kCut ? x.partial : -1, valid ? tok * p.num_q_heads + head : -1};
    };
    auto put_step = [&](uint32_t k) {
      if (step == 0) {
        // the buffers' last reader is the item two before: its S has run, its softmax (the epilogue waited for it) is over
        mbar_wait_limited(&sm.q_empty[k & 1u], ((k >> 1) & 1u) ^ 1u, abort_at);
        sm.row_factor[k & 1u][r] = row_factor;
      }
      const uint32_t w[8] = {raw[0].x, raw[0].y, raw[0].z, raw[0].w, raw[1].x, raw[1].y, raw[1].z, raw[1].w};
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        uint32_t h[2], l[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          // f16 holds what e4m3 can: elements under 2^-14 here are rounded to 0 by either
          const uint32_t x = pack_f16(__uint_as_float(w[i + j] << 16) * up, __uint_as_float(w[i + j] & 0xffff0000u) * up);
          h[j] = f16x2_to_e4m3x2(x);
          const uint32_t back = e4m3x2_to_f16x2((uint16_t)h[j]);
          const __half2 rest = __hsub2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&back));
          l[j] = f16x2_to_e4m3x2(*reinterpret_cast<const uint32_t*>(&rest));
        }
        hi[i >> 1] = __byte_perm(h[0], h[1], 0x5410);
        lo[i >> 1] = __byte_perm(l[0], l[1], 0x5410);
      }
      const uint32_t at = swz128(r, step);
      *reinterpret_cast<uint4*>(sm.q[k & 1u][0] + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
      *reinterpret_cast<uint4*>(sm.q[k & 1u][1] + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      if (step == kSteps - 1) {
        fence_proxy_async_smem();
        mbar_arrive(&sm.q_full[k & 1u]);
      }
      ++step;
    };
    // Bank conflicts: the eight lanes of a phase read and write 16-byte chunks of two rows, four chunks (half a row of
    // codes) each.  Under the 128-byte swizzle a row's chunk number is XOR-ed with row & 7; rows whose numbers
    // differ by 5 in those bits cover all banks both ways: reading, the four chunks of one row and the other four of
    // the other (bit 2); writing 16 codes as two chunks of f16, even chunks of one row and odd ones of the other (bit 0).
    const int pair = lane >> 3;                                    // rows {0,5}, {1,4}, {2,7}, {3,6} of each eight
    const int row0 = (warp & 3) * 32 + (lane & 4 ? pair ^ 5 : pair);
    // rows row0 + 8 i share row & 7: i is a constant offset, the other chunks are XORs of a constant
    const uint32_t rd_at = swz128(row0, lane & 3), wr_at = swz128(row0, 2 * (lane & 3));
    auto convert = [&](int kv_len, int step) {
      const int have = kv_len - step * kPfTile;                  // rows past the end are zero: 0 x NaN is NaN
      const int sv = it % kP8VStages, b = it & 1u;
      mbar_wait_limited(&sm.v_full[sv], (it / kP8VStages) & 1u, abort_at);
      if (it >= 2) mbar_wait_limited(&sm.pv_done[b], ((it - 2) >> 1) & 1u, abort_at);
#pragma unroll 1
      for (int half = 0; half < 2; ++half) {
        uint4 v[4];
        const uint8_t* const src = sm.v[sv] + (rd_at ^ (uint32_t)(64 * half));
#pragma unroll
        for (int i = 0; i < 4; ++i)
          v[i] = *reinterpret_cast<const uint4*>(src + 1024 * i);
        if (have < kPfTile) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (row0 + 8 * i >= have) v[i] = make_uint4(0u, 0u, 0u, 0u);
        }
        uint8_t* const dst = sm.v16[b] + half * kP8TileBytes;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
          for (int j = 0; j < 2; ++j)
            *reinterpret_cast<uint4*>(dst + (wr_at ^ (uint32_t)(16 * j)) + 1024 * i) =
                make_uint4(e4m3x2_to_f16x2((uint16_t)w[2 * j]), e4m3x2_to_f16x2((uint16_t)(w[2 * j] >> 16)),
                           e4m3x2_to_f16x2((uint16_t)w[2 * j + 1]), e4m3x2_to_f16x2((uint16_t)(w[2 * j + 1] >> 16)));
        }
      }
      mbar_arrive(&sm.v_empty[sv]);
      fence_proxy_async_smem();
      mbar_arrive(&sm.v16_full[b]);
      ++it;
    };
    // One instance of each piece of code (see the producer): iteration k works on item k - 1, whose Q was staged in the
    // iteration before; it stages item k behind its own last V tiles and writes item k - 2 behind its first.
    Row item{0, 0, -1, -1}, prev = item, next = item;
    int total = -1;                                  // items of this CTA, once known
#pragma unroll 1
    for (int k = 0; total < 0 || k < total + 2; ++k) {
      const int n = item.n_tiles;
      const int take_at = n > kSteps + 1 ? n - kSteps - 1 : 0;
#pragma unroll 1
      for (int tile = 0; tile == 0 || tile < n || step < kSteps; ++tile) {
        if (total < 0 && tile == take_at) {
          PrefillPiece rec;
          if (take_item(k, rec) >= 0)
            next = begin_q(rec);
          else
            total = k;
        }
        const bool stage = step < kSteps && (tile > 0 || k < 2);
        if (stage) load_step();
        if (tile < n) convert(item.kv_len, tile);
        if (stage) put_step(k);
        if (tile > 0 || k < 2) continue;
        const uint32_t item_no = k - 2;
        // ---- epilogue: row e of O out of tensor memory as soon as the item's last P V has run
        // a piece of a cut item leaves normalised fp32 rows and their log2 sums in its record
        const bool cut = kCut && prev.partial >= 0, to_f32 = cut || p.out_is_f32;
        const bool fits = !kCut || prev.partial < p.max_partials, valid = prev.out >= 0 && fits;
        if (!fits && r == 0 && p.status) atomicOr(p.status, B200_STATUS_BAD_LAUNCH);
        uint8_t* const row_at = cut ? reinterpret_cast<uint8_t*>(p.part + (int64_t)prev.partial * kPieceRecFloats + r * kPfHeadDim)
                                    : static_cast<uint8_t*>(p.out) + prev.out * (kPfHeadDim * (to_f32 ? 4 : 2));
        mbar_wait_limited(&sm.l_full, item_no & 1u, abort_at);
        const float m0 = sm.row_m[0][r], m1 = sm.row_m[1][r], mo = sm.row_mfin[r];
        const float mm = fmaxf(m0, m1);
        // Which group had the item's even tiles depends on what the CTA worked on before: the two products
        // are rounded alike (no fused multiply-add), so that the sum does not.
        const float lsum = mm == -INFINITY ? sm.row_l[0][r] + sm.row_l[1][r]
                                           : __fadd_rn(__fmul_rn(sm.row_l[0][r], fast_exp2(m0 - mm)),
                                                       __fmul_rn(sm.row_l[1][r], fast_exp2(m1 - mm)));
        mbar_arrive(&sm.l_empty);
        // O is in units of 2^(mo - kP8Lift), the sum in units of 2^mm; the factor between them in two halves, each of
        // which fp32 holds however far apart they are
        const float half_unit = fast_exp2((mo - (mm == -INFINITY ? 0.f : mm)) * 0.5f);
        const float inv = half_unit / lsum;
        const bool empty = lsum == 0.f;      // no visible key: zeros, whatever the accumulator holds
        mbar_wait_limited(&sm.o_done, item_no & 1u, abort_at);
        tc_fence_after();
#pragma unroll 1
        for (int q4 = 0; q4 < 4; ++q4) {
          uint32_t o[32];
          tmem_ld32(o_col + q4 * 32, o);
          tmem_wait_ld();
          if (q4 == 3) {                       // the whole row is out of tensor memory
            tc_fence_before();
            mbar_arrive(&sm.o_free);
          }
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            float2 x = __fmul2_rn(make_float2(__uint_as_float(o[i]), __uint_as_float(o[i + 1])), make_float2(half_unit, half_unit));
            x = __fmul2_rn(x, make_float2(inv, inv));
            o[i] = __float_as_uint(x.x);
            o[i + 1] = __float_as_uint(x.y);
          }
          if (empty) {
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = 0u;
          }
          if (valid) {
            if (to_f32) {
              uint4* dst = reinterpret_cast<uint4*>(row_at + q4 * 128);
#pragma unroll
              for (int i = 0; i < 8; ++i) dst[i] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
            } else {
              uint4* dst = reinterpret_cast<uint4*>(row_at + q4 * 64);
#pragma unroll
              for (int i = 0; i < 32; i += 8) {
                uint4 v;
                v.x = pack_bf16(__uint_as_float(o[i]), __uint_as_float(o[i + 1]));
                v.y = pack_bf16(__uint_as_float(o[i + 2]), __uint_as_float(o[i + 3]));
                v.z = pack_bf16(__uint_as_float(o[i + 4]), __uint_as_float(o[i + 5]));
                v.w = pack_bf16(__uint_as_float(o[i + 6]), __uint_as_float(o[i + 7]));
                dst[i >> 3] = v;
              }
            }
          }
        }
        if (valid) {
          if (kCut && prev.partial >= 0)
            p.part[(int64_t)prev.partial * kPieceRecFloats + kPfRows * kPfHeadDim + r] = empty ? -INFINITY : mm + fast_log2(lsum);
          else if (p.lse_out)
            p.lse_out[prev.out] = empty ? -INFINITY : mm * 0.6931471805599453f + __logf(lsum);
        }
      }
      prev = item;
      item = next;
      if (total == k) item.n_tiles = 0;
    }
  }
  // ---- teardown: everyone is done with tensor memory before it is released
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, kP8TmemCols);
  }
  // the last CTA to leave puts the queue back to zero for the next launch on this plan
  if (threadIdx.x == 0) {
    if (*abort_flag && p.status) atomicOr(p.status, B200_STATUS_WAIT_TIMEOUT);
    __threadfence();
    if (atomicAdd(p.work_counter + 1, 1) == (int)gridDim.x - 1) {
      p.work_counter[0] = 0;
      p.work_counter[1] = 0;
      __threadfence();
    }
  }
}

// Joins the pieces of cut items, a warp a row: the rows of a piece are normalised, the weights of the pieces are
// their sums 2^(log2 sum).  The order of the tiles is the order of the sum.  Bound by latency (at most 20 MB of records).
// A kernel of its own: inside the other one, by the last CTA to arrive, its registers cost every item 4 % and more.
__global__ void __launch_bounds__(256)
prefill_join_kernel(const Prefill8Params p) {
  grid_dep_wait();
  const int first_group = p.plan[kHdrOffGroups];
  // groups lie behind the pieces, to the end of what the header counts
  if (p.plan[kHdrPieces] == 0 || (int)blockIdx.x >= p.plan[kHdrGroups]) return;
  const PieceGroup g = reinterpret_cast<const PieceGroup*>(p.plan + first_group)[blockIdx.x];
  const int r = blockIdx.y * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int rg = g.row0 + r;
  if (rg >= g.q_len * p.group || g.q_start + g.q_len > p.num_tokens || g.part_begin + g.n_parts > p.max_partials) return;
  const float* const rec = p.part + (int64_t)g.part_begin * kPieceRecFloats;
  const float* const sums = rec + kPfRows * kPfHeadDim + r;
  float top = -INFINITY;
#pragma unroll 4
  for (int i = 0; i < g.n_parts; ++i) top = fmaxf(top, sums[(int64_t)i * kPieceRecFloats]);
  const float ref = top == -INFINITY ? 0.f : top;
  float total = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int i = 0; i < g.n_parts; ++i) {
    const float w = fast_exp2(sums[(int64_t)i * kPieceRecFloats] - ref);
    const float4 y = *reinterpret_cast<const float4*>(rec + (int64_t)i * kPieceRecFloats + r * kPfHeadDim + 4 * lane);
    total += w;
    acc.x += w * y.x;
    acc.y += w * y.y;
    acc.z += w * y.z;
    acc.w += w * y.w;
  }
  const float inv = total == 0.f ? 0.f : 1.f / total;
  const int64_t row = (int64_t)(g.q_start + rg / p.group) * p.num_q_heads + g.kv_head * p.group + rg % p.group;
  if (p.out_is_f32) {
    reinterpret_cast<float4*>(p.out)[row * 32 + lane] = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
  } else {
    reinterpret_cast<uint2*>(p.out)[row * 32 + lane] =
        make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
  }
  if (p.lse_out && lane == 0) p.lse_out[row] = total == 0.f ? -INFINITY : (top + fast_log2(total)) * 0.6931471805599453f;
}

}  // namespace b200

// Bytes that the pieces and groups of a plan of at most num_items items take at its end.
extern "C" size_t b200_prefill_split_bytes(int num_items, int num_ctas) {
  using namespace b200;
  if (num_items < 0 || num_ctas <= 0) return 0;
  return sizeof(PrefillPiece) * ((size_t)num_items + num_ctas) + sizeof(PieceGroup) * (size_t)num_ctas;
}
extern "C" size_t b200_prefill_split_workspace_bytes(int num_partials) {
  return num_partials < 0 ? 0 : sizeof(float) * b200::kPieceRecFloats * (size_t)num_partials;
}

// Where few items meet many SMs the longest sets the time.  The tiles are then dealt to num_ctas equal shares in the
// order of the list, items are cut where a share ends, and the pieces are sorted by length: handed out longest first, the
// big ones fill most of a share and the small ones what is left.
extern "C" int b200_prefill_split(int32_t* plan, size_t plan_bytes, int num_ctas, b200_prefill_plan_info* info,
                                  int* num_partials) try {
  using namespace b200;
  if (!plan || !info || !num_partials || num_ctas <= 0 || num_ctas > kMaxGroups || plan[0] != kPfMagic || info->num_items != plan[1]) {
    set_last_error("prefill_split: null pointer, no CTAs, or not a plan of b200_prefill_plan");
    return B200_EINVAL;
  }
  const int n = info->num_items;
  const PrefillItem* items = reinterpret_cast<const PrefillItem*>(plan + kPlanHeaderInts);
  const int base = kPlanHeaderInts + kPfItemInts * n;
  if (plan_bytes < base * sizeof(int32_t) + b200_prefill_split_bytes(n, num_ctas)) {
    set_last_error("prefill_split: plan buffer of %zu bytes is smaller than b200_prefill_split_bytes() asks for", plan_bytes);
    return B200_EPLAN;
  }
  for (int i = kHdrPieces; i <= kHdrGroups; ++i) plan[i] = 0;
  info->plan_ints = base;
  *num_partials = 0;
  constexpr int kLeast = 4;                                  // tiles of a piece
  int64_t total = 0, all_rows = 0;
  for (int i = 0; i < n; ++i) {
    total += items[i].n_tiles;
    all_rows += std::min(items[i].q_len * plan[kHdrHeadGroup] - items[i].row0, kPfRows);
  }
  if (n == 0 || total == 0 || n > 4 * num_ctas) return B200_OK;
  const float longest = (float)items[0].n_tiles, share = (float)total / num_ctas, rounds = (float)n / num_ctas;
  // What an item or piece costs besides its tiles, and the join, in tiles: fitted to steps measured both ways (four
  // 512-token chunks 122 us cut, 106 whole; three odd sequences 113 and 99; 16 drafts of 20 rows 38 and 42, or 53 and 69
  // over longer contexts; 2 x 64 rows over 32768 tokens 85 and 262).
  const float filled = (float)all_rows / ((float)n * kPfRows);
  const float item_cost = 3.f + 5.f * filled, join_cost = 2.f + 2.f * filled;
  const int per = std::max((int)std::ceil(share), 2 * kLeast);
  // the list is sorted: items[0] is the longest
  const float whole = rounds <= 1.f ? longest + item_cost
                                    : std::min(std::ceil(rounds) * (longest + item_cost),
                                               share + longest / 2 + item_cost * (rounds + 1));
  const float cut = per + item_cost * (rounds + 2) + join_cost;
  if (cut > 0.93f * whole) return B200_OK;

  std::vector<PrefillPiece> pieces;
  std::vector<PieceGroup> groups;
  pieces.reserve(n + num_ctas);
  int room = per, spare = num_ctas;                          // tiles left of the share; cuts the buffer has room for
  for (int i = 0; i < n; ++i) {
    const PrefillItem& x = items[i];
    const size_t first = pieces.size();
    int begin = 0;
    do {
      const int left = x.n_tiles - begin;
      int take = std::min(left, room);
      if (left - take < kLeast || spare == 0) take = left;   // no sliver behind a cut
      if (take < left) --spare;
      pieces.push_back(PrefillPiece{x.seq, x.kv_head, x.row0, take, x.kv_len, x.q_start, x.q_len, x.causal_base, begin,
                                    -1, 0, 0});
      begin += take;
      room -= take;
      if (room < kLeast) room += per;
    } while (begin < x.n_tiles);
    const int parts = (int)(pieces.size() - first);
    if (parts > 1) {
      for (int k = 0; k < parts; ++k) pieces[first + k].partial = *num_partials + k;
      groups.push_back(PieceGroup{*num_partials, parts, x.kv_head, x.row0, x.q_start, x.q_len, 0, 0});
      *num_partials += parts;
    }
  }
  if (groups.empty()) return B200_OK;
  // longest first, by counting: the list is made on the way of a step
  const int most = (int)longest + kLeast;
  std::vector<int> at(most + 2, 0);
  for (const PrefillPiece& x : pieces) ++at[most - std::min(x.n_tiles, most) + 1];
  for (int k = 0; k <= most; ++k) at[k + 1] += at[k];
  PrefillPiece* sorted = reinterpret_cast<PrefillPiece*>(plan + base);
  for (const PrefillPiece& x : pieces) sorted[at[most - std::min(x.n_tiles, most)]++] = x;
  const int off_groups = base + kPieceInts * (int)pieces.size();
  memcpy(plan + off_groups, groups.data(), groups.size() * sizeof(PieceGroup));
  plan[kHdrPieces] = (int)pieces.size();
  plan[kHdrOffPieces] = base;
  plan[kHdrOffGroups] = off_groups;
  plan[kHdrGroups] = (int)groups.size();
  info->plan_ints = off_groups + kPieceGroupInts * (int)groups.size();
  return B200_OK;
} catch (const std::exception& e) {
  b200::set_last_error("prefill_split: %s", e.what());
  return B200_ETOOLARGE;
}

extern "C" int b200_paged_prefill_gqa_fp8(const void* q, int64_t q_stride, const void* key_cache,
                                          const void* value_cache, const float* key_scale,
                                          const float* value_scale, int num_blocks, int block_size,
                                          const int32_t* block_table, int64_t bt_stride, int table_rows,
                                          int table_cols, int32_t* plan_dev, const b200_prefill_plan_info* info,
                                          int max_ctas, int num_tokens, int num_q_heads, int num_kv_heads,
                                          int head_dim, float scale, void* workspace, size_t workspace_bytes, void* out,
                                          int out_is_f32, float* lse_out, int32_t* status, void* stream) {
  using namespace b200;
  const char* who = "paged_prefill_gqa_fp8";
  int rc = check_fp8_cache(who, key_cache, value_cache, key_scale, value_scale, num_blocks, block_size, num_kv_heads,
                           head_dim);
  if (rc) return rc;
  if (info && info->num_items == 0) return B200_OK;
  if (!q || !block_table || !plan_dev || !out || num_q_heads <= 0 || num_q_heads % num_kv_heads || num_tokens < 0 ||
      max_ctas < 0 || table_rows <= 0 || table_cols <= 0) {
    set_last_error("%s: null pointer, bad head counts, a negative size or an empty block table", who);
    return B200_EINVAL;
  }
  if (reinterpret_cast<uintptr_t>(q) % 16 || q_stride % 8 || q_stride < (int64_t)num_q_heads * head_dim ||
      reinterpret_cast<uintptr_t>(out) % 16 || reinterpret_cast<uintptr_t>(plan_dev) % 16 ||
      reinterpret_cast<uintptr_t>(workspace) % 16) {
    set_last_error("%s: q, out, plan and workspace must be 16-byte aligned, the q token stride a multiple of 8 elements and >= Hq*D", who);
    return B200_EALIGN;
  }
  const int box_tokens = block_size < kPfTile ? block_size : kPfTile;
  CUtensorMap k_map, v_map;
  rc = get_fp8_cache_tensor_map(key_cache, num_blocks, block_size, num_kv_heads, box_tokens, &k_map);
  if (rc) return rc;
  rc = get_fp8_cache_tensor_map(value_cache, num_blocks, block_size, num_kv_heads, box_tokens, &v_map);
  if (rc) return rc;

  Prefill8Params p;
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
  const size_t records = workspace ? workspace_bytes / (kPieceRecFloats * sizeof(float)) : 0;
  p.max_partials = records > INT32_MAX ? INT32_MAX : (int)records;
  p.work_counter = plan_dev + 2;
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
  p.boxes_per_tile = kPfTile / box_tokens;
  p.out_is_f32 = out_is_f32;
  p.scale_log2 = scale * 1.4426950408889634f;

  const bool one_page = block_size >= kPfTile;
  const bool cut = records > 0;
  auto kernel = one_page ? (cut ? paged_prefill_fp8_kernel<true, true> : paged_prefill_fp8_kernel<true, false>)
                         : (cut ? paged_prefill_fp8_kernel<false, true> : paged_prefill_fp8_kernel<false, false>);
  const size_t smem = sizeof(Prefill8Smem);
  static bool attr_set[4][64] = {{false}};
  const int variant = 2 * one_page + cut;
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 64 || !attr_set[variant][dev]) {
    rc = check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem),
                    "paged_prefill_gqa_fp8 smem attribute");
    if (rc) return rc;
    if (dev < 64) attr_set[variant][dev] = true;
  }
  int grid = b200_sm_count();
  if (grid <= 0) grid = 148;
  if (info && !records && grid > info->num_items) grid = info->num_items;     // a cut plan has more pieces than items
  if (max_ctas > 0 && grid > max_ctas) grid = max_ctas;     // the rest of the SMs are left to another kernel
  rc = check_cuda(launch_pdl(kernel, dim3(grid), dim3(kP8Threads), smem, static_cast<cudaStream_t>(stream), k_map, v_map,
                             p),
                  "paged_prefill_gqa_fp8 launch");
  const int groups = p.max_partials / 2 < kMaxGroups ? p.max_partials / 2 : kMaxGroups;   // a cut item has two records or more
  if (rc || groups == 0) return rc;
  return check_cuda(launch_pdl(prefill_join_kernel, dim3(groups, kPfRows / 8), dim3(256), 0,
                               static_cast<cudaStream_t>(stream), p),
                    "paged_prefill_gqa_fp8 join launch");
}
