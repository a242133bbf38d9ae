// Work items of the wide-query attention kernels (16-bit and 8-bit caches).  The host plan is
//   [header: magic, item count, two words the kernels use as work-queue counters, ...]
//   [PrefillItem records, longest first]
// and, when b200_prefill_split has cut items along the keys for the 8-bit kernel (header: number of pieces, where they
// begin, where the groups begin and how many there are; all 0 in an uncut plan),
//   [PrefillPiece records, longest first] [PieceGroup records]
#pragma once
#include "common.cuh"
#include "decode_plan.h"

namespace b200 {

constexpr int kPfHeadDim = 128;
constexpr int kPfRows = 128;                                   // packed query rows per item
constexpr int kPfTile = 128;                                    // KV tokens per tile
constexpr int kPfItemInts = 8;
constexpr int kPfMagic = 0x70663030;

struct PrefillItem {
  int32_t seq, kv_head, row0, n_tiles;        // row0: first packed row of the pair this item owns
  int32_t kv_len, q_start, q_len, causal_base;
};
static_assert(sizeof(PrefillItem) == kPfItemInts * 4, "item layout");

// A run of an item's tiles: all of them, or one of several whose partial results are merged.
struct PrefillPiece {
  int32_t seq, kv_head, row0, n_tiles;        // n_tiles: of the piece
  int32_t kv_len, q_start, q_len, causal_base;
  int32_t tile_begin, partial, unused[2];     // partial: record of the piece's result, -1: the piece is the whole item
};
struct PieceGroup {                           // a cut item: its records lie one after the other, in the order of the tiles
  int32_t part_begin, n_parts;
  int32_t kv_head, row0, q_start, q_len;
  int32_t unused[2];
};
constexpr int kPieceInts = 12, kPieceGroupInts = 8;
constexpr int kHdrPieces = 4, kHdrOffPieces = 5, kHdrOffGroups = 6, kHdrGroups = 7;
constexpr int kHdrHeadGroup = 8;                                // query heads of a kv head
constexpr int kPieceRecFloats = kPfRows * kPfHeadDim + kPfRows;   // normalised rows, then their log2 sums
static_assert(sizeof(PrefillPiece) == kPieceInts * 4 && sizeof(PieceGroup) == kPieceGroupInts * 4, "piece layout");

// The order in which an item walks its KV tiles is free (online softmax), so every item
// starts at a different tile and wraps around: the row tiles of one (sequence, kv head)
// pair run on different SMs at the same time, and walking in step they would all ask the
// L2 for the same lines at the same moment.
constexpr int kPfTileRotation = 5;
#ifdef __CUDACC__
__device__ __forceinline__ int first_tile(const PrefillItem& item) {
  return item.n_tiles > 0 ? ((item.row0 / kPfRows) * kPfTileRotation) % item.n_tiles : 0;
}

__device__ __forceinline__ float fmax3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
#endif  // __CUDACC__

}  // namespace b200
