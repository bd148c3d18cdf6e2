// Internal interface of the few-rows attention (rows_attn_fwd.hip): a few query rows per sequence over
// many keys, the keys split over workgroups and the parts joined.
#pragma once

#include "gw_common.h"

namespace gw {

struct RowsParams {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* o;
  uint16_t* rest;       // nullable (packed): [Tq][H][D], what the rounding of o left
  float* lse;           // nullable
  float* part;          // parts of cut row tiles: [slot][Hk][rows of a tile][D] normalised outputs,
  float* part_lse;      // [slot][Hk][rows of a tile] log2 sums
  int2* cut;            // [tile] of a split call: where a row tile's parts are kept, and how many (paged: tile
                        // sequence * tiles of one + tile; packed: 2 sequence + tile)
  // Paged: table [B][table_width] page numbers (row stride table_stride), lens [B].
  const int32_t* table;
  const int32_t* lens;
  int64_t table_stride;
  int table_width, pages, page;
  // Packed: as in gw_packed_attn_fwd.
  const int32_t* cu_q;
  const int32_t* cu_k;
  int n;                // sequences (paged: B)
  int Tq, Tk;           // packed: tokens; paged: Tq = new tokens of a sequence
  int H, Hk, G, causal;
  int split;            // 0: one workgroup takes all keys of its rows (paged only)
  int want;             // parts per key head to aim at (split)
  int64_t qsb, qst, qsh, osb, ost, osh;   // packed: qsb = osb = 0
  int64_t ksp, kst, ksh, vsp, vst, vsh;   // per page (packed: 0), token, head
  float scale_log2;
};

// Packed: sequences of at most this many rows (tokens x heads of a group) are this kernel's.
constexpr int kRowsMax = 32;

// Parts per key head to aim at: about four workgroups per CU over all heads.
inline int rows_want(int64_t Hk) { return (int)(1024 / Hk > 0 ? 1024 / Hk : 1); }
// Row tiles of a call at most: the join's workgroups, and the entries of `cut`.
inline int64_t rows_tiles(bool paged, int64_t n, int64_t Tq, int64_t G, int64_t rows = 16) {
  return paged ? n * ((Tq * G + rows - 1) / rows) : 2 * (n + 2);
}
// Workspace of a split call. A tile is cut where its keys exceed the part length, so it has fewer than
// two parts per part length of keys, and all cut tiles fewer than 2 want.
inline size_t rows_workspace(int64_t tiles, int64_t Hk, int64_t D) {
  return (size_t)2 * rows_want(Hk) * Hk * 16 * (D + 1) * sizeof(float) + (size_t)tiles * sizeof(int2);
}
// Workgroups of the attention launch. Packed: a sequence of at most kRowsMax rows has one or two tiles, and all have
// no more than the rows in all allow.
inline int64_t rows_grid(bool paged, int64_t n, int64_t Tq, int64_t G, int64_t Hk, bool split) {
  int64_t tiles = rows_tiles(paged, n, Tq, G);
  if (!paged && Tq * G / 16 + n + 2 < tiles) tiles = Tq * G / 16 + n + 2;
  return (tiles + (split ? rows_want(Hk) : 0)) * Hk;
}
// Launches on checked arguments (dtype bf16 or fp16, D 64 or 128); p.split and p.want are set.
int rows_attn(int dtype, int D, bool paged, RowsParams p, void* workspace, hipStream_t stream);

}  // namespace gw
