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
  float* lse;           // nullable
  float* part;          // parts: [slot][Hk][16][D] normalised outputs, then [slot][Hk][16] log2 sums
  float* part_lse;
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
  int split;            // 0: one workgroup takes all keys of its rows
  int want;             // workgroups per key head to aim at (split)
  int64_t qsb, qst, qsh, osb, ost, osh;   // packed: qsb = osb = 0
  int64_t ksp, kst, ksh, vsp, vst, vsh;   // per page (packed: 0), token, head
  float scale_log2;
};

// Row tiles (16 rows of a key head) of all sequences at most.
int64_t rows_tiles(bool paged, int64_t n, int64_t Tq, int64_t G);
// Slots per key head at most, and the workspace that the parts take.
int64_t rows_slots(const RowsParams& p, bool paged);
size_t rows_workspace(int64_t slots, int64_t Hk, int64_t D);
// Launches on checked arguments (dtype bf16 or fp16, D 64 or 128).
int rows_attn(int dtype, int D, bool paged, RowsParams p, void* workspace, hipStream_t stream);

}  // namespace gw
