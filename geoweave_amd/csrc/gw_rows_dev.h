// Device pieces of the few-rows attention passes: sequences, scans over a wave and the join of parts, for 16-bit and
// 4-bit keys, and which part of which sequence's keys a workgroup takes, for 16-bit ones (4 bits: units, in their own pass).
#pragma once

#include "gw_packed.h"
#include "gw_rows.h"
#include "gw_rows_parts.h"

namespace gw {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
constexpr int kRows = 16;  // rows of a tile (token, head of the group); 4 bits: one or two tiles share a key read

__device__ __forceinline__ f32x4 mma16(BF16, uint4 a, uint4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma16(FP16, uint4 a, uint4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}

struct RowsSeq {
  int q0, lq, k0, lk;
};

template <bool PAGED>
__device__ __forceinline__ int rows_nseq(const RowsParams& p) { return PAGED ? p.n : p.n + 2; }

__device__ __forceinline__ int rows_bound(const int32_t* cu, int n, int T, int i) {
  if (i <= 0) return 0;
  if (i > n + 1) return T;
  return min(max(cu[i - 1], 0), T);
}

// Sequence i; packed: 0 and n + 1 are the tokens before the first and behind the last bound, without keys.
template <bool PAGED>
__device__ __forceinline__ RowsSeq rows_seq(const RowsParams& p, int i) {
  RowsSeq s;
  if constexpr (PAGED) {
    s.q0 = i;
    s.lq = p.Tq;
    s.k0 = 0;
    s.lk = (int)min((int64_t)max(p.lens[i], 0), (int64_t)p.table_width * p.page);
  } else {
    s.q0 = rows_bound(p.cu_q, p.n, p.Tq, i);
    s.lq = max(0, rows_bound(p.cu_q, p.n, p.Tq, i + 1) - s.q0);
    s.k0 = s.lk = 0;
    if (i >= 1 && i <= p.n) {
      s.k0 = rows_bound(p.cu_k, p.n, p.Tk, i);
      s.lk = max(0, rows_bound(p.cu_k, p.n, p.Tk, i + 1) - s.k0);
    }
  }
  return s;
}

// Inclusive sums over the lanes of a wave, by lane exchanges within the vector unit: within 16 lanes, then
// the last lane of each row on to the rows behind it.
template <int CTRL, int ROWS>
__device__ __forceinline__ int rows_dpp(int x) {
  return __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xF, false);
}
__device__ __forceinline__ int wave_scan(int x) {
  x += rows_dpp<0x111, 0xF>(x);  // row_shr 1, 2, 4, 8
  x += rows_dpp<0x112, 0xF>(x);
  x += rows_dpp<0x114, 0xF>(x);
  x += rows_dpp<0x118, 0xF>(x);
  x += rows_dpp<0x142, 0xA>(x);  // row_bcast 15 into rows 1 and 3
  x += rows_dpp<0x143, 0xC>(x);  // row_bcast 31 into rows 2 and 3
  return x;
}
__device__ __forceinline__ int lane_of(int x, int lane) { return __builtin_amdgcn_readlane(x, lane); }
// Sum over the wave of values below 2^62, 24 bits at a time (64 of those stay below 2^30).
__device__ __forceinline__ int64_t wave_sum64(int64_t x) {
  int64_t total = 0;
#pragma unroll
  for (int part = 0; part < 3; ++part) {
    const int piece = (int)((x >> (24 * part)) & 0xFFFFFF);
    total += (int64_t)lane_of(wave_scan(piece), 63) << (24 * part);
  }
  return total;
}

struct RowsPart {
  int seq, tile;    // seq < 0: nothing to do
  int part, parts;  // of this row tile
  int first;        // where the part 0 of a cut row tile is kept
  int len;          // keys of a part
};

// Row tiles of a sequence: packed, those of the longer ones are another kernel's.
template <bool PAGED>
__device__ __forceinline__ int rows_tiles_of(const RowsParams& p, const RowsSeq& s) {
  const int rows = s.lq * p.G;
  return PAGED || rows <= kRowsMax ? (rows + kRows - 1) / kRows : 0;
}

// Keys of a part: about p.want parts over all row tiles.
template <bool PAGED>
__device__ __forceinline__ int rows_part_len(const RowsParams& p, int lane) {
  const int nseq = rows_nseq<PAGED>(p);
  int64_t total = 0;
  for (int i = lane; i < nseq; i += 64) {
    const RowsSeq s = rows_seq<PAGED>(p, i);
    total += (int64_t)rows_tiles_of<PAGED>(p, s) * s.lk;
  }
  return rows_part_keys(wave_sum64(total), p.want);
}

// The part of slot `slot`.
template <bool PAGED>
__device__ __forceinline__ RowsPart rows_find(const RowsParams& p, int slot, int lane) {
  RowsPart r = {-1, 0, 0, 1, 0, 0x7fffff00};
  if (!p.split) {  // paged only: as many row tiles in each sequence
    const int rt = (p.Tq * p.G + kRows - 1) / kRows;
    r.seq = slot / rt;
    r.tile = slot - r.seq * rt;
    if (r.seq >= p.n) r.seq = -1;
    return r;
  }
  r.len = __builtin_amdgcn_readfirstlane(rows_part_len<PAGED>(p, lane));
  const int nseq = rows_nseq<PAGED>(p);
  int before = 0, cut_before = 0;
  for (int i0 = 0; i0 < nseq; i0 += 64) {
    const int i = i0 + lane;
    int tiles = 0, parts = 1;
    if (i < nseq) {
      const RowsSeq s = rows_seq<PAGED>(p, i);
      tiles = rows_tiles_of<PAGED>(p, s);
      parts = rows_parts(s.lk, r.len);
    }
    const int mine = tiles * parts, cut = parts > 1 ? mine : 0;
    const int incl = wave_scan(mine), cut_incl = wave_scan(cut);
    const uint64_t hit = __builtin_amdgcn_ballot_w64(before + incl > slot);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      const int at = slot - before - lane_of(incl - mine, l);
      r.parts = lane_of(parts, l);
      r.seq = i0 + l;
      r.tile = at / r.parts;
      r.part = at - r.tile * r.parts;
      r.first = cut_before + lane_of(cut_incl - cut, l) + r.tile * r.parts;
      break;
    }
    before += lane_of(incl, 63);
    cut_before += lane_of(cut_incl, 63);
  }
  return r;
}

// Largest over the four lanes (g = 0..3) of a row.
__device__ __forceinline__ float rows_max(float x) {
  x = fmaxf(x, __shfl_xor(x, 16));
  return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float rows_sum(float x) {
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

constexpr int kJoinParts = 1024;  // weights kept in LDS at a time

// Joins the parts of one row of a cut row tile of ROWS rows. D / 4 threads hold four dims each; the groups of them
// take the parts in turn, each part's row one 16-byte load per thread, and are summed in group order.
// UNITS: a row tile's first part is in slot cut.x (odd), the i-th behind it in slot cut.x + 2 i - 1.
template <typename E, int D, bool PAGED, int ROWS = kRows, bool UNITS = false>
__global__ __launch_bounds__(256) void rows_join_kernel(const RowsParams p) {
  constexpr int LPR = D / 4, GROUPS = 256 / LPR;
  __shared__ float w[kJoinParts];
  __shared__ float red[4];
  __shared__ float4 so[GROUPS][LPR];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int hk = blockIdx.x % p.Hk, row = blockIdx.y;
  const int at_tile = blockIdx.x / p.Hk;
  const int per = PAGED ? (p.Tq * p.G + ROWS - 1) / ROWS : 2;
  const int seq = at_tile / per, tile = at_tile - seq * per;
  const RowsSeq sq = rows_seq<PAGED>(p, seq);
  const int rr = tile * ROWS + row;
  if (rr >= sq.lq * p.G || (!PAGED && sq.lq * p.G > kRowsMax)) return;
  const int2 where = p.cut[at_tile];
  const int parts = where.y;
  // One part, or (packed bounds out of order, which may name more rows than there are) a tile that no
  // workgroup took and whose entry may hold anything.
  if (parts <= 1 || parts > 2 * p.want || (uint32_t)where.x > (uint32_t)(2 * p.want - parts)) return;
  auto slot = [](int i) { return UNITS ? 2 * i - (i > 0) : i; };
  const int64_t step = (int64_t)p.Hk * ROWS;
  const int64_t at = ((int64_t)where.x * p.Hk + hk) * ROWS + row;
  // The largest log2 sum (NaN if one is).
  float mx = -INFINITY;
  for (int i = tid; i < parts; i += 256) {
    const float x = p.part_lse[at + slot(i) * step];
    mx = x > mx || x != x ? x : mx;
    if (mx != mx) break;
  }
  auto top = [](float a, float b) { return a != a || a > b ? a : b; };
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) mx = top(mx, __shfl_xor(mx, d));
  if (lane == 0) red[wave] = mx;
  __syncthreads();
  mx = top(top(red[0], red[1]), top(red[2], red[3]));
  const int c = tid % LPR, grp = tid / LPR;
  float lt = 0.f;
  float4 out = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int p0 = 0; p0 < parts; p0 += kJoinParts) {
    const int np = min(kJoinParts, parts - p0);
    __syncthreads();
    for (int i = tid; i < np; i += 256) {
      const float x = p.part_lse[at + slot(p0 + i) * step];
      w[i] = x == -INFINITY ? 0.f : fexp2(x - mx);  // a part of which nothing is seen
    }
    __syncthreads();
#pragma unroll 4
    for (int i = grp; i < np; i += GROUPS) {
      const float f = w[i];
      const float4 x = reinterpret_cast<const float4*>(p.part + (at + slot(p0 + i) * step) * D)[c];
      lt += f;
      out.x = fmaf(x.x, f, out.x);
      out.y = fmaf(x.y, f, out.y);
      out.z = fmaf(x.z, f, out.z);
      out.w = fmaf(x.w, f, out.w);
    }
  }
  __shared__ float sl[GROUPS];
  so[grp][c] = out;
  if (c == 0) sl[grp] = lt;
  __syncthreads();
  if (grp != 0) return;
#pragma unroll
  for (int i = 1; i < GROUPS; ++i) {
    const float4 x = so[i][c];
    lt += sl[i];
    out.x += x.x;
    out.y += x.y;
    out.z += x.z;
    out.w += x.w;
  }
  const float inv = lt == 0.f ? 0.f : 1.f / lt;
  const int tk = rr / p.G, hd = hk * p.G + (rr - tk * p.G);
  const int64_t tg = PAGED ? (int64_t)seq * p.osb + (int64_t)tk * p.ost : (int64_t)(sq.q0 + tk) * p.ost;
  pk_store4<E>(p.o + tg + (int64_t)hd * p.osh + c * 4,
               !PAGED && p.rest ? p.rest + ((int64_t)(sq.q0 + tk) * p.H + hd) * D + c * 4 : nullptr, out.x * inv, out.y * inv,
               out.z * inv, out.w * inv);
  if (c == 0 && p.lse)
    p.lse[(int64_t)(PAGED ? seq * p.Tq + tk : sq.q0 + tk) * p.H + hd] =
        lt == 0.f ? -INFINITY : (mx + flog2(lt)) * kDLn2;
}

}  // namespace
}  // namespace gw
