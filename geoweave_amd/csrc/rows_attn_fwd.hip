// Attention of a few query rows per sequence over many keys (gfx950): one new token over a paged
// key-value cache, or packed sequences whose queries are few. D = 64 or 128.
//
//   o = sum_j 2^(s_j - m) v_j / sum_j 2^(s_j - m),  s = scale log2(e) q . k_j
// over disjoint parts of the keys, each with its own m; parts join by their log-sums:
//   o = sum_c 2^(L_c - L) o_c,  L = log2 sum_c 2^L_c.
//
// Bound by memory: each K and V row of a key head is read once, by one wave, for the up to 16 rows
// (token, head of the group) that share it. No LDS tile: a wave takes 32 keys at a time straight into
// the registers that the products read, the next 32 in flight meanwhile (16 KB per wave at D = 128).
// One token of 64 sequences of up to 32,976 keys, 32 heads over 8 of 128, pages of 16, bf16: 557 to 572 us, 5.0
// TB/s; five tokens of 8 sequences of up to 24,835 keys, 16 heads of 64: 95 us, 4.7 TB/s. Many new tokens read all
// keys once per 16 rows: 1,374 tokens x 16 heads of 64 over 20,000 keys 655 us.
//
// S^T = K Q^T (16x16x32): lane (g, i) reads 16 bytes of rows i and 16 + i and then holds
// the scores of keys 16 t + 4 g + r for row i. O^T += V^T P^T: the lane reads D / 16 dims of the 8
// rows that its scores stand for; exchanging 16-bit halves between those registers gives the
// operands of D / 16 products, in which dim (D / 16) i + u is operand row i of product u.
//
// Work is cut by keys, not by sequences: with the lengths on the device only, each workgroup sums
// (row tiles x keys) over the sequences, takes a part length that gives about `want` parts in all, and
// finds its own part by a second scan (64 sequences at a time). Where the row tiles alone
// fill the chip there is no split and no scan. A second launch joins the parts of rows that were cut.
//
// Table entries outside the pool are keys that nobody sees. Rows that are not keys (behind the length, or
// in such a page) are masked, and their V registers are cleared: what lies there cannot reach a result.
#include <math.h>

#include "gw_packed.h"
#include "gw_rows.h"
#include "gw_rows_parts.h"

namespace gw {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
constexpr int kRows = 16;

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

template <int DV>
struct RowsV;
template <>
struct RowsV<4> {
  uint32_t w[2];
  __device__ __forceinline__ void load(const uint16_t* p) {
    const uint2 x = *reinterpret_cast<const uint2*>(p);
    w[0] = x.x;
    w[1] = x.y;
  }
};
template <>
struct RowsV<8> {
  uint32_t w[4];
  __device__ __forceinline__ void load(const uint16_t* p) {
    const uint4 x = *reinterpret_cast<const uint4*>(p);
    w[0] = x.x;
    w[1] = x.y;
    w[2] = x.z;
    w[3] = x.w;
  }
};

template <typename E, int D, bool PAGED>
__global__ __launch_bounds__(256, 2) void rows_attn_kernel(const RowsParams p) {
  constexpr int KS = D / 32, DV = D / 16;
  __shared__ float so[4][kRows][D + 4];
  __shared__ float sm[4][kRows], sl[4][kRows];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, i16 = lane & 15;
  const int hk = blockIdx.x % p.Hk, slot = blockIdx.x / p.Hk;
  const RowsPart pt = rows_find<PAGED>(p, slot, lane);
  if (pt.seq < 0) return;
  if (p.split && pt.part == 0 && hk == 0 && threadIdx.x == 0)  // for the join
    p.cut[PAGED ? pt.seq * ((p.Tq * p.G + kRows - 1) / kRows) + pt.tile : 2 * pt.seq + pt.tile] = make_int2(pt.first, pt.parts);
  const RowsSeq sq = rows_seq<PAGED>(p, pt.seq);
  const int lk = __builtin_amdgcn_readfirstlane(sq.lk), k0 = __builtin_amdgcn_readfirstlane(sq.k0);
  const int rows = sq.lq * p.G;

  const int r = min(pt.tile * kRows + i16, rows - 1);
  const int tok = r / p.G, head = hk * p.G + (r - tok * p.G);
  const int64_t qb = PAGED ? (int64_t)pt.seq * p.qsb + (int64_t)tok * p.qst : (int64_t)(sq.q0 + tok) * p.qst;
  uint4 qf[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s)
    qf[s] = *reinterpret_cast<const uint4*>(p.q + qb + (int64_t)head * p.qsh + 32 * s + 8 * g);
  const int lim = p.causal ? min(tok + lk - sq.lq, lk - 1) : lk - 1;
  // Rows are token-major: the tile's first row sees the fewest keys.
  const int lim_lo = __builtin_amdgcn_readfirstlane(lim);

  const int kb = (int)min((int64_t)pt.part * pt.len, (int64_t)lk);
  const int ke = (int)min((int64_t)kb + pt.len, (int64_t)lk);

  f32x4 acc[DV];
#pragma unroll
  for (int u = 0; u < DV; ++u) acc[u] = (f32x4){0.f, 0.f, 0.f, 0.f};
  float m = -3.4028234663852886e38f, l = 0.f;

  const uint16_t* kbase = p.k + (int64_t)hk * p.ksh;
  const uint16_t* vbase = p.v + (int64_t)hk * p.vsh;
  const int32_t* trow = PAGED ? p.table + (int64_t)pt.seq * p.table_stride : nullptr;

  // One block of 32 keys: where its rows lie, one per lane (lanes l and l + 32 alike).
  struct Where {
    int page, at;
    uint32_t ok;  // bit j: key j of the block is one
  };
  auto where = [&](int j0) __attribute__((always_inline)) {
    Where w;
    const int key = min(j0 + (lane & 31), lk - 1);  // lk > 0 here
    bool ok = j0 + (lane & 31) < ke;
    if constexpr (PAGED) {
      const int pg = key / p.page;
      w.at = key - pg * p.page;
      const int id = trow[pg];
      const bool in = (uint32_t)id < (uint32_t)p.pages;
      w.page = in ? id : 0;
      ok = ok && in;
    } else {
      w.page = 0;
      w.at = k0 + key;
    }
    w.ok = (uint32_t)__builtin_amdgcn_ballot_w64(ok);
    return w;
  };
  struct Block {
    uint4 k[2][KS];
    RowsV<DV> v[8];
  };
  auto fetch = [&](const Where& w, Block& b) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int src = 16 * t + i16;
      const int64_t page = PAGED ? __shfl(w.page, src) : 0, at = __shfl(w.at, src);
      const uint16_t* row = kbase + (PAGED ? page * p.ksp : 0) + at * p.kst + 8 * g;
#pragma unroll
      for (int s = 0; s < KS; ++s) b.k[t][s] = *reinterpret_cast<const uint4*>(row + 32 * s);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int src = 16 * (j / 4) + 4 * g + j % 4;
      const int64_t page = PAGED ? __shfl(w.page, src) : 0, at = __shfl(w.at, src);
      b.v[j].load(vbase + (PAGED ? page * p.vsp : 0) + at * p.vst + DV * i16);
    }
  };
  bool unclean = false;
  auto compute = [&](int j0, uint32_t ok, Block& b) __attribute__((always_inline)) {
    f32x4 s[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      s[t] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) s[t] = mma16(E{}, b.k[t][ks], qf[ks], s[t]);
    }
    if (ok != 0xFFFFFFFFu || j0 + 31 > lim_lo) {
      const uint32_t mine = ok >> (4 * g);
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (!((mine >> (16 * t + u)) & 1u) || j0 + 16 * t + 4 * g + u > lim) s[t][u] = -INFINITY;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (!((mine >> (16 * (j / 4) + j % 4)) & 1u)) {
#pragma unroll
          for (int u = 0; u < DV / 2; ++u) b.v[j].w[u] = 0u;
        }
      if (j0 + 31 > lim_lo) {  // some rows see some of these keys only: see pk_clear_not_finite
        uint32_t any = 0u;
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int u = 0; u < DV / 2; ++u) any |= pk_not_finite_bits<E>(b.v[j].w[u]);
        if (__builtin_amdgcn_ballot_w64((any & 0x80008000u) != 0u) != 0ull) {
          unclean = true;
#pragma unroll
          for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int u = 0; u < DV / 2; ++u) b.v[j].w[u] = pk_finite_word<E>(b.v[j].w[u]);
        }
      }
    }
    float w[8];
    auto weights = [&](float nm) __attribute__((always_inline)) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int u = 0; u < 4; ++u) w[4 * t + u] = fexp2(fmaf(s[t][u], p.scale_log2, nm));
      return ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
    };
    float ls = weights(-m);
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(!(ls <= kPkSumCap<E>)) != 0ull, 0)) {
      const bool up = rows_max(ls <= kPkSumCap<E> ? 0.f : 1.f) > 0.f;  // this row, not the tile's others
      float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                       fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
      mx = rows_max(mx);
      const float mn = up ? fmaxf(m, mx * p.scale_log2 - kPkBelow<E>) : m;
      const float alpha = fexp2(m - mn);
      m = mn;
      l *= alpha;
#pragma unroll
      for (int u = 0; u < DV; ++u) acc[u] *= alpha;
      ls = weights(-mn);
    }
    l += ls;
    const uint4 pb = pack_quad<E>(w);
#pragma unroll
    for (int u = 0; u < DV; ++u) {
      uint32_t a[4];
#pragma unroll
      for (int h = 0; h < 4; ++h)
        a[h] = __builtin_amdgcn_perm(b.v[2 * h + 1].w[u / 2], b.v[2 * h].w[u / 2], (u & 1) ? 0x07060302u : 0x05040100u);
      acc[u] = mma16(E{}, make_uint4(a[0], a[1], a[2], a[3]), pb, acc[u]);
    }
  };

  const int j_first = kb + 32 * wave;
  if (j_first < ke) {
    Block b0, b1;
    Where w0 = where(j_first), w1 = where(j_first + 128);
    fetch(w0, b0);
    // Blocks of this wave every 128 keys; rows of a block are found two blocks ahead.
    int j = j_first;
#pragma unroll 1
    while (true) {
      const Where w2 = where(j + 256);
      fetch(w1, b1);
      compute(j, w0.ok, b0);
      if (j + 128 >= ke) break;
      w0 = where(j + 384);
      fetch(w2, b0);
      compute(j + 128, w1.ok, b1);
      if (j + 256 >= ke) break;
      // the next round: block j + 256 (in b0, rows w2), block j + 384 (rows w0)
      w1 = w0;
      w0 = w2;
      j += 256;
    }
  }

  if (__builtin_expect(unclean, 0)) {
    // This wave's blocks behind the first row's last key: their V entries that are not finite go to the rows
    // that see them.
    for (int j0 = j_first; j0 < ke; j0 += 128) {
      if (j0 + 31 <= lim_lo) continue;
      const Where w = where(j0);
      for (int i = 0; i < 32; ++i) {
        if (!((w.ok >> i) & 1u)) continue;
        const int64_t page = __shfl(w.page, i), at = __shfl(w.at, i);
        const uint16_t* row = vbase + (PAGED ? page * p.vsp : 0) + at * p.vst + 4 * DV * g;
        for (int x = 0; x < 4 * DV; ++x) {
          const uint32_t h = row[x];
          if (!pk_not_finite<E>(h) || j0 + i > lim) continue;
          const float f = in_to_float(__is_same(E, FP16), h);
#pragma unroll
          for (int u = 0; u < DV; ++u)
#pragma unroll
            for (int rr = 0; rr < 4; ++rr)
              if (rr * DV + u == x) acc[u][rr] += f;
        }
      }
    }
  }

  // The four waves' parts, joined in wave order.
  const float lw = rows_sum(l);
  if (g == 0) {
    sm[wave][i16] = m;
    sl[wave][i16] = lw;
  }
#pragma unroll
  for (int rr = 0; rr < 4; ++rr)
#pragma unroll
    for (int u = 0; u < DV; ++u) so[wave][i16][(4 * g + rr) * DV + u] = acc[u][rr];
  __syncthreads();
  const int row = threadIdx.x >> 4, c = threadIdx.x & 15;  // 16 threads per row, DV dims each
  const int rr = pt.tile * kRows + row;
  if (rr >= rows) return;
  float mx = sm[0][row];
#pragma unroll
  for (int w = 1; w < 4; ++w) mx = fmaxf(mx, sm[w][row]);
  float lt = 0.f, out[DV];
#pragma unroll
  for (int u = 0; u < DV; ++u) out[u] = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float f = fexp2(sm[w][row] - mx);
    lt = fmaf(sl[w][row], f, lt);
#pragma unroll
    for (int u = 0; u < DV; ++u) out[u] = fmaf(so[w][row][c * DV + u], f, out[u]);
  }
  const float inv = lt == 0.f ? 0.f : 1.f / lt;
#pragma unroll
  for (int u = 0; u < DV; ++u) out[u] = lt == 0.f ? 0.f : out[u] * inv;
  const float l2 = lt == 0.f ? -INFINITY : mx + flog2(lt);
  if (pt.parts > 1) {
    const int64_t at = ((int64_t)(pt.first + pt.part) * p.Hk + hk) * kRows + row;
    float* dst = p.part + at * D + c * DV;
#pragma unroll
    for (int u = 0; u < DV; u += 4) *reinterpret_cast<float4*>(dst + u) = make_float4(out[u], out[u + 1], out[u + 2], out[u + 3]);
    if (c == 0) p.part_lse[at] = l2;
    return;
  }
  const int tk = rr / p.G, hd = hk * p.G + (rr - tk * p.G);
  const int64_t tg = PAGED ? (int64_t)pt.seq * p.osb + (int64_t)tk * p.ost : (int64_t)(sq.q0 + tk) * p.ost;
  uint16_t* dst = p.o + tg + (int64_t)hd * p.osh + c * DV;
  uint16_t* rest = !PAGED && p.rest ? p.rest + ((int64_t)(sq.q0 + tk) * p.H + hd) * D + c * DV : nullptr;
#pragma unroll
  for (int u = 0; u < DV; u += 4)
    pk_store4<E>(dst + u, rest ? rest + u : nullptr, out[u], out[u + 1], out[u + 2], out[u + 3]);
  if (c == 0 && p.lse) p.lse[(int64_t)(PAGED ? pt.seq * p.Tq + tk : sq.q0 + tk) * p.H + hd] = l2 * kDLn2;
}

// Joins the parts of one row of a cut row tile. D / 4 threads hold four dims each; the groups of them
// take the parts in turn, each part's row one 16-byte load per thread, and are summed in group order.
constexpr int kJoinParts = 1024;  // weights kept in LDS at a time

template <typename E, int D, bool PAGED>
__global__ __launch_bounds__(256) void rows_join_kernel(const RowsParams p) {
  constexpr int LPR = D / 4, GROUPS = 256 / LPR;
  __shared__ float w[kJoinParts];
  __shared__ float red[4];
  __shared__ float4 so[GROUPS][LPR];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int hk = blockIdx.x % p.Hk, row = blockIdx.y;
  const int at_tile = blockIdx.x / p.Hk;
  const int per = PAGED ? (p.Tq * p.G + kRows - 1) / kRows : 2;
  const int seq = at_tile / per, tile = at_tile - seq * per;
  const RowsSeq sq = rows_seq<PAGED>(p, seq);
  const int rr = tile * kRows + row;
  if (rr >= sq.lq * p.G || (!PAGED && sq.lq * p.G > kRowsMax)) return;
  const int2 where = p.cut[at_tile];
  const int parts = where.y;
  // One part, or (packed bounds out of order, which may name more rows than there are) a tile that no
  // workgroup took and whose entry may hold anything.
  if (parts <= 1 || parts > 2 * p.want || (uint32_t)where.x > (uint32_t)(2 * p.want - parts)) return;
  const int64_t step = (int64_t)p.Hk * kRows;
  const int64_t at = ((int64_t)where.x * p.Hk + hk) * kRows + row;
  // The largest log2 sum (NaN if one is).
  float mx = -INFINITY;
  for (int i = tid; i < parts; i += 256) {
    const float x = p.part_lse[at + i * step];
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
      const float x = p.part_lse[at + (p0 + i) * step];
      w[i] = x == -INFINITY ? 0.f : fexp2(x - mx);  // a part of which nothing is seen
    }
    __syncthreads();
#pragma unroll 4
    for (int i = grp; i < np; i += GROUPS) {
      const float f = w[i];
      const float4 x = reinterpret_cast<const float4*>(p.part + (at + (p0 + i) * step) * D)[c];
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

template <typename E, int D, bool PAGED>
int rows_launch(const RowsParams& p, hipStream_t stream) {
  const int64_t joins = rows_tiles(PAGED, p.n, p.Tq, p.G) * p.Hk, grid = rows_grid(PAGED, p.n, p.Tq, p.G, p.Hk, p.split);
  GW_CHECK_GRID(grid, 256);
  if (p.split) GW_CHECK_GRID(joins, 256);
  hipLaunchKernelGGL((rows_attn_kernel<E, D, PAGED>), dim3((uint32_t)grid), dim3(256), 0, stream, p);
  GW_HIP_LAUNCH_CHECK("rows attention");
  if (p.split) {
    const int64_t rows = (int64_t)p.Tq * p.G;
    hipLaunchKernelGGL((rows_join_kernel<E, D, PAGED>), dim3((uint32_t)joins, (uint32_t)(rows < kRows ? rows : kRows)),
                       dim3(256), 0, stream, p);
    GW_HIP_LAUNCH_CHECK("rows attention (join)");
  }
  return GW_OK;
}

template <typename E>
int rows_dim(int D, bool paged, const RowsParams& p, hipStream_t s) {
  if (D == 64) return paged ? rows_launch<E, 64, true>(p, s) : rows_launch<E, 64, false>(p, s);
  return paged ? rows_launch<E, 128, true>(p, s) : rows_launch<E, 128, false>(p, s);
}

}  // namespace

int rows_attn(int dtype, int D, bool paged, RowsParams p, void* workspace, hipStream_t stream) {
  if (p.split) {
    p.part = static_cast<float*>(workspace);
    p.part_lse = p.part + (int64_t)2 * p.want * p.Hk * kRows * D;
    p.cut = reinterpret_cast<int2*>(p.part_lse + (int64_t)2 * p.want * p.Hk * kRows);
  }
  return dtype == GW_DTYPE_BF16 ? rows_dim<BF16>(D, paged, p, stream) : rows_dim<FP16>(D, paged, p, stream);
}

}  // namespace gw

// Row tiles that reach sixteen workgroups per CU are not split: every workgroup of a split call scans the lengths, and
// even batches lose by it (32 heads over 8 of 64, pages of 16, 512 sequences of 1,000 keys 224 us, 232 split; of 200
// keys 44 and 74; 5,000 of 20 keys, one head, 32 and 221). One sequence of 60,000 keys among 511 of 1,000 is the
// price: 702 us, 274 split.
static bool paged_split(int64_t B, int64_t N, int64_t Hq, int64_t Hk) {
  return B * ((N * (Hq / Hk) + gw::kRows - 1) / gw::kRows) * Hk < 4096;
}

extern "C" size_t gw_paged_attn_fwd_workspace_size(int64_t B, int64_t N, int64_t Hq, int64_t Hk, int64_t D) {
  using namespace gw;
  if (B < 1 || N < 1 || Hk < 1 || Hq < Hk || D < 1 || !paged_split(B, N, Hq, Hk)) return 0;
  return rows_workspace(rows_tiles(true, B, N, Hq / Hk), Hk, D);
}

extern "C" int gw_paged_attn_fwd(int dtype, const void* q, const int64_t* q_strides, const void* k,
                                 const int64_t* k_strides, const void* v, const int64_t* v_strides,
                                 const int32_t* block_table, int64_t table_stride, const int32_t* lens, void* o,
                                 const int64_t* o_strides, float* lse, int64_t B, int64_t N, int64_t Hq, int64_t Hk,
                                 int64_t D, int64_t pages, int64_t page_size, int64_t table_width, int causal,
                                 float softmax_scale, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace gw;
  clear_error();
  GW_CHECK_ARG(dtype == GW_DTYPE_BF16 || dtype == GW_DTYPE_FP16, "unknown dtype %d", dtype);
  if (D != 64 && D != 128) return set_error(GW_ERR_UNSUPPORTED, "head dim %lld is not 64 or 128", (long long)D);
  GW_CHECK_ARG(B >= 0 && N >= 0 && pages >= 0 && table_width >= 0, "negative size");
  GW_CHECK_ARG(page_size >= 1 && page_size < (1ll << 31) && pages < (1ll << 31), "page size %lld, pages %lld",
               (long long)page_size, (long long)pages);
  GW_CHECK_ARG(Hk >= 1 && Hq >= Hk && Hq % Hk == 0, "%lld query heads are no multiple of %lld key heads", (long long)Hq,
               (long long)Hk);
  GW_CHECK_ARG(softmax_scale > 0.f && softmax_scale <= 3.0e38f, "the softmax scale must be positive and finite");
  if (B == 0 || N == 0) return GW_OK;
  if (table_width > 0x7FFFF000ll / page_size || B > 0x7FFFFFFFll / Hq / N)
    return set_error(GW_ERR_UNSUPPORTED, "keys of a sequence and new tokens x heads must stay below 2^31");
  GW_CHECK_ARG(q && o && lens && q_strides && k_strides && v_strides && o_strides, "a tensor is missing");
  GW_CHECK_ARG((k && v) || pages == 0, "the cache is missing");
  GW_CHECK_ARG(block_table || table_width == 0, "the block table is missing");
  auto ok = [](const void* x, const int64_t* s) {
    return aligned16(x) && s[0] % 8 == 0 && s[1] % 8 == 0 && s[2] % 8 == 0;
  };
  GW_CHECK_ARG(ok(q, q_strides) && ok(k, k_strides) && ok(v, v_strides) && ok(o, o_strides),
               "q, k, v and o need 16-byte aligned rows");
  RowsParams p = {};
  p.q = static_cast<const uint16_t*>(q);
  p.k = static_cast<const uint16_t*>(k);
  p.v = static_cast<const uint16_t*>(v);
  p.o = static_cast<uint16_t*>(o);
  p.lse = lse;
  p.table = block_table;
  p.lens = lens;
  p.table_stride = table_stride;
  p.table_width = pages == 0 ? 0 : (int)table_width;  // an empty pool holds no keys
  p.pages = (int)pages;
  p.page = (int)page_size;
  p.n = (int)B;
  p.Tq = (int)N;
  p.H = (int)Hq;
  p.Hk = (int)Hk;
  p.G = (int)(Hq / Hk);
  p.causal = causal != 0;
  p.qsb = q_strides[0];
  p.qst = q_strides[1];
  p.qsh = q_strides[2];
  p.osb = o_strides[0];
  p.ost = o_strides[1];
  p.osh = o_strides[2];
  p.ksp = k_strides[0];
  p.kst = k_strides[1];
  p.ksh = k_strides[2];
  p.vsp = v_strides[0];
  p.vst = v_strides[1];
  p.vsh = v_strides[2];
  p.scale_log2 = softmax_scale * kDLog2e;
  p.split = paged_split(B, N, Hq, Hk);
  p.want = rows_want(Hk);
  const size_t need = gw_paged_attn_fwd_workspace_size(B, N, Hq, Hk, D);
  GW_CHECK_ARG(need == 0 || (workspace && aligned16(workspace) && workspace_bytes >= need),
               "workspace of %zu bytes, %zu are needed", workspace_bytes, need);
  return rows_attn(dtype, (int)D, true, p, workspace, static_cast<hipStream_t>(stream));
}
