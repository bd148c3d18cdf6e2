// Attention of a few new tokens per sequence over a paged cache in 4 bits (gfx950). D = 64 or 128.
//
// Formulas, parts and joins are those of rows_attn_fwd.hip; the cache's format is in gw_fp4.h. What a key
// costs is its 17/16 D bytes (K and V), a quarter of a 16-bit cache's, so here the instructions per key count:
//
// Codes become 16-bit values by the conversion instruction, two of a row at a time with their power of two: exact, so that
// the products are those of the values themselves.
//   S^T = K Q^T (16x16x32): lane (g, i) reads the D / 4 dims from D / 4 g on of key i, which are its operands of the
// D / 32 products one after the other, and holds q of row i in the same order. In fp16, the scores of a key with a unit
// outside the normal numbers (2^-13 to 2^13) are those of K in bf16 and q in two bf16 terms, exact.
// The block-scaled product (16x16x128, fp4 x fp8, q in e4m3 terms) would take K without a conversion, but sums
// 2^-17 of the magnitudes off (measured; 3e-4 in a score of 13 whose magnitudes are 32), and is not faster here.
//   O^T += V^T P^T (16x16x32): the scores of a lane stand for eight keys; exchanging halves between those keys'
// registers gives the operand of each product. P is the sum of two bf16 terms (16 bits; one term has 2^-9, which is a
// 16-bit output's own rounding again, and fp16 would bound V's range).
//
// Work is cut into units of equal cost (64-key blocks, and four more for a row tile's start and end), one for each workgroup that
// the chip holds at once, over all row tiles, one behind the other: a unit may end one tile, take others whole and begin
// another, so that all workgroups end together whatever the lengths, and each finds its place once. Parts of one length, as in
// rows_attn_fwd.hip, left the last round of workgroups partly empty: 32 streams to 109,920 keys, 16 heads of 64: 524 us, by
// units 486 (and 430 with RUNS). A tile that lies in several units is joined by a second launch. Where the row tiles alone fill the
// chip many times there is no split and no scan.
//
// A wave takes 64 keys at a time, the next 64 keys' rows in flight meanwhile, and the page numbers of the 64 behind.
// Pages of a multiple of 16 slots whose scales lie slot behind slot, 16-byte aligned (RUNS; fp4_paged_cache is like that): 16 keys
// from a multiple of 16 on lie in one page, so their addresses are a scalar offset and fixed ones of the lanes, and a lane
// reads the scales of its keys itself. Else a lane finds the page, slot and scales of one key and hands them to the
// lanes that need them (the 32 streams in pages of 100: 469 to 495 us).
//
// Bound by memory where rows are few: those 32 streams 414 us of the kernel alone, 5.2 TB/s; one token of 64 sequences to
// 32,976 keys, 32 heads over 8 of 128, pages of 16: 113 to 117 us, 5.0 TB/s. With 64 rows over a key (8 tokens x 8 heads) no
// unit is full (vector unit 49 % busy, matrix cores 26 %; two waves per SIMD wait for data and for each other; a key is
// converted twice): 73 us for 31 GFLOP; four row tiles to a wave (one wave per SIMD) took 87 for 82.
//
// Rows that are not keys (behind the length, in a page outside the pool) are masked, and their scales count as 2^-127:
// what lies there cannot reach a result. A masked weight is 0, but 0 * inf is NaN, so values of V that are no finite number (gw_fp4.h:
// NaN under a scale of 255, inf from 2^128 on, under 253 and 254) count as 0 in the products and are added afterwards to the
// rows that see them.
#include <math.h>
#include <string.h>

#include <type_traits>

#include "gw_fp4.h"
#include "gw_rows_dev.h"

namespace gw {
namespace {

// Workgroups that a CU holds.
constexpr int fp4_resident(int D, int RT) { return D == 64 && RT == 1 ? 3 : 2; }

struct Fp4AttnParams : RowsParams {  // want: units per key head
  const uint8_t* kc;
  const uint8_t* vc;
  const uint8_t* ksc;
  const uint8_t* vsc;
  int64_t kssp, ksst, kssh, vssp, vsst, vssh;  // scales: per page, slot, head (bytes)
  uint32_t kup, kut, vup, vut;                 // codes: per page and slot, in units of 16 bytes
  uint32_t page_inverse;                       // floor(2^32 / page), 2^32 - 1 for pages of one slot
  int64_t khead, vhead;                        // codes: per head (bytes)
};

// An fp16 operand of q as two bf16 ones: the rounded values, and what that leaves (at most three bits: exact).
__device__ __forceinline__ void fp4_split_query(uint4 q, uint4& high, uint4& low) {
  float f[8], rest[8];
  unpack8<FP16>(q, f);
  high = pack_quad<BF16>(f);
  unpack8<BF16>(high, rest);
#pragma unroll
  for (int j = 0; j < 8; ++j) rest[j] = rest[j] == f[j] ? 0.f : f[j] - rest[j];  // inf leaves nothing
  low = pack_quad<BF16>(rest);
}
// Whether the values of a unit 2^e (its float) are normal fp16 numbers, e from -13 to 13.
__device__ __forceinline__ bool fp4_fits_fp16(float unit) { return (__float_as_uint(unit) >> 23) - 114u <= 26u; }

// Keys of sequence i, and 64-key blocks of as many keys (one, of nothing, for none: its rows are written too).
__device__ __forceinline__ int fp4_length(const RowsParams& p, int i) {
  return (int)min((int64_t)max(p.lens[i], 0), (int64_t)p.table_width * p.page);
}
__device__ __forceinline__ int fp4_blocks(int lk) { return lk > 64 ? (int)(((int64_t)lk + 63) >> 6) : 1; }

// What a row tile costs beside its blocks, in blocks: its first rows' way from the lengths over the table, and its end.
constexpr int kTileCost = 4;

struct Fp4Place {
  int seq, lk;
  int64_t before;  // cost of the sequences before it
};
// The sequence that holds place `at` of all sequences' costs in a row (TOTAL: their sum, as `before`), by one wave, 64
// sequences at a time (a sequence has fewer than 2^25 - 63 blocks, so the costs of 64 stay below 2^31). first: the keys of
// sequence `lane`.
template <bool TOTAL>
__device__ __forceinline__ Fp4Place fp4_blocks_before(const RowsParams& p, int first, int64_t at, int lane) {
  Fp4Place r = {0, 0, 0};
  for (int i0 = 0; i0 < p.n; i0 += 64) {
    int lk = first;
    if (i0 > 0 && i0 + lane < p.n) lk = fp4_length(p, i0 + lane);
    const int mine = i0 + lane < p.n ? fp4_blocks(lk) + kTileCost : 0;
    const int incl = wave_scan(mine);
    if constexpr (!TOTAL) {
      const uint64_t hit = __builtin_amdgcn_ballot_w64(r.before + incl > at);
      if (hit) {
        const int l = __builtin_ctzll(hit);
        r.seq = i0 + l;
        r.lk = lane_of(lk, l);
        r.before += lane_of(incl - mine, l);
        return r;
      }
    }
    r.before += lane_of(incl, 63);
  }
  return r;
}

// x / y of positive values, by 32 bits where they fit (a quarter of the instructions).
__device__ __forceinline__ int64_t fp4_div(int64_t x, int64_t y) {
  if (((x | y) >> 32) == 0) return (uint32_t)x / (uint32_t)y;
  return x / y;
}

template <typename E, int D, int RT, bool RUNS>
__global__ __launch_bounds__(256, fp4_resident(D, RT)) void fp4_attn_kernel(const Fp4AttnParams p) {
  constexpr int DV = D / 16, ROWS = kRows * RT;
  typedef typename std::conditional<D == 128, uint4, uint2>::type KWord;  // what a lane reads of a key of K
  constexpr int VW = D == 128 ? 16 : 8;  // words of V that a lane reads of 64 keys
  __shared__ float so[4][kRows][D + 4];
  __shared__ float sm[4][kRows], sl[4][kRows];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, i16 = lane & 15;
  const int hk = blockIdx.x % p.Hk, unit = blockIdx.x / p.Hk;
  const int T = (p.Tq * p.G + ROWS - 1) / ROWS;  // row tiles of a sequence

  // Where the unit begins: row tile `tile` of sequence `seq`, place `skip` of its blocks (negative: before them); the cost that the
  // unit still has; where the tile's blocks begin among all costs.
  int tile, seq, lk;
  int64_t skip = 0, left = 1, begin = 0, L = 1;
  if (!p.split) {
    seq = unit / T;
    tile = unit - seq * T;
    lk = fp4_length(p, seq);
  } else {
    const int first = fp4_length(p, min(lane, p.n - 1));
    const int64_t S = fp4_blocks_before<true>(p, first, 0, lane).before;
    L = fp4_div(T * S + p.want - 1, p.want);
    L = ((L > 4 ? L : 4) + 3) / 4 * 4;  // as many blocks for every wave
    const int64_t from = unit * L;
    if (from >= T * S) return;
    left = min(L, T * S - from);
    tile = (int)fp4_div(from, S);
    const Fp4Place at = fp4_blocks_before<false>(p, first, from - tile * S, lane);
    seq = at.seq;
    lk = at.lk;
    begin = tile * S + at.before + kTileCost;
    skip = from - begin;
  }

  for (;; begin += kTileCost, skip = -kTileCost) {
    if (p.split && skip < 0) {
      left += skip;
      skip = 0;
      if (left <= 0) return;  // the next unit's
    }
    lk = __builtin_amdgcn_readfirstlane(lk);
    const int lq = p.Tq;
    const int64_t blocks = fp4_blocks(lk);
    const int rows = lq * p.G;
    // Units that the tile lies in, and this one's place among them.
    const int first_unit = (int)fp4_div(begin, L), parts = p.split ? (int)fp4_div(begin + blocks - 1, L) - first_unit + 1 : 1;
    const int part = unit - first_unit;
    if (p.split && part == 0 && hk == 0 && threadIdx.x == 0) p.cut[seq * T + tile] = make_int2(2 * first_unit + 1, parts);
    const int64_t take = p.split ? min(blocks - skip, left) : blocks;

    uint4 q[RT][D / 32];  // a lane's dims of row i16
    int lim[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const int r = min(tile * ROWS + t * kRows + i16, rows - 1);
      const int tok = r / p.G, head = hk * p.G + (r - tok * p.G);
      const uint16_t* row = p.q + (int64_t)seq * p.qsb + (int64_t)tok * p.qst + (int64_t)head * p.qsh + D / 4 * g;
#pragma unroll
      for (int s = 0; s < D / 32; ++s) q[t][s] = *reinterpret_cast<const uint4*>(row + 8 * s);
      lim[t] = p.causal ? min(tok + lk - lq, lk - 1) : lk - 1;
    }
    // Rows are token-major: the tile's first row sees the fewest keys.
    const int lim_lo = __builtin_amdgcn_readfirstlane(lim[0]);

    const int kb = (int)(skip * 64), ke = (int)min((skip + take) * 64, (int64_t)lk);

    f32x4 acc[RT][DV];
    float m[RT], l[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
#pragma unroll
      for (int u = 0; u < DV; ++u) acc[t][u] = (f32x4){0.f, 0.f, 0.f, 0.f};
      m[t] = -3.4028234663852886e38f;
      l[t] = 0.f;
    }

    // A lane's part of a row: K D / 8 bytes at D / 8 g; V 4 bytes at 4 i16 (D = 64: at 4 (i16 & 7), of the keys 32 .. 63
    // in the lanes i16 >= 8).
    const uint8_t *const kcodes = p.kc + hk * p.khead, *const vcodes = p.vc + hk * p.vhead;
    const uint32_t klane = D / 8 * g, vlane = 4 * (D == 128 ? i16 : i16 & 7);
    const uint8_t* kscales = p.ksc + hk * p.kssh;
    const uint8_t* vscales = p.vsc + hk * p.vssh;
    const int32_t* trow = p.table + (int64_t)__builtin_amdgcn_readfirstlane(seq) * p.table_stride;
    // A scale byte as a float's exponent (the conversions read no more of it), from byte 0 to 3 of a word.
    auto unit_of = [](uint32_t scales, int byte) __attribute__((always_inline)) {
      return __uint_as_float(__builtin_amdgcn_alignbit(scales, scales, (8 * byte + 9) & 31) & 0x7f800000u);
    };
    // Which 32 of a row the lane's dims belong to.
    const int kgroup = D == 128 ? g : g >> 1, vgroup = D == 128 ? i16 >> 2 : (i16 & 7) >> 2;

    // Page and slot of key j0 + lane (RUNS: of key j0 + 16 (lane & 3)).
    struct Where {
      int id, at;
    };
    auto find = [&](int j0) __attribute__((always_inline)) {
      Where w;
      const int key = min(RUNS ? j0 + 16 * (lane & 3) : j0 + lane, lk - 1);  // lk > 0 here
      int pg = (int)__umulhi((uint32_t)key, p.page_inverse);               // at most one too few
      w.at = key - pg * p.page;
      if (w.at >= p.page) {
        ++pg;
        w.at -= p.page;
      }
      w.id = trow[pg];
      return w;
    };
    struct Block {
      KWord k[4];
      uint32_t v[VW];
      uint32_t ks[RUNS ? 4 : 1];           // scales: RUNS: of key 16 t + i16, and of keys 16 t + 4 g .. + 3;
      uint32_t vs[RUNS ? 4 * D / 32 : 1];  // else of key j0 + lane
      uint64_t ok;                         // bit j: key j of the block is one
    };
    // RUNS: fixed offsets of the lanes; a run's own is the scalar offset of a buffer load.
    const uint32_t krun = 16 * i16 * p.kut + klane;
    uint32_t vrun[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) vrun[r] = 16 * (4 * g + r) * p.vut + vlane;
    const auto kbuf = uniform_rsrc(reinterpret_cast<const char*>(kcodes)), vbuf = uniform_rsrc(reinterpret_cast<const char*>(vcodes));
    const auto ksbuf = uniform_rsrc(reinterpret_cast<const char*>(kscales)), vsbuf = uniform_rsrc(reinterpret_cast<const char*>(vscales));
    auto fetch = [&](const Where& w, int j0, Block& b) __attribute__((always_inline)) {
      if constexpr (RUNS) {
        const int n = min(ke - (j0 + 16 * (lane & 3)), 16);
        const bool ok = n > 0 && (uint32_t)w.id < (uint32_t)p.pages;
        const uint32_t id = ok ? w.id : 0, at = ok ? w.at : 0;
        const uint32_t ko = (id * p.kup + at * p.kut) << 4, vo = (id * p.vup + at * p.vut) << 4;
        const uint32_t kso = id * (uint32_t)p.kssp + at * (D / 32), vso = id * (uint32_t)p.vssp + at * (D / 32);
        b.ok = ~0ull;
        if (__builtin_amdgcn_ballot_w64(!ok || n < 16) != 0ull) {
          const uint32_t bits = ok ? 0xFFFFu >> (16 - n) : 0u;
          b.ok = (uint64_t)(uint32_t)(lane_of((int)bits, 0) | lane_of((int)bits, 1) << 16) |
                 (uint64_t)(uint32_t)(lane_of((int)bits, 2) | lane_of((int)bits, 3) << 16) << 32;
        }
        const uint32_t vhalf[2] = {(uint32_t)__shfl((int)vo, 2 * (i16 >> 3)), (uint32_t)__shfl((int)vo, 2 * (i16 >> 3) + 1)};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int ks = lane_of((int)kso, i), vs = lane_of((int)vso, i);
          if constexpr (D == 128) {
            b.ks[i] = __builtin_amdgcn_raw_buffer_load_b32(ksbuf, i16 * 4, ks, 0);
            const auto x = __builtin_amdgcn_raw_buffer_load_b128(vsbuf, g * 16, vs, 0);
#pragma unroll
            for (int j = 0; j < 4; ++j) b.vs[4 * i + j] = x[j];
          } else {
            b.ks[i] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(ksbuf, i16 * 2, ks, 0);
            const auto x = __builtin_amdgcn_raw_buffer_load_b64(vsbuf, g * 8, vs, 0);
            b.vs[2 * i] = x[0];
            b.vs[2 * i + 1] = x[1];
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (D == 128) {
            const auto x = __builtin_amdgcn_raw_buffer_load_b128(kbuf, krun, lane_of((int)ko, i), 0);
            b.k[i] = make_uint4(x[0], x[1], x[2], x[3]);
          } else {
            const auto x = __builtin_amdgcn_raw_buffer_load_b64(kbuf, krun, lane_of((int)ko, i), 0);
            b.k[i] = make_uint2(x[0], x[1]);
          }
        }
#pragma unroll
        for (int j = 0; j < VW; ++j)
          b.v[j] = D == 128 ? __builtin_amdgcn_raw_buffer_load_b32(vbuf, vrun[j & 3], lane_of((int)vo, j >> 2), 0)
                            : __builtin_amdgcn_raw_buffer_load_b32(vbuf, vrun[j & 3] + vhalf[(j >> 2) & 1], 0, 0);
      } else {
        const bool ok = j0 + lane < ke && (uint32_t)w.id < (uint32_t)p.pages;
        b.ok = __builtin_amdgcn_ballot_w64(ok);
        const int64_t id = ok ? w.id : 0, at = ok ? w.at : 0;
        b.ks[0] = b.vs[0] = 0u;
        if (ok) {
          const uint8_t* ks = kscales + id * p.kssp + at * p.ksst;
          const uint8_t* vs = vscales + id * p.vssp + at * p.vsst;
          if constexpr (D == 128) {
            b.ks[0] = *reinterpret_cast<const uint32_t*>(ks);
            b.vs[0] = *reinterpret_cast<const uint32_t*>(vs);
          } else {
            b.ks[0] = *reinterpret_cast<const uint16_t*>(ks);
            b.vs[0] = *reinterpret_cast<const uint16_t*>(vs);
          }
        }
        const uint32_t ko = (uint32_t)id * p.kup + (uint32_t)at * p.kut, vo = (uint32_t)id * p.vup + (uint32_t)at * p.vut;
        // All exchanges first, then the loads: one by one, each would wait for its own.
        uint32_t krow[4], vrow[VW];
#pragma unroll
        for (int t = 0; t < 4; ++t) krow[t] = (uint32_t)__shfl((int)ko, 16 * t + i16);
#pragma unroll
        for (int j = 0; j < VW; ++j)
          vrow[j] = (uint32_t)__shfl((int)vo, 32 * (D == 128 ? j >> 3 : i16 >> 3) + 16 * ((j >> 2) & 1) + 4 * g + (j & 3));
#pragma unroll
        for (int j = 0; j < VW; j += 8)
          asm volatile("" : "+v"(vrow[j]), "+v"(vrow[j + 1]), "+v"(vrow[j + 2]), "+v"(vrow[j + 3]), "+v"(vrow[j + 4]),
                       "+v"(vrow[j + 5]), "+v"(vrow[j + 6]), "+v"(vrow[j + 7]));
#pragma unroll
        for (int t = 0; t < 4; ++t) b.k[t] = *reinterpret_cast<const KWord*>(kcodes + klane + ((uint64_t)krow[t] << 4));
#pragma unroll
        for (int j = 0; j < VW; ++j)
          b.v[j] = *reinterpret_cast<const uint32_t*>(vcodes + vlane + ((uint64_t)vrow[j] << 4));
      }
    };
    // Units of key 32 h + 16 t + i16 of K, and of key 32 h + 16 (j >> 2) + 4 g + (j & 3) of V, for the lane's dims.
    auto k_unit = [&](const Block& b, int h, int t) __attribute__((always_inline)) {
      return unit_of(RUNS ? b.ks[RUNS ? 2 * h + t : 0] : (uint32_t)__shfl((int)b.ks[0], 32 * h + 16 * t + i16), kgroup);
    };
    auto v_unit = [&](const Block& b, int h, int j) __attribute__((always_inline)) {
      if constexpr (!RUNS) return unit_of((uint32_t)__shfl((int)b.vs[0], 32 * h + 16 * (j >> 2) + 4 * g + (j & 3)), vgroup);
      const int i = 2 * h + (j >> 2), r = j & 3;
      return D == 128 ? unit_of(b.vs[RUNS ? i * 4 + r : 0], vgroup) : unit_of(b.vs[RUNS ? i * 2 + (r >> 1) : 0], vgroup + 2 * (r & 1));
    };

    bool unclean = false;
    auto compute = [&](int j0, Block& b) __attribute__((always_inline)) {
      if constexpr (D == 64) {
        // Words of keys 0 .. 31 in the lanes i16 < 8, of keys 32 .. 63 in the others, become words whose low half is
        // of keys 0 .. 31 and the high half of keys 32 .. 63: dims 8 (i16 & 7) + 4 (i16 >> 3) .. + 3.
        const uint32_t pick = i16 < 8 ? 0x05040100u : 0x03020706u;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          b.v[j] = __builtin_amdgcn_perm((uint32_t)__builtin_amdgcn_update_dpp(0, (int)b.v[j], 0x128, 0xF, 0xF, true), b.v[j],
                                         pick);  // row_ror 8
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int jh = j0 + 32 * h;
        if (jh >= ke) break;
        const uint32_t ok = (uint32_t)(b.ok >> (32 * h));
        f32x4 sc[RT][2];
        const float ku[2] = {k_unit(b, h, 0), k_unit(b, h, 1)};
        // Keys whose dims all lie in fp16's range take the products in fp16, whatever the other keys of the wave are: a
        // row's scores keep their bits when a key that it does not see, or an unused slot, changes.
        uint64_t fits[2] = {~0ull, ~0ull};
        if constexpr (__is_same(E, FP16)) {
          fits[0] = __builtin_amdgcn_ballot_w64(fp4_fits_fp16(ku[0]));
          fits[1] = __builtin_amdgcn_ballot_w64(fp4_fits_fp16(ku[1]));
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) sc[rt][t] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int s = 0; s < D / 32; ++s) {
            const uint4 x = fp4_operand<E>(reinterpret_cast<const uint32_t*>(&b.k[2 * h + t])[s], ku[t]);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) sc[rt][t] = mma16(E{}, x, q[rt][s], sc[rt][t]);
          }
          if (__builtin_expect(fits[t] != ~0ull, 0)) {
            // Bit u: key 16 t + 4 g + u is of that kind (lanes i, i + 16, i + 32 and i + 48 hold parts of key i).
            uint32_t mine = (uint32_t)fits[t] & (uint32_t)(fits[t] >> 32);
            mine = (mine & mine >> 16) >> (4 * g);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
              f32x4 wide = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
              for (int s = 0; s < D / 32; ++s) {
                const uint4 x = fp4_operand<BF16>(reinterpret_cast<const uint32_t*>(&b.k[2 * h + t])[s], ku[t]);
                uint4 high, low, x16 = q[rt][s];
                asm volatile("" : "+v"(x16.x), "+v"(x16.y), "+v"(x16.z), "+v"(x16.w));  // here, not ahead of the loop
                fp4_split_query(x16, high, low);
                wide = mma16(BF16{}, x, high, wide);
                wide = mma16(BF16{}, x, low, wide);
              }
#pragma unroll
              for (int u = 0; u < 4; ++u) sc[rt][t][u] = (mine >> u) & 1u ? sc[rt][t][u] : wide[u];
            }
          }
        }
        float unit[8];
        uint32_t top = 0u;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          unit[j] = v_unit(b, h, j);
          top = max(top, __float_as_uint(unit[j]));
        }
        if (RUNS && ok != 0xFFFFFFFFu) {  // (else the scales of what is no key are 0 already)
          const uint32_t mine = ok >> (4 * g);
          top = 0u;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if (!((mine >> (16 * (j >> 2) + (j & 3))) & 1u)) unit[j] = 0.f;
            top = max(top, __float_as_uint(unit[j]));
          }
        }
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(top >= kFp4Beyond << 23) != 0ull, 0)) {  // seen to afterwards
          unclean = true;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            uint32_t& x = b.v[D == 128 ? 8 * h + j : j];  // D = 64: this half's values are in its low or high 16 bits
            const uint32_t half = D == 128 ? 0xFFFFFFFFu : h == 0 ? 0xFFFFu : 0xFFFF0000u;
            const uint32_t scale = __float_as_uint(unit[j]) >> 23;
            x &= ~(fp4_beyond(x, scale) & half);
            if (scale == kFp4NaN) unit[j] = 0.f;
          }
        }
        uint32_t hi[RT][4], lo[RT][4];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          f32x4(&s)[2] = sc[rt];
          if (ok != 0xFFFFFFFFu || jh + 31 > lim_lo) {
            const uint32_t mine = ok >> (4 * g);
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
              for (int u = 0; u < 4; ++u)
                if (!((mine >> (16 * t + u)) & 1u) || jh + 16 * t + 4 * g + u > lim[rt]) s[t][u] = -INFINITY;
          }
          float w[8];
          auto weights = [&](float nm) __attribute__((always_inline)) {
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
              for (int u = 0; u < 4; ++u) w[4 * t + u] = fexp2(fmaf(s[t][u], p.scale_log2, nm));
            return ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
          };
          float ls = weights(-m[rt]);
          if (__builtin_expect(__builtin_amdgcn_ballot_w64(!(ls <= kPkSumCap<BF16>)) != 0ull, 0)) {
            const bool up = rows_max(ls <= kPkSumCap<BF16> ? 0.f : 1.f) > 0.f;  // this row, not the tile's others
            float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                             fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
            mx = rows_max(mx);
            const float mn = up ? fmaxf(m[rt], mx * p.scale_log2) : m[rt];
            const float alpha = fexp2(m[rt] - mn);
            m[rt] = mn;
            l[rt] *= alpha;
#pragma unroll
            for (int u = 0; u < DV; ++u) acc[rt][u] *= alpha;
            ls = weights(-mn);
          }
          l[rt] += ls;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            hi[rt][i] = pack_pair(BF16{}, w[2 * i], w[2 * i + 1]);
            float a, c;
            unpack2(BF16{}, hi[rt][i], a, c);
            lo[rt][i] = pack_pair(BF16{}, w[2 * i] - a, w[2 * i + 1] - c);
          }
        }
        // Two dims at a time: their values of eight keys, pairs of dims turned into pairs of keys.
        auto two = [&](auto byte, int u) __attribute__((always_inline)) {
          uint32_t x[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] = fp4_pair<decltype(byte)::value>(BF16{}, b.v[D == 128 ? 8 * h + j : j], unit[j]);
          uint32_t a[2][4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            a[0][i] = __builtin_amdgcn_perm(x[2 * i + 1], x[2 * i], 0x05040100u);
            a[1][i] = __builtin_amdgcn_perm(x[2 * i + 1], x[2 * i], 0x07060302u);
          }
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const uint4 v = make_uint4(a[n][0], a[n][1], a[n][2], a[n][3]);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
              acc[rt][u + n] = mma16(BF16{}, v, make_uint4(hi[rt][0], hi[rt][1], hi[rt][2], hi[rt][3]), acc[rt][u + n]);
              acc[rt][u + n] = mma16(BF16{}, v, make_uint4(lo[rt][0], lo[rt][1], lo[rt][2], lo[rt][3]), acc[rt][u + n]);
            }
          }
        };
        if constexpr (D == 128) {
          two(std::integral_constant<int, 0>{}, 0);
          two(std::integral_constant<int, 1>{}, 2);
          two(std::integral_constant<int, 2>{}, 4);
          two(std::integral_constant<int, 3>{}, 6);
        } else if (h == 0) {
          two(std::integral_constant<int, 0>{}, 0);
          two(std::integral_constant<int, 1>{}, 2);
        } else {
          two(std::integral_constant<int, 2>{}, 0);
          two(std::integral_constant<int, 3>{}, 2);
        }
      }
    };

    const int j_first = kb + 64 * wave;
    if (j_first < ke) {
      // Blocks of this wave every 256 keys. The order of the loads (pages, then the next block's rows) lets a wait for
      // either leave what was issued behind it in flight.
      Block b0, b1;
      Where w0 = find(j_first), w1 = find(j_first + 256);
      fetch(w0, j_first, b0);
      int j = j_first;
#pragma unroll 1
      while (true) {
        w0 = find(j + 512);
        fetch(w1, j + 256, b1);
        compute(j, b0);
        if (j + 256 >= ke) break;
        w1 = find(j + 768);
        fetch(w0, j + 512, b0);
        compute(j + 256, b1);
        if (j + 512 >= ke) break;
        j += 512;
      }
    }

    // Dim of entry u of accumulator row r = 4 g + rr (its operand row, i16 above).
    auto dim_of = [](int r, int u) { return D == 128 ? 8 * r + u : 8 * (r & 7) + 4 * (r >> 3) + u; };
    if (__builtin_expect(unclean, 0)) {
      // This wave's values that are no finite numbers go to the rows that see them.
      for (int j0 = j_first; j0 < ke; j0 += 256) {
        for (int i = 0; i < min(64, ke - j0); ++i) {
          const int pg = (j0 + i) / p.page, id = trow[pg];
          if ((uint32_t)id >= (uint32_t)p.pages) continue;
          const int at = j0 + i - pg * p.page;
          // The lane's dims are of one power.
          const uint32_t scale = (vscales + id * p.vssp + at * p.vsst)[D == 128 ? g : g & 1];
          if (scale < kFp4Beyond) continue;
          const uint8_t* codes = vcodes + ((uint64_t)((uint32_t)id * p.vup + (uint32_t)at * p.vut) << 4);
#pragma unroll
          for (int rr = 0; rr < 4; ++rr) {
            const uint8_t* word = codes + dim_of(4 * g + rr, 0) / 2;
            const uint32_t w = D == 128 ? *reinterpret_cast<const uint32_t*>(word) : *reinterpret_cast<const uint16_t*>(word);
            const uint32_t hit = fp4_beyond(w, scale);
#pragma unroll
            for (int u = 0; u < DV; ++u) {
              if (!((hit >> (4 * u)) & 1u)) continue;
              const float f = scale == kFp4NaN ? __uint_as_float(0x7fc00000u) : (w >> (4 * u)) & 8u ? -INFINITY : INFINITY;
#pragma unroll
              for (int rt = 0; rt < RT; ++rt)
                if (j0 + i <= lim[rt]) acc[rt][u][rr] += f;
            }
          }
        }
      }
    }

    // The four waves' parts, joined in wave order, a row tile at a time.
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      if (t > 0) __syncthreads();
      const float lw = rows_sum(l[t]);
      if (g == 0) {
        sm[wave][i16] = m[t];
        sl[wave][i16] = lw;
      }
#pragma unroll
      for (int rr = 0; rr < 4; ++rr)
#pragma unroll
        for (int u = 0; u < DV; ++u) so[wave][i16][dim_of(4 * g + rr, u)] = acc[t][u][rr];
      __syncthreads();
      const int row = threadIdx.x >> 4, c = threadIdx.x & 15;  // 16 threads per row, DV dims each
      const int rr = tile * ROWS + t * kRows + row;
      if (rr >= rows) continue;
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
      if (parts > 1) {
        const int64_t at = ((int64_t)(2 * unit + (part == 0)) * p.Hk + hk) * ROWS + t * kRows + row;
        float* dst = p.part + at * D + c * DV;
#pragma unroll
        for (int u = 0; u < DV; u += 4)
          *reinterpret_cast<float4*>(dst + u) = make_float4(out[u], out[u + 1], out[u + 2], out[u + 3]);
        if (c == 0) p.part_lse[at] = l2;
        continue;
      }
      const int tk = rr / p.G, hd = hk * p.G + (rr - tk * p.G);
      uint16_t* dst = p.o + (int64_t)seq * p.osb + (int64_t)tk * p.ost + (int64_t)hd * p.osh + c * DV;
#pragma unroll
      for (int u = 0; u < DV; u += 4) pk_store4<E>(dst + u, nullptr, out[u], out[u + 1], out[u + 2], out[u + 3]);
      if (c == 0 && p.lse) p.lse[(int64_t)(seq * p.Tq + tk) * p.H + hd] = l2 * kDLn2;
    }
    left -= take;
    if (!p.split || left <= 0) return;
    // The next row tile: that of the next sequence, or of the first.
    begin += blocks;
    if (++seq == p.n) {
      seq = 0;
      ++tile;
    }
    lk = fp4_length(p, seq);
    __syncthreads();  // the joins' rows
  }
}

// ---------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------

// Row tiles of a workgroup: two where there are more than 16 rows.
int fp4_row_tiles(int64_t N, int64_t G) { return N * G > kRows ? 2 : 1; }

// Whether the keys are split: up to eight rounds of the chip's workgroups by the row tiles alone (as paged_split in
// rows_attn_fwd.hip: every workgroup of a split call scans the lengths).
bool fp4_split(int64_t B, int64_t N, int64_t Hq, int64_t Hk) {
  const int64_t rows = kRows * fp4_row_tiles(N, Hq / Hk);
  return B * ((N * (Hq / Hk) + rows - 1) / rows) * Hk < 4096;
}

// Units per key head of a split call.
int fp4_units(int64_t D, int RT, int64_t Hk) {
  const int64_t n = 256 * fp4_resident((int)D, RT) / Hk;
  return (int)(n > 0 ? n : 1);
}

template <typename E, int D, int RT>
int fp4_launch(const Fp4AttnParams& p, bool runs, hipStream_t stream) {
  constexpr int ROWS = kRows * RT;
  const int64_t tiles = rows_tiles(true, p.n, p.Tq, p.G, ROWS), joins = tiles * p.Hk;
  const int64_t grid = (p.split ? p.want : tiles) * p.Hk;
  GW_CHECK_GRID(grid, 256);
  if (p.split) GW_CHECK_GRID(joins, 256);
  if (runs) {
    hipLaunchKernelGGL((fp4_attn_kernel<E, D, RT, true>), dim3((uint32_t)grid), dim3(256), 0, stream, p);
  } else {
    hipLaunchKernelGGL((fp4_attn_kernel<E, D, RT, false>), dim3((uint32_t)grid), dim3(256), 0, stream, p);
  }
  GW_HIP_LAUNCH_CHECK("paged attention, 4 bits");
  if (p.split) {
    const int64_t rows = (int64_t)p.Tq * p.G;
    hipLaunchKernelGGL((rows_join_kernel<E, D, true, ROWS, true>), dim3((uint32_t)joins, (uint32_t)(rows < ROWS ? rows : ROWS)),
                       dim3(256), 0, stream, static_cast<const RowsParams&>(p));
    GW_HIP_LAUNCH_CHECK("paged attention, 4 bits (join)");
  }
  return GW_OK;
}

template <typename E>
int fp4_dim(int D, int RT, const Fp4AttnParams& p, bool runs, hipStream_t s) {
  if (D == 64) return RT == 1 ? fp4_launch<E, 64, 1>(p, runs, s) : fp4_launch<E, 64, 2>(p, runs, s);
  return RT == 1 ? fp4_launch<E, 128, 1>(p, runs, s) : fp4_launch<E, 128, 2>(p, runs, s);
}

}  // namespace
}  // namespace gw

extern "C" size_t gw_paged_attn_fp4_fwd_workspace_size(int64_t B, int64_t N, int64_t Hq, int64_t Hk, int64_t D) {
  using namespace gw;
  if (B < 1 || N < 1 || Hk < 1 || Hq < Hk || D < 1 || N > 0x7FFFFFFFll || Hq > 0x7FFFFFFFll || B > 0x7FFFFFFFll / Hq / N ||
      !fp4_split(B, N, Hq, Hk))
    return 0;
  const int RT = fp4_row_tiles(N, Hq / Hk);
  const int64_t rows = kRows * RT;
  return (size_t)2 * fp4_units(D, RT, Hk) * Hk * rows * (D + 1) * sizeof(float) +
         (size_t)rows_tiles(true, B, N, Hq / Hk, rows) * sizeof(int2);
}

extern "C" int gw_paged_attn_fp4_fwd(int dtype, const void* q, const int64_t* q_strides, const void* k,
                                     const int64_t* k_strides, const void* k_scales, const int64_t* k_scale_strides,
                                     const void* v, const int64_t* v_strides, const void* v_scales,
                                     const int64_t* v_scale_strides, const int32_t* block_table, int64_t table_stride,
                                     const int32_t* lens, void* o, const int64_t* o_strides, float* lse, int64_t B,
                                     int64_t N, int64_t Hq, int64_t Hk, int64_t D, int64_t pages, int64_t page_size,
                                     int64_t table_width, int causal, float softmax_scale, void* workspace,
                                     size_t workspace_bytes, void* stream) {
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
  GW_CHECK_ARG(q && o && lens && q_strides && k_strides && v_strides && o_strides && k_scale_strides && v_scale_strides,
               "a tensor is missing");
  GW_CHECK_ARG((k && v && k_scales && v_scales) || pages == 0, "the cache is missing");
  GW_CHECK_ARG(block_table || table_width == 0, "the block table is missing");
  auto ok = [](const void* x, const int64_t* s, int64_t unit) {
    return aligned16(x) && s[0] % unit == 0 && s[1] % unit == 0 && s[2] % unit == 0;
  };
  GW_CHECK_ARG(ok(q, q_strides, 8) && ok(o, o_strides, 8) && ok(k, k_strides, 16) && ok(v, v_strides, 16),
               "q, k, v and o need 16-byte aligned rows");
  const int64_t per = D / 32;
  auto scales_ok = [per](const void* x, const int64_t* s) {
    return reinterpret_cast<uintptr_t>(x) % per == 0 && s[0] % per == 0 && s[1] % per == 0 && s[2] % per == 0;
  };
  GW_CHECK_ARG(scales_ok(k_scales, k_scale_strides) && scales_ok(v_scales, v_scale_strides),
               "scales need rows aligned to their %lld bytes", (long long)per);
  for (const int64_t* s : {k_scale_strides, v_scale_strides})
    GW_CHECK_ARG(s[0] >= 0 && s[1] >= 0 && s[2] >= 0, "negative strides of a cache");
  for (const int64_t* s : {k_strides, v_strides}) {
    GW_CHECK_ARG(s[0] >= 0 && s[1] >= 0 && s[2] >= 0, "negative strides of a cache");
    // Offsets of rows are 32 bits of 16 bytes.
    const unsigned __int128 span = (unsigned __int128)s[0] * (uint64_t)(pages > 0 ? pages - 1 : 0) +
                                   (unsigned __int128)s[1] * (uint64_t)(page_size - 1);
    if (span >= ((unsigned __int128)1 << 36)) return set_error(GW_ERR_UNSUPPORTED, "a cache of more than 2^36 bytes of codes");
  }
  Fp4AttnParams p = {};
  p.q = static_cast<const uint16_t*>(q);
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
  p.kc = static_cast<const uint8_t*>(k);
  p.vc = static_cast<const uint8_t*>(v);
  p.ksc = static_cast<const uint8_t*>(k_scales);
  p.vsc = static_cast<const uint8_t*>(v_scales);
  p.kup = (uint32_t)(k_strides[0] / 16);
  p.kut = (uint32_t)(k_strides[1] / 16);
  p.khead = k_strides[2];
  p.vup = (uint32_t)(v_strides[0] / 16);
  p.vut = (uint32_t)(v_strides[1] / 16);
  p.vhead = v_strides[2];
  p.kssp = k_scale_strides[0];
  p.ksst = k_scale_strides[1];
  p.kssh = k_scale_strides[2];
  p.vssp = v_scale_strides[0];
  p.vsst = v_scale_strides[1];
  p.vssh = v_scale_strides[2];
  p.page_inverse = page_size == 1 ? 0xFFFFFFFFu : (uint32_t)((1ull << 32) / (uint64_t)page_size);
  p.scale_log2 = softmax_scale * kDLog2e;
  p.split = fp4_split(B, N, Hq, Hk);
  const size_t need = gw_paged_attn_fp4_fwd_workspace_size(B, N, Hq, Hk, D);
  GW_CHECK_ARG(need == 0 || (workspace && aligned16(workspace) && workspace_bytes >= need),
               "workspace of %zu bytes, %zu are needed", workspace_bytes, need);
  const int RT = fp4_row_tiles(N, Hq / Hk);
  p.want = fp4_units(D, RT, Hk);
  if (p.split) {
    const int64_t rows = kRows * RT;
    p.part = static_cast<float*>(workspace);
    p.part_lse = p.part + (int64_t)2 * p.want * p.Hk * rows * D;
    p.cut = reinterpret_cast<int2*>(p.part_lse + (int64_t)2 * p.want * p.Hk * rows);
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  // Runs of 16 slots: scales slot behind slot, a lane's of four keys (D / 8 bytes) in one aligned load, and a head's rows within
  // 32-bit offsets.
  auto within = [&](const int64_t* st, int64_t row) {
    return st[0] < (1ll << 31) && st[1] < (1ll << 27) && st[0] * (pages > 0 ? pages - 1 : 0) + st[1] * (page_size - 1) + row < (1ll << 32);
  };
  auto scale_runs = [&](const void* x, const int64_t* st) {
    return st[1] == D / 32 && reinterpret_cast<uintptr_t>(x) % 16 == 0 && st[0] % 16 == 0 && st[2] % 16 == 0 && within(st, D / 32);
  };
  const bool runs = page_size % 16 == 0 && scale_runs(k_scales, k_scale_strides) && scale_runs(v_scales, v_scale_strides) &&
                    within(k_strides, D / 2) && within(v_strides, D / 2);
  return dtype == GW_DTYPE_BF16 ? fp4_dim<BF16>((int)D, RT, p, runs, s) : fp4_dim<FP16>((int)D, RT, p, runs, s);
}
