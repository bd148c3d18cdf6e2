// Attention of a few new tokens per sequence over a paged cache in 4 bits (gfx950). D = 64 or 128.
//
// Formulas, parts and joins are those of rows_attn_fwd.hip; the cache's format is in gw_fp4.h. What a key
// costs is its 17/16 D bytes (K and V), a quarter of a 16-bit cache's, so here the instructions per key count:
//
// Codes become bf16 by the conversion instruction, two values of a row at a time with their power of two: exact, so that
// the products are those of the values themselves.
//   S^T = K Q^T (16x16x32): lane (g, i) reads the D / 4 dims from D / 4 g on of key i, which are its operands of the
// D / 32 products one after the other, and holds q of row i in the same order (fp16: as two bf16 terms, exact).
// The block-scaled product (16x16x128, fp4 x fp8, q in e4m3 terms) would take K without a conversion, but sums
// 2^-17 of the magnitudes off (measured; 3e-4 in a score of 13 whose magnitudes are 32), and is not faster here.
//   O^T += V^T P^T (16x16x32): the scores of a lane stand for eight keys; exchanging halves between those keys'
// registers gives the operand of each product. P is the sum of two bf16 terms (16 bits; one term has 2^-9, which is a
// 16-bit output's own rounding again, and fp16 would bound V's range).
//
// A wave takes 64 keys at a time, one lane each for the page, the slot and the scales, which it hands to the
// lanes that need them; the next 64 keys' rows are in flight meanwhile, and the page numbers of the 64 behind.
//
// Rows that are not keys (behind the length, in a page outside the pool) are masked, and their scales are 2^-127:
// what lies there cannot reach a result. Codes are always finite; a scale of 255 makes 32 values NaN: such values of V
// count as 0 in the products and are added afterwards to the rows that see them.
#include <math.h>
#include <string.h>

#include <type_traits>

#include "gw_fp4.h"
#include "gw_rows_dev.h"

namespace gw {
namespace {

struct Fp4AttnParams : RowsParams {
  const uint8_t* kc;
  const uint8_t* vc;
  const uint8_t* ksc;
  const uint8_t* vsc;
  int64_t kssp, ksst, kssh, vssp, vsst, vssh;  // scales: per page, slot, head (bytes)
  uint32_t kup, kut, vup, vut;                 // codes: per page and slot, in units of 16 bytes
  int64_t khead, vhead;                        // codes: per head (bytes)
};

// A lane's dims of a row of q as bf16 operands, and for fp16 what their rounding leaves (at most three bits: exact).
template <typename E, int D>
struct Fp4Query {
  static constexpr int TERMS = __is_same(E, FP16) ? 2 : 1;
  uint4 b[TERMS][D / 32];

  __device__ __forceinline__ void load(const uint16_t* row) {
#pragma unroll
    for (int s = 0; s < D / 32; ++s) {
      const uint4 x = *reinterpret_cast<const uint4*>(row + 8 * s);
      if constexpr (TERMS == 1) {
        b[0][s] = x;
      } else {
        float f[8], rest[8];
        unpack8<FP16>(x, f);
        b[0][s] = pack_quad<BF16>(f);
        unpack8<BF16>(b[0][s], rest);
#pragma unroll
        for (int j = 0; j < 8; ++j) rest[j] = rest[j] == f[j] ? 0.f : f[j] - rest[j];  // inf leaves nothing
        b[1][s] = pack_quad<BF16>(rest);
      }
    }
  }
};

template <typename E, int D, int RT>
__global__ __launch_bounds__(256, 2) void fp4_attn_kernel(const Fp4AttnParams p) {
  constexpr int DV = D / 16, ROWS = kRows * RT;
  typedef typename std::conditional<D == 128, uint4, uint2>::type KWord;  // what a lane reads of a key of K
  constexpr int VW = D == 128 ? 16 : 8;  // words of V that a lane reads of 64 keys
  __shared__ float so[4][kRows][D + 4];
  __shared__ float sm[4][kRows], sl[4][kRows];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, i16 = lane & 15;
  const int hk = blockIdx.x % p.Hk, slot = blockIdx.x / p.Hk;
  const RowsPart pt = rows_find<true, ROWS>(p, slot, lane);
  if (pt.seq < 0) return;
  if (p.split && pt.part == 0 && hk == 0 && threadIdx.x == 0)  // for the join
    p.cut[pt.seq * ((p.Tq * p.G + ROWS - 1) / ROWS) + pt.tile] = make_int2(pt.first, pt.parts);
  const RowsSeq sq = rows_seq<true>(p, pt.seq);
  const int lk = __builtin_amdgcn_readfirstlane(sq.lk);
  const int rows = sq.lq * p.G;

  Fp4Query<E, D> q[RT];
  int lim[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int r = min(pt.tile * ROWS + t * kRows + i16, rows - 1);
    const int tok = r / p.G, head = hk * p.G + (r - tok * p.G);
    q[t].load(p.q + (int64_t)pt.seq * p.qsb + (int64_t)tok * p.qst + (int64_t)head * p.qsh + D / 4 * g);
    lim[t] = p.causal ? min(tok + lk - sq.lq, lk - 1) : lk - 1;
  }
  // Rows are token-major: the tile's first row sees the fewest keys.
  const int lim_lo = __builtin_amdgcn_readfirstlane(lim[0]);

  const int kb = (int)min((int64_t)pt.part * pt.len, (int64_t)lk);
  const int ke = (int)min((int64_t)kb + pt.len, (int64_t)lk);

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
  const uint8_t* kbase = p.kc + hk * p.khead + D / 8 * g;
  const uint8_t* vbase = p.vc + hk * p.vhead + 4 * (D == 128 ? i16 : i16 & 7);
  const uint8_t* kscales = p.ksc + hk * p.kssh;
  const uint8_t* vscales = p.vsc + hk * p.vssh;
  const int32_t* trow = p.table + (int64_t)pt.seq * p.table_stride;
  // Rotations that bring the scale byte of a lane's dims to a float's exponent.
  const int krotate = (8 * (D == 128 ? g : g >> 1) + 9) & 31;
  const int vrotate = (8 * (D == 128 ? i16 >> 2 : (i16 & 7) >> 2) + 9) & 31;
  auto unit_of = [](uint32_t scales, int rotate) __attribute__((always_inline)) {
    return __uint_as_float(__builtin_amdgcn_alignbit(scales, scales, rotate) & 0x7f800000u);
  };

  // Block of 64 keys, lane j's key j0 + j: its page number.
  struct Page {
    int id, at;
  };
  auto find = [&](int j0) __attribute__((always_inline)) {
    Page w;
    const int key = min(j0 + lane, lk - 1);  // lk > 0 here
    const int pg = key / p.page;
    w.at = key - pg * p.page;
    w.id = trow[pg];
    return w;
  };
  struct Block {
    KWord k[4];
    uint32_t v[VW];
    uint32_t ks, vs;  // this lane's key's scales
    uint64_t ok;      // bit j: key j of the block is one
  };
  auto fetch = [&](const Page& w, int j0, Block& b) __attribute__((always_inline)) {
    const bool ok = j0 + lane < ke && (uint32_t)w.id < (uint32_t)p.pages;
    b.ok = __builtin_amdgcn_ballot_w64(ok);
    const int64_t id = ok ? w.id : 0, at = ok ? w.at : 0;
    b.ks = b.vs = 0u;
    if (ok) {
      const uint8_t* ks = kscales + id * p.kssp + at * p.ksst;
      const uint8_t* vs = vscales + id * p.vssp + at * p.vsst;
      if constexpr (D == 128) {
        b.ks = *reinterpret_cast<const uint32_t*>(ks);
        b.vs = *reinterpret_cast<const uint32_t*>(vs);
      } else {
        b.ks = *reinterpret_cast<const uint16_t*>(ks);
        b.vs = *reinterpret_cast<const uint16_t*>(vs);
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
    for (int t = 0; t < 4; ++t) b.k[t] = *reinterpret_cast<const KWord*>(kbase + ((uint64_t)krow[t] << 4));
#pragma unroll
    for (int j = 0; j < VW; ++j) b.v[j] = *reinterpret_cast<const uint32_t*>(vbase + ((uint64_t)vrow[j] << 4));
  };

  bool unclean = false;
  auto compute = [&](int j0, Block& b) __attribute__((always_inline)) {
    // A power of two that is not a number, in V: 0 here, and seen to afterwards.
    uint32_t bad = b.vs & (b.vs >> 4) & 0x0F0F0F0Fu;
    bad &= bad >> 2;
    bad &= bad >> 1;  // bit 0 of each byte: 255
    if (__builtin_expect(__builtin_amdgcn_ballot_w64((bad & 0x01010101u) != 0u) != 0ull, 0)) {
      unclean = true;
      b.vs &= ~((bad & 0x01010101u) * 255u);
    }
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
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const float unit = unit_of((uint32_t)__shfl((int)b.ks, 32 * h + 16 * t + i16), krotate);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) sc[rt][t] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < D / 32; ++s) {
          const uint32_t w = reinterpret_cast<const uint32_t*>(&b.k[2 * h + t])[s];
          const uint4 x = make_uint4(fp4_pair<0>(BF16{}, w, unit), fp4_pair<1>(BF16{}, w, unit), fp4_pair<2>(BF16{}, w, unit),
                                     fp4_pair<3>(BF16{}, w, unit));
#pragma unroll
          for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int y = 0; y < Fp4Query<E, D>::TERMS; ++y) sc[rt][t] = mma16(BF16{}, x, q[rt].b[y][s], sc[rt][t]);
        }
      }
      float unit[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) unit[j] = unit_of((uint32_t)__shfl((int)b.vs, 32 * h + 16 * (j >> 2) + 4 * g + (j & 3)), vrotate);
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
    Page w0 = find(j_first), w1 = find(j_first + 256);
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
    // This wave's values that are not numbers go to the rows that see them.
    for (int j0 = j_first; j0 < ke; j0 += 256) {
      const Page w = find(j0);
      const bool ok = j0 + lane < ke && (uint32_t)w.id < (uint32_t)p.pages;
      const uint64_t on = __builtin_amdgcn_ballot_w64(ok);
      for (int i = 0; i < 64; ++i) {
        if (!((on >> i) & 1ull)) continue;
        const uint8_t* src = vscales + (int64_t)__shfl(w.id, i) * p.vssp + (int64_t)__shfl(w.at, i) * p.vsst;
        for (int x = 0; x < D / 32; ++x) {
          if (src[x] != kFp4NaN) continue;
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) {
            if (j0 + i > lim[rt]) continue;
#pragma unroll
            for (int u = 0; u < DV; ++u)
#pragma unroll
              for (int rr = 0; rr < 4; ++rr)
                if (dim_of(4 * g + rr, u) >> 5 == x) acc[rt][u][rr] = __uint_as_float(0x7fc00000u);
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
    const int rr = pt.tile * ROWS + t * kRows + row;
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
    if (pt.parts > 1) {
      const int64_t at = ((int64_t)(pt.first + pt.part) * p.Hk + hk) * ROWS + t * kRows + row;
      float* dst = p.part + at * D + c * DV;
#pragma unroll
      for (int u = 0; u < DV; u += 4)
        *reinterpret_cast<float4*>(dst + u) = make_float4(out[u], out[u + 1], out[u + 2], out[u + 3]);
      if (c == 0) p.part_lse[at] = l2;
      continue;
    }
    const int tk = rr / p.G, hd = hk * p.G + (rr - tk * p.G);
    uint16_t* dst = p.o + (int64_t)pt.seq * p.osb + (int64_t)tk * p.ost + (int64_t)hd * p.osh + c * DV;
#pragma unroll
    for (int u = 0; u < DV; u += 4) pk_store4<E>(dst + u, nullptr, out[u], out[u + 1], out[u + 2], out[u + 3]);
    if (c == 0 && p.lse) p.lse[(int64_t)(pt.seq * p.Tq + tk) * p.H + hd] = l2 * kDLn2;
  }
}

// ---------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------

// Row tiles of a workgroup: two where there are more than 16 rows.
int fp4_row_tiles(int64_t N, int64_t G) { return N * G > kRows ? 2 : 1; }

// As paged_split in rows_attn_fwd.hip, in workgroups.
bool fp4_split(int64_t B, int64_t N, int64_t Hq, int64_t Hk) {
  const int64_t rows = kRows * fp4_row_tiles(N, Hq / Hk);
  return B * ((N * (Hq / Hk) + rows - 1) / rows) * Hk < 4096;
}

template <typename E, int D, int RT>
int fp4_launch(const Fp4AttnParams& p, hipStream_t stream) {
  constexpr int ROWS = kRows * RT;
  const int64_t tiles = rows_tiles(true, p.n, p.Tq, p.G, ROWS), joins = tiles * p.Hk;
  const int64_t grid = (tiles + (p.split ? p.want : 0)) * p.Hk;
  GW_CHECK_GRID(grid, 256);
  if (p.split) GW_CHECK_GRID(joins, 256);
  hipLaunchKernelGGL((fp4_attn_kernel<E, D, RT>), dim3((uint32_t)grid), dim3(256), 0, stream, p);
  GW_HIP_LAUNCH_CHECK("paged attention, 4 bits");
  if (p.split) {
    const int64_t rows = (int64_t)p.Tq * p.G;
    hipLaunchKernelGGL((rows_join_kernel<E, D, true, ROWS>), dim3((uint32_t)joins, (uint32_t)(rows < ROWS ? rows : ROWS)),
                       dim3(256), 0, stream, static_cast<const RowsParams&>(p));
    GW_HIP_LAUNCH_CHECK("paged attention, 4 bits (join)");
  }
  return GW_OK;
}

template <typename E>
int fp4_dim(int D, int RT, const Fp4AttnParams& p, hipStream_t s) {
  if (D == 64) return RT == 1 ? fp4_launch<E, 64, 1>(p, s) : fp4_launch<E, 64, 2>(p, s);
  return RT == 1 ? fp4_launch<E, 128, 1>(p, s) : fp4_launch<E, 128, 2>(p, s);
}

}  // namespace
}  // namespace gw

extern "C" size_t gw_paged_attn_fp4_fwd_workspace_size(int64_t B, int64_t N, int64_t Hq, int64_t Hk, int64_t D) {
  using namespace gw;
  if (B < 1 || N < 1 || Hk < 1 || Hq < Hk || D < 1 || N > 0x7FFFFFFFll || Hq > 0x7FFFFFFFll || B > 0x7FFFFFFFll / Hq / N ||
      !fp4_split(B, N, Hq, Hk))
    return 0;
  const int64_t rows = kRows * fp4_row_tiles(N, Hq / Hk);
  return rows_workspace(rows_tiles(true, B, N, Hq / Hk, rows), Hk, D, rows);
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
  for (const int64_t* s : {k_strides, v_strides}) {
    GW_CHECK_ARG(s[0] >= 0 && s[1] >= 0, "negative strides of a cache");
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
  p.scale_log2 = softmax_scale * kDLog2e;
  p.split = fp4_split(B, N, Hq, Hk);
  p.want = rows_want(Hk);
  const size_t need = gw_paged_attn_fp4_fwd_workspace_size(B, N, Hq, Hk, D);
  GW_CHECK_ARG(need == 0 || (workspace && aligned16(workspace) && workspace_bytes >= need),
               "workspace of %zu bytes, %zu are needed", workspace_bytes, need);
  const int RT = fp4_row_tiles(N, Hq / Hk);
  if (p.split) {
    const int64_t rows = kRows * RT;
    p.part = static_cast<float*>(workspace);
    p.part_lse = p.part + (int64_t)2 * p.want * p.Hk * rows * D;
    p.cut = reinterpret_cast<int2*>(p.part_lse + (int64_t)2 * p.want * p.Hk * rows);
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  return dtype == GW_DTYPE_BF16 ? fp4_dim<BF16>((int)D, RT, p, s) : fp4_dim<FP16>((int)D, RT, p, s);
}
