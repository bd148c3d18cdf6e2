// Attention over packed sequences of different lengths, forward (gfx950): bidirectional or causal,
// grouped heads, D = 64 or 128.
//
// For query token i of a sequence of Lq queries and Lk keys and head h (key head h / G):
//   p_j = softmax_j(scale q_i . k_j) over j < Lk (causal: j <= i + Lk - Lq),  o_i = sum_j p_j v_j.
// One pass over the keys with a running reference maximum m and sum l (held in fp32, in the exp2
// domain): o = (sum_j 2^(s_j - m) v_j) / l. m is raised only when a lane's 16 weights sum past a cap
// (gw_packed.h), so P fits fp16 and no maximum is taken per tile otherwise; but for roundings the result does not
// depend on which m was used, and m depends on the row's own scores alone. P is rounded to the inputs'
// 16-bit type for the second product (half a step, 2^-8 or 2^-11 of a weight, with errors that average out over
// the keys; fp16 weights below 2^-24 of a row's largest lose more, 2^-35 of that largest at most); sums add the
// fp32 weights.
//
// The rows of a key head are (token, head of the group), token-major, so a group's heads share the
// K and V tiles. 4 waves per workgroup, each QPW blocks of 32 rows; tiles of 64 keys go from memory
// straight to LDS, a tile ahead. Products are transposed (S^T = K Q^T, O^T += V^T P^T,
// v_mfma_f32_32x32x16): a lane holds 16 keys of one row, the softmax stays in its registers and the
// packed weights are the second product's operand as they are; V is read from its row-major tile by
// transposing LDS reads. The next 32 keys' scores are issued before the current weights are formed.
//
// Bound by the matrix cores and the vector unit together (one exp2, half a pack and an add per score): 43,968
// tokens x 16 heads of 64 in bf16 7.6 to 7.8 ms, 1.01 to 1.04 PFLOP/s with the matrix cores busy 55 % of the
// time; 12 causal sequences of up to 8,844 tokens, 16 heads over 4 of 128 in fp16, 1.50 ms, 0.98 PFLOP/s (57 %).
// Heads of 128 keep 36 to 40 bytes of scratch a lane, written and read outside the loops.
// Tiles by falling work, as in the backward, need a launch of their own here (7 to 14 us) and
// saved 4 us of 57 on 96 short sequences, 20 of 428 on six long ones.
//
// Rows of K and V behind a sequence's end arrive as zeros (the loads' descriptor ends there), so
// what lies in memory behind it, inf and NaN included, cannot reach a result.
#include <math.h>

#include "gw_packed.h"
#include "gw_rows.h"

namespace gw {
namespace {

struct PackedFwdParams {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  uint16_t* o;
  uint16_t* rest;  // nullable: [Tq][H][D], what the rounding of o left
  float* lse;
  const int32_t* cu_q;
  const int32_t* cu_k;
  int n, Tq, Tk, H, Hk, G, causal;
  int skip_rows;      // sequences of at most this many rows are another kernel's
  int split;          // parts that a tile's keys are cut into
  float* part;        // split > 1: [part][Tq][H][D] outputs, [part][Tq][H] log2 sums
  float* part_lse;
  int64_t qst, qsh, kst, ksh, vst, vsh, ost, osh;
  float scale_log2;
};

template <typename E, int D, int QPW>
__global__ __launch_bounds__(256, 2) void packed_attn_fwd_kernel(const PackedFwdParams p) {
  constexpr int KS = D / 16, DB = D / 32, BM = 128 * QPW;
  constexpr int kTileBytes = 64 * 2 * D;
  // Two buffers of each tile as arrays of their own, indexed at compile time: the compiler then
  // knows which LDS reads a load in flight can overlap, and waits for none of them in the loop.
  __shared__ __align__(16) uint8_t kt0[kTileBytes], kt1[kTileBytes], vt0[kTileBytes], vt1[kTileBytes];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, half = lane >> 5;
  const int hk = blockIdx.x % p.Hk;  // consecutive workgroups (different XCDs) take different heads
  const PackedTile pt = pk_find_tile(p.cu_q, p.n, p.Tq, p.G, BM, blockIdx.x / p.Hk);
  const int rows = pt.len * p.G;  // fits: the host bounds Tq * H
  const int ntile = (rows + BM - 1) / BM;
  if (pt.tile >= ntile || rows <= p.skip_rows) return;
  // Causal: the tiles with the most keys first.
  const int row0 = (p.causal ? ntile - 1 - pt.tile : pt.tile) * BM;
  int k0, lk;
  pk_other(p.cu_k, p.n, p.Tk, pt.seq, k0, lk);
  const int shift = lk - pt.len;  // causal: token i sees keys up to i + shift
  const float sl2 = p.scale_log2;

  // This lane's row of each block: its token and head, and its last key.
  int lim[QPW];
  int tok[QPW], head[QPW];
  bool on[QPW];
  uint4 qa[QPW][KS];
#pragma unroll
  for (int a = 0; a < QPW; ++a) {
    const int base = row0 + (wave * QPW + a) * 32;
    const int r = min(base + col, rows - 1);
    on[a] = base + col < rows;
    tok[a] = r / p.G;
    head[a] = hk * p.G + (r - tok[a] * p.G);
    lim[a] = p.causal ? min(tok[a] + shift, lk - 1) : lk - 1;
    const uint16_t* qr = p.q + (int64_t)(pt.start + tok[a]) * p.qst + (int64_t)head[a] * p.qsh + half * 8;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qa[a][ks] = *reinterpret_cast<const uint4*>(qr + ks * 16);
  }
  // The last keys of the wave's and of the workgroup's last row.
  auto last_key = [&](int r) { return p.causal ? min(min(r, rows - 1) / p.G + shift, lk - 1) : lk - 1; };
  const int lim_wave = row0 + wave * QPW * 32 < rows ? last_key(row0 + (wave + 1) * QPW * 32 - 1) : -1;
  const int keys = last_key(row0 + BM - 1) + 1;
  // This part's tiles of 64 keys.
  const int all = keys > 0 ? (keys + 63) >> 6 : 0;
  const int per = p.split > 1 ? (all + p.split - 1) / p.split : all;
  const int tk0 = min((int)blockIdx.y * per, all), ntk = min(per, all - tk0);

  f32x16 acc[QPW][DB];
  float m[QPW], l[QPW];  // m: the same in lanes l and l ^ 32; l: this lane's keys only
#pragma unroll
  for (int a = 0; a < QPW; ++a) {
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[a][db][r] = 0.f;
    m[a] = -3.4028234663852886e38f;  // finite: s - m stays -inf at masked entries
    l[a] = 0.f;
  }

  PkRows<D, 256> krows, vrows;
  krows.init(p.k + (int64_t)k0 * p.kst + (int64_t)hk * p.ksh, p.kst, lk, tid);
  vrows.init(p.v + (int64_t)k0 * p.vst + (int64_t)hk * p.vsh, p.vst, lk, tid);

  const PkLane<D> at(lane);
  auto sub_qk = [&](auto masked, const uint8_t* kt, int st, int j0, f32x16 (&s)[QPW]) __attribute__((always_inline)) {
    uint4 ka[KS];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) ka[ks] = at.row(kt, st, ks);
#pragma unroll
    for (int a = 0; a < QPW; ++a)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[a][r] = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int a = 0; a < QPW; ++a) s[a] = mma(E{}, ka[ks], qa[a][ks], s[a]);
    if constexpr (decltype(masked)::value) {
#pragma unroll
      for (int a = 0; a < QPW; ++a) {
        const int room = lim[a] - j0 - 4 * half;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[a][r] = 8 * (r / 4) + r % 4 <= room ? s[a][r] : -INFINITY;
      }
    }
  };
  bool unclean = false;  // V holds inf or NaN in tiles that some rows see only in part
  auto sub_pv = [&](auto masked, const uint8_t* vt, int st, f32x16 (&s)[QPW]) __attribute__((always_inline)) {
    uint4 va[2 * DB];
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) va[2 * db + ks] = at.col(vt, st, ks, db);
    if constexpr (decltype(masked)::value) {
      if (p.causal) unclean |= pk_clear_not_finite<E>(va);
    }
#pragma unroll
    for (int a = 0; a < QPW; ++a) {
      uint4 pb[2];
      auto weights = [&](float nm) __attribute__((always_inline)) {
        float w[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) w[r] = fexp2(fmaf(s[a][r], sl2, nm));
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) pb[ks] = pack_quad<E>(w + 8 * ks);
        float t[2] = {w[0], w[8]};
#pragma unroll
        for (int r = 1; r < 8; ++r) {
          t[0] += w[r];
          t[1] += w[8 + r];
        }
        return t[0] + t[1];
      };
      float ls = weights(-m[a]);
      if (__builtin_expect(__builtin_amdgcn_ballot_w64(!(ls <= kPkSumCap<E>)) != 0ull, 0)) {
        // A row's weights have grown past the cap (or these are its first keys): it moves its reference to (fp16:
        // below) its largest score here if that is higher. The block's other rows keep theirs, so that a row's
        // roundings depend on what it sees alone.
        const bool up = pair_max(ls <= kPkSumCap<E> ? 0.f : 1.f) > 0.f;
        float mx = s[a][0];
#pragma unroll
        for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[a][r]);
        mx = pair_max(mx);
        const float mn = up ? fmaxf(m[a], mx * sl2 - kPkBelow<E>) : m[a];
        const float alpha = fexp2(m[a] - mn);
        m[a] = mn;
        l[a] *= alpha;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[a][db][r] *= alpha;
        ls = weights(-mn);
      }
      l[a] += ls;
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int db = 0; db < DB; ++db) acc[a][db] = mma(E{}, va[2 * db + ks], pb[ks], acc[a][db]);
    }
  };

  if (ntk > 0) {
    krows.load(tk0, kt0);
    vrows.load(tk0, vt0);
    pk_tile_barrier();
    const int full = min(max(((last_key(row0) + 1) >> 6) - tk0, 0), ntk);  // tiles that every row sees whole
    pk_tiles(ntk, full, [&](auto masked, auto buf, int n) __attribute__((always_inline)) {
      constexpr int B = decltype(buf)::value;
      const uint8_t *kc = B ? kt1 : kt0, *vc = B ? vt1 : vt0;
      // Past the end the last tile again, into the buffer that no wave reads any more.
      krows.load(tk0 + min(n + 1, ntk - 1), B ? kt0 : kt1);
      vrows.load(tk0 + min(n + 1, ntk - 1), B ? vt0 : vt1);
      const int j0 = 64 * (tk0 + n);
      if (j0 <= lim_wave) {
        f32x16 s0[QPW], s1[QPW];
        sub_qk(masked, kc, 0, j0, s0);
        sub_qk(masked, kc, 1, j0 + 32, s1);
        sub_pv(masked, vc, 0, s0);
        sub_pv(masked, vc, 1, s1);
      }
      pk_tile_barrier();
    });
    if (__builtin_expect(unclean, 0)) {
      const int end = min(64 * (tk0 + ntk), min(lk, lim_wave + 1));
      for (int j = 64 * (tk0 + (full & ~1)); j < end; ++j) {  // pk_tiles masks from an even tile on
        const uint16_t* vr = p.v + (int64_t)(k0 + j) * p.vst + (int64_t)hk * p.vsh;
#pragma unroll
        for (int a = 0; a < QPW; ++a) pk_add_not_finite<E>(vr, half, j <= lim[a], acc[a]);
      }
    }
  }

  // o = O / l, lse = (m + log2 l) ln 2; a part keeps its o in fp32 and its log2 sum.
#pragma unroll
  for (int a = 0; a < QPW; ++a) {
    const float lt = pair_sum(l[a]);
    const float inv = lt == 0.f ? 0.f : 1.f / lt;  // no keys: o = 0; NaN stays NaN
    const int64_t t = pt.start + tok[a];
    if (p.split > 1) {
      if (!on[a]) continue;
      const int64_t at = ((int64_t)blockIdx.y * p.Tq + t) * p.H + head[a];
      if (half == 0) p.part_lse[at] = lt == 0.f ? -INFINITY : m[a] + flog2(lt);
      if (lt == 0.f) continue;  // a part without weight is not read
      float* dst = p.part + at * D + 4 * half;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<float4*>(dst + 32 * db + 8 * g) =
              make_float4(acc[a][db][4 * g] * inv, acc[a][db][4 * g + 1] * inv, acc[a][db][4 * g + 2] * inv,
                          acc[a][db][4 * g + 3] * inv);
      continue;
    }
    uint16_t* orow = p.o + t * p.ost + (int64_t)head[a] * p.osh;
#pragma unroll
    for (int db = 0; db < DB; ++db) {
      if (p.rest)
        pk_store_col<E, true>(orow + 32 * db, acc[a][db], inv, half, on[a], p.rest + (t * p.H + head[a]) * D + 32 * db);
      else
        pk_store_col<E>(orow + 32 * db, acc[a][db], inv, half, on[a]);
    }
    if (on[a] && half == 0 && p.lse) p.lse[t * p.H + head[a]] = lt == 0.f ? -INFINITY : (m[a] + flog2(lt)) * kDLn2;
  }
}

// Joins the parts of each row (token, head): D / 4 threads of four dims, parts in order.
template <typename E, int D>
__global__ __launch_bounds__(256) void packed_join_kernel(const PackedFwdParams p) {
  constexpr int LPR = D / 4;
  const int64_t row = (int64_t)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
  const int c = threadIdx.x % LPR;
  const int64_t total = (int64_t)p.Tq * p.H;
  if (row >= total) return;
  const int64_t t = row / p.H;
  const int head = (int)(row - t * p.H);
  if (p.skip_rows > 0) {
    const PackedTile pt = pk_token(p.cu_q, p.n, p.Tq, (int)t);
    if (pt.len * p.G <= p.skip_rows) return;
  }
  float mx = -INFINITY, lt = 0.f;
  bool nan = false;
  for (int i = 0; i < p.split; ++i) {
    const float x = p.part_lse[i * total + row];
    nan |= x != x;
    mx = fmaxf(mx, x);
  }
  if (nan) mx = NAN;
  float4 out = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int i = 0; i < p.split; ++i) {
    const float x = p.part_lse[i * total + row];
    if (x == -INFINITY) continue;
    const float f = fexp2(x - mx);
    const float4 y = reinterpret_cast<const float4*>(p.part + (i * total + row) * D)[c];
    lt += f;
    out.x = fmaf(y.x, f, out.x);
    out.y = fmaf(y.y, f, out.y);
    out.z = fmaf(y.z, f, out.z);
    out.w = fmaf(y.w, f, out.w);
  }
  const float inv = lt == 0.f ? 0.f : 1.f / lt;
  pk_store4<E>(p.o + t * p.ost + (int64_t)head * p.osh + 4 * c, p.rest ? p.rest + row * D + 4 * c : nullptr, out.x * inv,
               out.y * inv, out.z * inv, out.w * inv);
  if (c == 0 && p.lse) p.lse[row] = lt == 0.f ? -INFINITY : (mx + flog2(lt)) * kDLn2;
}

// What a call launches, from the sizes that the host knows.
// - Few-rows kernel (rows_attn_fwd.hip): where a sequence's rows are few on average and its keys many, the
//   sequences of at most kRowsMax rows are split over all workgroups there; the tile kernel skips them. Up to 1,024
//   sequences, since each of its workgroups scans them all: one query of 1,100 sequences of 600 keys, 8 heads of 64,
//   took 539 us there and takes 273 in tiles of 128 rows; 4,000 sequences, 4 heads, 1,906 and 436.
// - Tile kernel: rows in blocks of 128 (D = 64: or 256), and the keys of each tile cut into `split` parts
//   where the tiles alone leave workgroup slots (two per CU) empty.
struct FwdPlan {
  bool rows, tiles;
  int qpw, split;
  size_t rows_bytes, split_bytes;
};

FwdPlan packed_fwd_plan(int64_t n, int64_t Tq, int64_t Tk, int64_t Hq, int64_t Hk, int64_t D) {
  FwdPlan f = {};
  const int64_t G = Hq / Hk, rows = Tq * G, seqs = n > 0 ? n : 1, keys = Tk / seqs;
  f.rows = n <= 1024 && rows / seqs <= 128 && keys >= 512;
  f.tiles = !f.rows || rows > kRowsMax;
  // 256 rows per workgroup (each K and V operand read from LDS feeds two products) where sequences are
  // long and the tiles fill the chip twice; 128 rows keep three workgroups on a CU in place of two and
  // waste less of a sequence's last tile. Measured, 128 and 256 rows: 43,968 tokens 8.04 and 7.77 ms,
  // 4 x 1,374 tokens 42.7 and 49.3 us.
  f.qpw = D == 64 && rows / seqs >= 2048 && (rows / 256) * Hk >= 1024 ? 2 : 1;
  const int64_t wgs = (rows / (128 * f.qpw) + (rows / seqs < 128 ? n : n / 2) + 1) * Hk;
  int64_t split = f.rows && rows / seqs <= 16 ? 1 : 512 / (wgs > 0 ? wgs : 1);
  if (split > keys / 512) split = keys / 512;
  if (split > 16) split = 16;
  f.split = split > 1 ? (int)split : 1;
  f.rows_bytes = f.rows ? (rows_workspace(rows_tiles(false, n, Tq, G), Hk, D) + 255) / 256 * 256 : 0;
  f.split_bytes = f.tiles && f.split > 1 ? (size_t)f.split * Tq * Hq * (D + 1) * sizeof(float) : 0;
  return f;
}

inline int64_t fwd_grid(int64_t n, int64_t Tq, int64_t Hq, int64_t Hk, int qpw) {
  return (Tq * (Hq / Hk) / (128 * qpw) + n + 2) * Hk;
}
inline int64_t fwd_join_grid(int64_t Tq, int64_t Hq, int64_t D) { return (Tq * Hq * (D / 4) + 255) / 256; }

template <typename E, int D, int QPW>
int packed_fwd_launch(const PackedFwdParams& p, hipStream_t stream) {
  const dim3 grid((uint32_t)fwd_grid(p.n, p.Tq, p.H, p.Hk, QPW), (uint32_t)p.split);
  hipLaunchKernelGGL((packed_attn_fwd_kernel<E, D, QPW>), grid, dim3(256), 0, stream, p);
  GW_HIP_LAUNCH_CHECK("gw_packed_attn_fwd");
  if (p.split > 1) {
    hipLaunchKernelGGL((packed_join_kernel<E, D>), dim3((uint32_t)fwd_join_grid(p.Tq, p.H, D)), dim3(256), 0, stream, p);
    GW_HIP_LAUNCH_CHECK("gw_packed_attn_fwd (join)");
  }
  return GW_OK;
}

template <typename E>
int packed_fwd_dim(const PackedFwdParams& p, int64_t D, int qpw, hipStream_t stream) {
  if (D == 128) return packed_fwd_launch<E, 128, 1>(p, stream);
  return qpw == 2 ? packed_fwd_launch<E, 64, 2>(p, stream) : packed_fwd_launch<E, 64, 1>(p, stream);
}

}  // namespace
}  // namespace gw

extern "C" size_t gw_packed_attn_fwd_workspace_size(int64_t n, int64_t Tq, int64_t Tk, int64_t Hq, int64_t Hk, int64_t D) {
  if (n < 0 || Tq < 1 || Tk < 0 || Hk < 1 || Hq < Hk || D < 1) return 0;
  const gw::FwdPlan f = gw::packed_fwd_plan(n, Tq, Tk, Hq, Hk, D);
  return f.rows_bytes + f.split_bytes;
}

extern "C" int gw_packed_attn_fwd(int dtype, const void* q, const int64_t* q_strides, const void* k,
                                  const int64_t* k_strides, const void* v, const int64_t* v_strides,
                                  const int32_t* cu_q, const int32_t* cu_k, void* o, const int64_t* o_strides,
                                  void* o_rest, float* lse, int64_t n, int64_t Tq, int64_t Tk, int64_t Hq, int64_t Hk,
                                  int64_t D, int causal, float softmax_scale, void* workspace, size_t workspace_bytes,
                                  void* stream) {
  using namespace gw;
  clear_error();
  PackedArgs a = {dtype, n, Tq, Tk, Hq, Hk, D, softmax_scale};
  const int rc = pk_check_args(a);
  if (rc != GW_OK) return rc;
  if (Tq == 0) return GW_OK;
  GW_CHECK_ARG(q && o && cu_q && cu_k && q_strides && k_strides && v_strides && o_strides && (Tk == 0 || (k && v)),
               "a tensor is missing");
  GW_CHECK_ARG(pk_rows_ok(q, q_strides) && pk_rows_ok(k, k_strides) && pk_rows_ok(v, v_strides) &&
                   pk_rows_ok(o, o_strides) && aligned16(o_rest),
               "q, k, v and o need 16-byte aligned rows, with token strides in [0, 2^24)");
  PackedFwdParams p = {};
  p.q = static_cast<const uint16_t*>(q);
  p.k = static_cast<const uint16_t*>(k);
  p.v = static_cast<const uint16_t*>(v);
  p.o = static_cast<uint16_t*>(o);
  p.rest = static_cast<uint16_t*>(o_rest);
  p.lse = lse;
  p.cu_q = cu_q;
  p.cu_k = cu_k;
  p.n = (int)n;
  p.Tq = (int)Tq;
  p.Tk = (int)Tk;
  p.H = (int)Hq;
  p.Hk = (int)Hk;
  p.G = (int)(Hq / Hk);
  p.causal = causal != 0;
  p.qst = q_strides[0];
  p.qsh = q_strides[1];
  p.kst = k_strides[0];
  p.ksh = k_strides[1];
  p.vst = v_strides[0];
  p.vsh = v_strides[1];
  p.ost = o_strides[0];
  p.osh = o_strides[1];
  p.scale_log2 = softmax_scale * kDLog2e;
  const FwdPlan f = packed_fwd_plan(n, Tq, Tk, Hq, Hk, D);
  GW_CHECK_ARG(f.rows_bytes + f.split_bytes == 0 ||
                   (workspace && aligned16(workspace) && workspace_bytes >= f.rows_bytes + f.split_bytes),
               "workspace of %zu bytes, %zu are needed", workspace_bytes, f.rows_bytes + f.split_bytes);
  // All launches fit, or none is made.
  if (f.rows) {
    GW_CHECK_GRID(rows_grid(false, n, Tq, Hq / Hk, Hk, true), 256);
    GW_CHECK_GRID(rows_tiles(false, n, Tq, Hq / Hk) * Hk, 256);
  }
  if (f.tiles) GW_CHECK_GRID(fwd_grid(n, Tq, Hq, Hk, f.qpw), 256);
  if (f.tiles && f.split > 1) GW_CHECK_GRID(fwd_join_grid(Tq, Hq, D), 256);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (f.rows) {
    RowsParams r = {};
    r.q = p.q;
    r.k = p.k;
    r.v = p.v;
    r.o = p.o;
    r.rest = p.rest;
    r.lse = lse;
    r.cu_q = cu_q;
    r.cu_k = cu_k;
    r.n = p.n;
    r.Tq = p.Tq;
    r.Tk = p.Tk;
    r.H = p.H;
    r.Hk = p.Hk;
    r.G = p.G;
    r.causal = p.causal;
    r.split = 1;
    r.want = rows_want(Hk);
    r.qst = p.qst;
    r.qsh = p.qsh;
    r.ost = p.ost;
    r.osh = p.osh;
    r.kst = p.kst;
    r.ksh = p.ksh;
    r.vst = p.vst;
    r.vsh = p.vsh;
    r.scale_log2 = p.scale_log2;
    const int rr = rows_attn(dtype, (int)D, false, r, workspace, s);
    if (rr != GW_OK || !f.tiles) return rr;
    p.skip_rows = kRowsMax;
  }
  p.split = f.split;
  if (f.split > 1) {
    p.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + f.rows_bytes);
    p.part_lse = p.part + (int64_t)f.split * Tq * Hq * D;
  }
  return dtype == GW_DTYPE_BF16 ? packed_fwd_dim<BF16>(p, D, f.qpw, s) : packed_fwd_dim<FP16>(p, D, f.qpw, s);
}
