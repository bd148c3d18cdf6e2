// Backward of the attention over packed sequences (gfx950): dQ, dK, dV without atomics on the
// gradients, D = 64 or 128.
//
// With P the softmax weights (formed again from the forward's lse) and delta_i = o_i . do_i, from o as it
// was before its rounding (the forward keeps what the rounding left: where a row sees few keys, dP - delta
// nearly cancels, and a delta from the rounded o would double the error of dQ and dK; what the rounding of the
// forward's weights left in o, half a step of P|V| at most, stays in delta):
//   dV = P^T dO,  dP = dO V^T,  dS = P (dP - delta),  dQ = scale dS K,  dK = scale dS^T Q.
// Two passes, so that every gradient is summed by one workgroup in a fixed order: the dQ pass has the
// forward's shape (rows of a key head in registers, K and V tiles through LDS: three products per
// pair), the dK/dV pass keeps 32 keys per wave in registers and takes Q and dO tiles of every head of
// the group through LDS (four products per pair; the heads of a group are summed in its registers).
// Seven products in place of five, but no sum depends on timing. Products are transposed as in
// the forward, so P and dS never leave the registers; K^T, Q^T and dO^T operands are transposing
// reads of the same LDS tiles.
//
// P and dS enter their products in the inputs' 16-bit type (half a step of each entry). fp16 has few
// exponents for them: P is scaled by 2^14, dS by a power of two of the lane's row (dQ) or key (dK) that follows the
// largest entry as it comes (PkFit), so that an entry keeps all its bits down to 2^-23 of the largest and no
// row or key depends on what it does not meet. (One power per sequence from the largest |do| and |v|: a row with 2^12
// times the others' dO beside a key with 2^6 times the others' v left the dK of the keys behind it 5 times their bound
// off.) The powers are exact and taken out of the fp32 sums again.
//
// Bound as the forward is, by the matrix cores and the vector unit (smallest of four traced passes): six
// sequences of 3,013 to 4,795 tokens, 16 heads of 64 in bf16, dQ 554 us (1.01 PFLOP/s, matrix cores busy 60 % of the
// time), dK/dV 789 us (0.95, 52 %), the statistics 28 us; the same with heads of 128 dQ 1,028 us (1.1 PFLOP/s), dK/dV
// 1,672 (0.90). Causal, fp16, 16 heads over 4 of 128: 55 + 568 + 940 us. 96 causal sequences of 17 to 697 tokens, 16
// heads over 8 of 64: 26 + 55 + 81 us; the lists of tiles by falling work took 61 + 103 to 54 + 79.
//
// Rows behind a sequence's end add 0 to every gradient, and rows that see no key have P = 0.
#include <math.h>

#include "gw_packed.h"

namespace gw {
namespace {

struct PackedBwdParams {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  const uint16_t* o;
  const uint16_t* rest;  // [Tq][H][D] what the rounding of o left
  const uint16_t* dout;
  const float* lse;
  uint16_t* dq;
  uint16_t* dk;
  uint16_t* dv;
  float* nlse;        // [H][Tq] -lse / scale (fp16: + 14 / (scale log2 e)), -inf for a row without keys: the
                      // products' start of S - lse / scale
  float* ndelta;      // [H][Tq] -delta
  int2* order_q;      // tiles of the dQ and of the dK/dV pass by falling work, or null
  int2* order_k;
  int split_dq, split_dkv;  // parts at most that a workgroup's inner loop is cut into,
  int per_dq, per_dkv;      // one for each so many tiles of 64
  float* part_dq;     // cut rows: [part][Tq][H][D]
  float* part_dkv;    // cut rows: [part][dk, dv][Tk][Hk][D]
  const int32_t* cu_q;
  const int32_t* cu_k;
  int n, Tq, Tk, H, Hk, G, causal;
  int64_t qst, qsh, kst, ksh, vst, vsh, ost, osh, gst, gsh;
  int64_t dqst, dqsh, dkst, dksh, dvst, dvsh;
  float scale, scale_log2;
};

constexpr int kBwdTile = 128;  // rows of a dQ workgroup, keys of a dK/dV workgroup

// Workgroup slots per key head of the two passes.
__host__ __device__ inline int dq_slots(const PackedBwdParams& p) {
  return (int)((int64_t)p.Tq * p.G / kBwdTile) + p.n + 2;
}
__host__ __device__ inline int dkv_slots(const PackedBwdParams& p) { return p.Tk / kBwdTile + p.n + 2; }

// Parts of a loop over `work` tiles of 64.
__device__ __forceinline__ int pk_parts(int work, int split, int per) {
  return split > 1 ? min(split, max(1, (work + per - 1) / per)) : 1;
}
// Tiles of 64 keys that block x (kBwdTile rows) of a sequence of len queries and lk keys meets.
__device__ __forceinline__ int dq_work(const PackedBwdParams& p, int len, int lk, int x) {
  const int last = (min((x + 1) * kBwdTile, len * p.G) - 1) / p.G;
  const int keys = p.causal ? min(last + lk - len, lk - 1) + 1 : lk;
  return keys > 0 ? (keys + 63) >> 6 : 0;
}
// First tile of 64 queries that meets block x (kBwdTile keys) of a sequence of len keys and lq queries, and how
// many tiles do, those of all heads of the group.
__device__ __forceinline__ int dkv_first(const PackedBwdParams& p, int len, int lq, int x) {
  return p.causal ? max(0, x * kBwdTile - (len - lq)) >> 6 : 0;
}
__device__ __forceinline__ int dkv_work(const PackedBwdParams& p, int len, int lq, int x) {
  return max(0, ((lq + 63) >> 6) - dkv_first(p, len, lq, x)) * p.G;  // fits: the host bounds Tq * H
}

// fp16: P enters its product times 2^14.
template <typename E>
constexpr float kPScale = __is_same(E, FP16) ? 14.f : 0.f;

// fp16: dS of a lane's row or key enters its product times 2^e. An entry that would pass 2^15 lowers e to where the
// largest of the step lies in [2^9, 2^10), and the lane's sums follow (lanes l and l ^ 32 hold the same row or
// key and sum into each other's accumulators: e is the same in both). The start is above what any entry but 0 allows
// (2^60 times the smallest product of two fp16 values, 2^-48), and within fp32 for the largest, 2^40. inf and
// NaN leave e as it is.
constexpr int kFitStart = 60;
struct PkFit {
  int e = kFitStart;
  // ds: all entries times 2^e of which none has entered its product yet. The power that was taken out, 2^-x
  // (x = 0 nearly always).
  template <int N, int DB>
  __device__ __forceinline__ int fit(float (&ds)[N], f32x16 (&acc)[DB]) {
    float mx = fabsf(ds[0]);
#pragma unroll
    for (int i = 1; i < N; ++i) mx = fmaxf(mx, fabsf(ds[i]));
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(mx > 32768.f) == 0ull, 1)) return 0;
    mx = pair_max(mx);
    int x = 0;
    if (mx > 32768.f && mx < INFINITY) {
      (void)frexpf(mx, &x);  // mx < 2^x
      x -= 10;
    }
    const float f = ldexpf(1.f, -x);
#pragma unroll
    for (int i = 0; i < N; ++i) ds[i] *= f;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[db][i] *= f;
    e -= x;
    return x;
  }
};

// Statistics of 256 / (D / 8) rows at a time: D / 8 lanes per (token, head) row.
constexpr int kStatTokens = 16;

// Workgroups 0 and 1 form the lists of the two passes' tiles, the others take query rows.
template <typename E, int D>
__global__ __launch_bounds__(256) void packed_bwd_stats_kernel(const PackedBwdParams p) {
  constexpr int LPR = D / 8;
  __shared__ uint32_t top[kPkClasses + 1];
  if (blockIdx.x == 0) {
    if (p.order_q) pk_order<false>(p.cu_q, p.Tq, p.cu_k, p.Tk, p.n, p.G, kBwdTile, p.causal, dq_slots(p), p.order_q, top,
                                   [&](int work) { return pk_parts(work, p.split_dq, p.per_dq); });
    return;
  }
  if (blockIdx.x == 1) {
    if (p.order_k) pk_order<true>(p.cu_k, p.Tk, p.cu_q, p.Tq, p.n, 1, kBwdTile, p.causal, dkv_slots(p), p.order_k, top,
                                  [&](int work) { return pk_parts(work * p.G, p.split_dkv, p.per_dkv); });
    return;
  }
  const PackedTile pt = pk_find_tile(p.cu_q, p.n, p.Tq, 1, kStatTokens, blockIdx.x - 2);
  const int t0 = pt.tile * kStatTokens;
  if (t0 >= pt.len) return;
  const int rows = min(kStatTokens, pt.len - t0) * p.H;
  const int li = threadIdx.x % LPR;
  for (int r = threadIdx.x / LPR; r < rows; r += 256 / LPR) {
    const int t = pt.start + t0 + r / p.H, h = r % p.H;
    float a[8], b[8], c[8];
    unpack8<E>(*reinterpret_cast<const uint4*>(p.o + (int64_t)t * p.ost + (int64_t)h * p.osh + li * 8), a);
    unpack8<E>(*reinterpret_cast<const uint4*>(p.rest + ((int64_t)t * p.H + h) * D + li * 8), c);
    unpack8<E>(*reinterpret_cast<const uint4*>(p.dout + (int64_t)t * p.gst + (int64_t)h * p.gsh + li * 8), b);
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s = fmaf(a[i] + c[i], b[i], s);
    s = group_sum<LPR>(s);
    if (li == 0) {
      const float l = p.lse[(int64_t)t * p.H + h];
      const int64_t at = (int64_t)h * p.Tq + t;
      p.nlse[at] = l == -INFINITY ? -INFINITY : (kPScale<E> - l * kDLog2e) / p.scale_log2;
      p.ndelta[at] = -s;
    }
  }
}

// The same column in fp32.
__device__ __forceinline__ void pk_store_part(float* row, const f32x16& acc, float f, int half, bool on) {
  if (!on) return;
#pragma unroll
  for (int g = 0; g < 4; ++g)
    *reinterpret_cast<float4*>(row + 8 * g + 4 * half) =
        make_float4(acc[4 * g] * f, acc[4 * g + 1] * f, acc[4 * g + 2] * f, acc[4 * g + 3] * f);
}

// ---------------------------------------------------------------------------------------
// dQ: the forward's decomposition.
// ---------------------------------------------------------------------------------------
template <typename E, int D>
__global__ __launch_bounds__(256, D == 64 ? 3 : 2) void packed_bwd_dq_kernel(const PackedBwdParams p) {
  constexpr int KS = D / 16, DB = D / 32, BM = kBwdTile;
  constexpr int kTileBytes = 64 * 2 * D;
  constexpr bool kFp16 = __is_same(E, FP16);
  __shared__ __align__(16) uint8_t kt0[kTileBytes], kt1[kTileBytes], vt0[kTileBytes], vt1[kTileBytes];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, half = lane >> 5;
  const int hk = blockIdx.x % p.Hk, part = blockIdx.x / p.Hk % p.split_dq;
  const PackedTile pt = pk_tile(p.order_q, p.cu_q, p.n, p.Tq, p.G, BM, blockIdx.x / p.Hk / p.split_dq);
  const int rows = pt.len * p.G;
  const int ntile = (rows + BM - 1) / BM;
  if (pt.tile < 0 || pt.tile >= ntile) return;
  const int row0 = (p.causal ? ntile - 1 - pt.tile : pt.tile) * BM;
  int k0, lk;
  pk_other(p.cu_k, p.n, p.Tk, pt.seq, k0, lk);
  const int all = dq_work(p, pt.len, lk, row0 / BM), parts = pk_parts(all, p.split_dq, p.per_dq);
  if (part >= parts) return;
  const int shift = lk - pt.len;
  const float sl2 = p.scale_log2;

  const int base = row0 + wave * 32;
  const bool on = base + col < rows;
  const int row = min(base + col, rows - 1);
  const int tok = row / p.G, head = hk * p.G + (row - tok * p.G);
  const int lim = p.causal ? min(tok + shift, lk - 1) : lk - 1;
  const int64_t t = pt.start + tok;
  uint4 qa[KS], ga[KS];
  {
    const uint16_t* qr = p.q + t * p.qst + (int64_t)head * p.qsh + half * 8;
    const uint16_t* gr = p.dout + t * p.gst + (int64_t)head * p.gsh + half * 8;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      qa[ks] = *reinterpret_cast<const uint4*>(qr + ks * 16);
      ga[ks] = *reinterpret_cast<const uint4*>(gr + ks * 16);
    }
  }
  PkFit fit;
  const int64_t srow = (int64_t)head * p.Tq + t;
  float nlse = p.nlse[srow] * sl2;  // fp16: p 2^e = 2^(s - lse + e)
  if (kFp16) nlse += (float)kFitStart - kPScale<E>;
  // dP - delta: in bf16 at D = 128 delta is where the products start, in a register block of its own; at D = 64,
  // where three waves share a SIMD's registers, it is added afterwards (with the block 124 bytes of
  // scratch a lane and half as much time again on 6 sequences of 3,013 to 4,795 tokens), and so it is in fp16 (4 % more
  // with the block).
  constexpr bool kAddDelta = D == 64 || kFp16;
  const float ndelta = p.ndelta[srow];
  f32x16 dp0;
#pragma unroll
  for (int r = 0; r < 16; ++r) dp0[r] = kAddDelta ? 0.f : ndelta;
  auto last_key = [&](int r) { return p.causal ? min(min(r, rows - 1) / p.G + shift, lk - 1) : lk - 1; };
  const int lim_wave = base < rows ? last_key(base + 31) : -1;
  // This part's tiles of 64 keys.
  const int per = (all + parts - 1) / parts;
  const int tk0 = min(part * per, all), ntk = min(per, all - tk0);

  f32x16 acc[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[db][r] = 0.f;

  PkRows<D, 256> krows, vrows;
  krows.init(p.k + (int64_t)k0 * p.kst + (int64_t)hk * p.ksh, p.kst, lk, tid);
  vrows.init(p.v + (int64_t)k0 * p.vst + (int64_t)hk * p.vsh, p.vst, lk, tid);

  const PkLane<D> at(lane);
  struct Rows {
    uint4 k[KS], v[KS];
  };
  auto fetch = [&](const uint8_t* kt, const uint8_t* vt, int st, Rows& r) __attribute__((always_inline)) {
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      r.k[ks] = at.row(kt, st, ks);
      r.v[ks] = at.row(vt, st, ks);
    }
  };
  // Three steps: the products S and dP while the column operands of K are read; dS; the product dQ while
  // `next` reads the next sub-tile's row operands. Kept in this order at D = 64, where that fits three
  // waves per SIMD (with two the six sequences above took 7 % longer; left to the compiler, two waves as long as three).
  auto step = []() __attribute__((always_inline)) {
    if constexpr (D == 64) __builtin_amdgcn_sched_barrier(0);
  };
  bool unclean = false;  // K holds inf or NaN in tiles that some rows see only in part
  auto sub = [&](auto masked, const uint8_t* kt, int st, int j0, Rows& r, auto&& next) __attribute__((always_inline)) {
    // fp16 at D = 128: read behind the fit, whose branch they would have to outlive (100 bytes of scratch a lane and
    // 20 % more time).
    constexpr bool kLate = kFp16 && D == 128;
    uint4 kc[2 * DB];
    auto columns = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) kc[2 * db + ks] = at.col(kt, st, ks, db);
    };
    auto clear = [&]() __attribute__((always_inline)) {
      if (decltype(masked)::value && p.causal) unclean |= pk_clear_not_finite<E>(kc);
    };
    if constexpr (!kLate) columns();
    f32x16 s, dp = dp0;
#pragma unroll
    for (int x = 0; x < 16; ++x) s[x] = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      s = mma(E{}, r.k[ks], qa[ks], s);
      dp = mma(E{}, r.v[ks], ga[ks], dp);
    }
    step();
    float ds[16];
#pragma unroll
    for (int x = 0; x < 16; ++x) ds[x] = fexp2(fmaf(s[x], sl2, nlse)) * (kAddDelta ? dp[x] + ndelta : dp[x]);
    if constexpr (decltype(masked)::value) {
      const int room = lim - j0 - 4 * half;
#pragma unroll
      for (int x = 0; x < 16; ++x) ds[x] = 8 * (x / 4) + x % 4 <= room ? ds[x] : 0.f;
    }
    if constexpr (!kLate) clear();
    if constexpr (kFp16) nlse -= (float)fit.fit(ds, acc);
    const uint4 b[2] = {pack_quad<E>(ds), pack_quad<E>(ds + 8)};
    if constexpr (kLate) {
      columns();
      clear();
    }
    step();
    next();
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int db = 0; db < DB; ++db) acc[db] = mma(E{}, kc[2 * db + ks], b[ks], acc[db]);
    step();
  };

  if (ntk > 0) {
    krows.load(tk0, kt0);
    vrows.load(tk0, vt0);
    pk_tile_barrier();
    const int full = min(max(((last_key(row0) + 1) >> 6) - tk0, 0), ntk);  // tiles that every row sees whole
    pk_tiles(ntk, full, [&](auto masked, auto buf, int n) __attribute__((always_inline)) {
      constexpr int B = decltype(buf)::value;
      const uint8_t *kc = B ? kt1 : kt0, *vc = B ? vt1 : vt0;
      krows.load(tk0 + min(n + 1, ntk - 1), B ? kt0 : kt1);
      vrows.load(tk0 + min(n + 1, ntk - 1), B ? vt0 : vt1);
      const int j0 = 64 * (tk0 + n);
      if (j0 <= lim_wave) {
        Rows r0, r1;
        fetch(kc, vc, 0, r0);
        sub(masked, kc, 0, j0, r0, [&]() __attribute__((always_inline)) { fetch(kc, vc, 1, r1); });
        sub(masked, kc, 1, j0 + 32, r1, []() {});
      }
      pk_tile_barrier();
    });
    if (__builtin_expect(unclean, 0)) {
      const int end = min(64 * (tk0 + ntk), min(lk, lim_wave + 1));
      for (int j = 64 * (tk0 + (full & ~1)); j < end; ++j)  // pk_tiles masks from an even tile on
        pk_add_not_finite<E, true>(p.k + (int64_t)(k0 + j) * p.kst + (int64_t)hk * p.ksh, half, j <= lim, acc);
    }
  }
  // The weight of a row that sees one key is 1 whatever its score: no gradient, where rounding would
  // leave dP - delta a little off 0.
  const float unscale = lim == 0 ? 0.f : kFp16 ? fminf(ldexpf(p.scale, -fit.e), 3e38f) : p.scale;
  if (parts > 1) {
    float* dst = p.part_dq + (((int64_t)part * p.Tq + t) * p.H + head) * D;
#pragma unroll
    for (int db = 0; db < DB; ++db) pk_store_part(dst + 32 * db, acc[db], unscale, half, on);
    return;
  }
  uint16_t* dst = p.dq + t * p.dqst + (int64_t)head * p.dqsh;
#pragma unroll
  for (int db = 0; db < DB; ++db) pk_store_col<E>(dst + 32 * db, acc[db], unscale, half, on);
}

// ---------------------------------------------------------------------------------------
// dK and dV, D = 64: 4 waves x 32 keys of one key head; tiles of 64 query tokens of each head of the group. A
// lane holds one key and 16 queries of S = Q K^T and dP = dO V^T, whose products start at -lse / scale
// and -delta. (64 keys per wave, one wave per SIMD, read half as much from LDS and took 20 % longer: the
// products and the weights of one wave do not overlap enough.)
// ---------------------------------------------------------------------------------------
template <typename E>
__global__ __launch_bounds__(256, 2) void packed_bwd_dkv_kernel(const PackedBwdParams p) {
  constexpr int D = 64, KS = D / 16, DB = D / 32, BN = kBwdTile;
  constexpr int kTileBytes = 64 * 2 * D;
  constexpr bool kFp16 = __is_same(E, FP16);
  __shared__ __align__(16) uint8_t qt0[kTileBytes], qt1[kTileBytes], gt0[kTileBytes], gt1[kTileBytes];
  __shared__ __align__(16) float nl0[64], nl1[64], nd0[64], nd1[64];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, half = lane >> 5;
  const int hk = blockIdx.x % p.Hk, part = blockIdx.x / p.Hk % p.split_dkv;
  const PackedTile pt = pk_tile(p.order_k, p.cu_k, p.n, p.Tk, 1, BN, blockIdx.x / p.Hk / p.split_dkv);
  const int key0 = pt.tile * BN;
  if (key0 < 0 || key0 >= pt.len) return;
  int q0, lq;
  pk_other(p.cu_q, p.n, p.Tq, pt.seq, q0, lq);
  const int all = dkv_work(p, pt.len, lq, pt.tile), parts = pk_parts(all, p.split_dkv, p.per_dkv);
  if (part >= parts) return;
  const int shift = pt.len - lq;  // causal: key j is seen by tokens i >= j - shift
  const float sl2 = p.scale_log2;
  const int wkey = key0 + wave * 32;

  const int key = wkey + col;
  const bool on = key < pt.len;

  // Stationary operands: K and V rows of this lane's key.
  uint4 kb[KS], vb[KS];
  {
    const int64_t t = pt.start + min(key, pt.len - 1);
    const uint16_t* kr = p.k + t * p.kst + (int64_t)hk * p.ksh + half * 8;
    const uint16_t* vr = p.v + t * p.vst + (int64_t)hk * p.vsh + half * 8;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      kb[ks] = *reinterpret_cast<const uint4*>(kr + ks * 16);
      vb[ks] = *reinterpret_cast<const uint4*>(vr + ks * 16);
    }
  }
  // fp16: dS = P (dP - delta) 2^e, P 2^14.
  PkFit fit;
  float dscale = ldexpf(1.f, kFitStart - 14);

  f32x16 ak[DB], av[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) ak[db][r] = av[db][r] = 0.f;

  const int first = dkv_first(p, pt.len, lq, pt.tile);  // first tile with a query that sees a key
  const int ntq = (lq + 63) >> 6;
  const int per = ntq > first ? ntq - first : 0;
  // This part's tiles, head by head of the group.
  const int share = (all + parts - 1) / parts, t0 = min(part * share, all), total = min(share, all - t0);

  PkRows<D, 256> qrows, grows;
  const uint16_t* qbase = p.q + (int64_t)q0 * p.qst + (int64_t)hk * p.G * p.qsh;
  const uint16_t* gbase = p.dout + (int64_t)q0 * p.gst + (int64_t)hk * p.G * p.gsh;
  const int64_t sbase = (int64_t)hk * p.G * p.Tq + q0;
  qrows.init(qbase, p.qst, lq, tid);
  grows.init(gbase, p.gst, lq, tid);
  // The tile that is loaded next: head of the group and tile of its queries.
  int ld_h = per > 0 ? t0 / per : 0;
  int ld_t = first + t0 - ld_h * per;
  auto load = [&](uint8_t* qd, uint8_t* gd, float* ld, float* dd) __attribute__((always_inline)) {
    qrows.base = uniform_ptr(reinterpret_cast<const char*>(qbase + (int64_t)ld_h * p.qsh));
    grows.base = uniform_ptr(reinterpret_cast<const char*>(gbase + (int64_t)ld_h * p.gsh));
    qrows.template load<true>(ld_t, qd);
    grows.load(ld_t, gd);
    // 64 lse and 64 delta, 4 bytes a lane (their start is only 4-byte aligned): waves 0 and 1. A tile's rows behind
    // the last query repeat its Q and lse, and have dO = 0 and delta = 0: they add 0 to every key, and their
    // weights are finite where the last query's are (zeros of Q would make NaN with a key's inf, whose weights are 0
    // where it scores -inf).
    const int64_t sat = sbase + (int64_t)ld_h * p.Tq + ld_t * 64;
    const int64_t left = (int64_t)(lq - ld_t * 64) * 4;
    const int last = (int)min(left, (int64_t)256) - 4;
    if (wave == 0)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(pk_rsrc(reinterpret_cast<const char*>(p.nlse + sat), left),
                                               (__attribute__((address_space(3))) void*)ld, 4, min(lane * 4, last), 0, 0, 0);
    if (wave == 1)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(pk_rsrc(reinterpret_cast<const char*>(p.ndelta + sat), left),
                                               (__attribute__((address_space(3))) void*)dd, 4, lane * 4, 0, 0, 0);
    if (++ld_t == ntq) {
      ld_t = first;
      if (++ld_h == p.G) ld_h = p.G - 1;  // past the end: a tile again that no wave uses
    }
  };

  const PkLane<D> at(lane);
  bool unclean = false;  // dO or Q holds inf or NaN in tiles that see some keys only in part
  // A sub-tile of 32 queries. Entry x of this lane is query i0 + 8 (x / 4) + 4 half + x % 4.
  auto sub = [&](auto masked, const uint8_t* qt, const uint8_t* gt, const float* nl, const float* nd, int st, int i0)
                 __attribute__((always_inline)) {
    f32x16 s, dp;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const float4 x = *reinterpret_cast<const float4*>(nl + 32 * st + 8 * g + 4 * half);
      const float4 y = *reinterpret_cast<const float4*>(nd + 32 * st + 8 * g + 4 * half);
      s[4 * g] = x.x;
      s[4 * g + 1] = x.y;
      s[4 * g + 2] = x.z;
      s[4 * g + 3] = x.w;
      dp[4 * g] = y.x;
      dp[4 * g + 1] = y.y;
      dp[4 * g + 2] = y.z;
      dp[4 * g + 3] = y.w;
    }
    // Operands of the products in the order of their use, read PRE products ahead; the scheduling barriers
    // keep the compiler from reading them all at once, for which there are no registers (4 % less time on the
    // six sequences above).
    constexpr int PRE = 2;
    auto row = [&](int i) __attribute__((always_inline)) { return i < KS ? at.row(qt, st, i) : at.row(gt, st, i - KS); };
    // Columns for each 16 queries and 32 dims: of dO, then of Q.
    auto column = [&](int i) __attribute__((always_inline)) {
      return at.col(i % 2 ? qt : gt, st, i / 2 / DB, i / 2 % DB);
    };
    uint4 a[PRE], c[PRE];
#pragma unroll
    for (int i = 0; i < PRE; ++i) a[i] = row(i);
#pragma unroll
    for (int i = 0; i < 2 * KS; ++i) {
      if (i < KS)
        s = mma(E{}, a[i % PRE], kb[i % KS], s);
      else
        dp = mma(E{}, a[i % PRE], vb[i % KS], dp);
      if (i + PRE < 2 * KS)
        a[i % PRE] = row(i + PRE);
      else
        c[i + PRE - 2 * KS] = column(i + PRE - 2 * KS);
      __builtin_amdgcn_sched_barrier(0);
    }
    float w[16], ds[16];
#pragma unroll
    for (int x = 0; x < 16; ++x) w[x] = fexp2(s[x] * sl2);
#pragma unroll
    for (int x = 0; x < 16; ++x) ds[x] = kFp16 ? w[x] * dscale * dp[x] : w[x] * dp[x];
    if constexpr (decltype(masked)::value) {
      const int need = key - shift - i0 - 4 * half;
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        const bool sees = 8 * (x / 4) + x % 4 >= need;
        w[x] = sees ? w[x] : 0.f;
        ds[x] = sees ? ds[x] : 0.f;
      }
      if (wkey == 0 && i0 <= -shift && -shift < i0 + 32) {  // the row that sees the first key only has dS = 0
#pragma unroll
        for (int x = 0; x < 16; ++x) ds[x] = 8 * (x / 4) + x % 4 + 4 * half == -shift - i0 ? 0.f : ds[x];
      }
    }
    if constexpr (kFp16) dscale = ldexpf(dscale, -fit.fit(ds, ak));
    const uint4 pb[2] = {pack_quad<E>(w), pack_quad<E>(w + 8)}, sb[2] = {pack_quad<E>(ds), pack_quad<E>(ds + 8)};
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 4 * DB; ++i) {
      const int ks = i / 2 / DB, db = i / 2 % DB;
      uint4 q[1] = {c[i % PRE]};
      if constexpr (decltype(masked)::value) {
        unclean |= pk_clear_not_finite<E>(q);
      }
      if (i % 2 == 0)
        av[db] = mma(E{}, q[0], pb[ks], av[db]);
      else
        ak[db] = mma(E{}, q[0], sb[ks], ak[db]);
      if (i + PRE < 4 * DB) c[i % PRE] = column(i + PRE);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  if (total > 0) {
    load(qt0, gt0, nl0, nd0);
    pk_tile_barrier();
    int cur = first + t0 % per;  // the tile that is computed
    // Queries of tiles from `full` on see every key of the workgroup's block.
    const int full = p.causal ? (key0 + BN - 1 - shift + 63) >> 6 : first;
    auto tile = [&](auto buf) __attribute__((always_inline)) {
      constexpr int B = decltype(buf)::value;
      const uint8_t *qc = B ? qt1 : qt0, *gc = B ? gt1 : gt0;
      const float *lc = B ? nl1 : nl0, *dc = B ? nd1 : nd0;
      load(B ? qt0 : qt1, B ? gt0 : gt1, B ? nl0 : nl1, B ? nd0 : nd1);
      if (wkey < pt.len) {
        if (cur >= full) {
          sub(PkInt<0>{}, qc, gc, lc, dc, 0, 64 * cur);
          sub(PkInt<0>{}, qc, gc, lc, dc, 1, 64 * cur + 32);
        } else if (64 * cur + 63 + shift >= wkey) {
          sub(PkInt<1>{}, qc, gc, lc, dc, 0, 64 * cur);
          sub(PkInt<1>{}, qc, gc, lc, dc, 1, 64 * cur + 32);
        }
      }
      if (++cur == ntq) cur = first;
      pk_tile_barrier();
    };
    int n = 0;
#pragma unroll 1
    for (; n + 1 < total; n += 2) {
      tile(PkInt<0>{});
      tile(PkInt<1>{});
    }
    if (n < total) tile(PkInt<0>{});
    if (__builtin_expect(unclean, 0)) {
      for (int x = t0; x < t0 + total; ++x) {
        const int h = x / per, i0 = 64 * (first + x % per);
        for (int i = i0; i < min(i0 + 64, min(64 * full, lq)); ++i) {
          pk_add_not_finite<E>(gbase + (int64_t)i * p.gst + (int64_t)h * p.gsh, half, key <= i + shift, av);
          pk_add_not_finite<E, true>(qbase + (int64_t)i * p.qst + (int64_t)h * p.qsh, half, key <= i + shift, ak);
        }
      }
    }
  }
  // Rows of a sequence of one key all have dS = 0.
  const float fk = pt.len == 1 ? 0.f : kFp16 ? fminf(ldexpf(p.scale, -fit.e), 3e38f) : p.scale;
  const float fv = kFp16 ? ldexpf(1.f, -14) : 1.f;
  const int64_t t = pt.start + (on ? key : 0);
  if (parts > 1) {
    const int64_t step = (int64_t)p.Tk * p.Hk * D;
    float* dst = p.part_dkv + 2 * part * step + (t * p.Hk + hk) * D;
#pragma unroll
    for (int db = 0; db < DB; ++db) {
      pk_store_part(dst + 32 * db, ak[db], fk, half, on);
      pk_store_part(dst + step + 32 * db, av[db], fv, half, on);
    }
    return;
  }
  uint16_t* dkr = p.dk + t * p.dkst + (int64_t)hk * p.dksh;
  uint16_t* dvr = p.dv + t * p.dvst + (int64_t)hk * p.dvsh;
#pragma unroll
  for (int db = 0; db < DB; ++db) {
    pk_store_col<E>(dkr + 32 * db, ak[db], fk, half, on);
    pk_store_col<E>(dvr + 32 * db, av[db], fv, half, on);
  }
}

// The same for D = 128, where one wave cannot hold K, V, dK and dV and leave room for another on its SIMD: waves
// w and w + 4 share 32 keys. The first holds K and dV: S, P and P^T dO. The second holds V and dK: dP, dS
// and dS^T Q, with P from the first through LDS in fp32. A barrier in the middle of a tile hands P over; the
// two meet on one SIMD, where the products of one run beside the weights of the other. Six sequences of 3,013 to
// 4,795 tokens, 16 heads, bf16: 1,660 to 1,670 us, 2,062 with one wave per SIMD that holds all four, and longer still
// with dV and dK in a pass each. 12 bytes of scratch a lane, outside the loop.
template <typename E>
__global__ __launch_bounds__(512, 2) void packed_bwd_dkv_pair_kernel(const PackedBwdParams p) {
  constexpr int D = 128, KS = D / 16, DB = D / 32, BN = kBwdTile;
  constexpr int kTileBytes = 64 * 2 * D;
  constexpr bool kFp16 = __is_same(E, FP16);
  __shared__ __align__(16) uint8_t qt0[kTileBytes], qt1[kTileBytes], gt0[kTileBytes], gt1[kTileBytes];
  __shared__ __align__(16) float nl0[64], nl1[64], nd0[64], nd1[64];
  __shared__ __align__(16) float4 weights[4][2][4][64];  // [keys][sub-tile][quad][lane]

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), kw = wave & 3;
  const int col = lane & 31, half = lane >> 5;
  const int hk = blockIdx.x % p.Hk, part = blockIdx.x / p.Hk % p.split_dkv;
  const PackedTile pt = pk_tile(p.order_k, p.cu_k, p.n, p.Tk, 1, BN, blockIdx.x / p.Hk / p.split_dkv);
  const int key0 = pt.tile * BN;
  if (key0 < 0 || key0 >= pt.len) return;
  int q0, lq;
  pk_other(p.cu_q, p.n, p.Tq, pt.seq, q0, lq);
  const int all = dkv_work(p, pt.len, lq, pt.tile), parts = pk_parts(all, p.split_dkv, p.per_dkv);
  if (part >= parts) return;
  const int shift = pt.len - lq;  // causal: key j is seen by tokens i >= j - shift
  const float sl2 = p.scale_log2;
  const int wkey = key0 + kw * 32;
  const int key = wkey + col;
  const bool on = key < pt.len;

  const int first = dkv_first(p, pt.len, lq, pt.tile);  // first tile with a query that sees a key
  const int ntq = (lq + 63) >> 6;
  const int per = ntq > first ? ntq - first : 0;
  // This part's tiles, head by head of the group.
  const int share = (all + parts - 1) / parts, t0 = min(part * share, all), total = min(share, all - t0);

  PkRows<D, 512> qrows, grows;
  const uint16_t* qbase = p.q + (int64_t)q0 * p.qst + (int64_t)hk * p.G * p.qsh;
  const uint16_t* gbase = p.dout + (int64_t)q0 * p.gst + (int64_t)hk * p.G * p.gsh;
  const int64_t sbase = (int64_t)hk * p.G * p.Tq + q0;
  qrows.init(qbase, p.qst, lq, tid);
  grows.init(gbase, p.gst, lq, tid);
  int ld_h = per > 0 ? t0 / per : 0;
  int ld_t = first + t0 - ld_h * per;
  auto load = [&](uint8_t* qd, uint8_t* gd, float* ld, float* dd) __attribute__((always_inline)) {
    qrows.base = uniform_ptr(reinterpret_cast<const char*>(qbase + (int64_t)ld_h * p.qsh));
    grows.base = uniform_ptr(reinterpret_cast<const char*>(gbase + (int64_t)ld_h * p.gsh));
    qrows.template load<true>(ld_t, qd);
    grows.load(ld_t, gd);
    const int64_t sat = sbase + (int64_t)ld_h * p.Tq + ld_t * 64;
    const int64_t left = (int64_t)(lq - ld_t * 64) * 4;
    const int last = (int)min(left, (int64_t)256) - 4;
    if (wave == 0)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(pk_rsrc(reinterpret_cast<const char*>(p.nlse + sat), left),
                                               (__attribute__((address_space(3))) void*)ld, 4, min(lane * 4, last), 0, 0, 0);
    if (wave == 4)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(pk_rsrc(reinterpret_cast<const char*>(p.ndelta + sat), left),
                                               (__attribute__((address_space(3))) void*)dd, 4, lane * 4, 0, 0, 0);
    if (++ld_t == ntq) {
      ld_t = first;
      if (++ld_h == p.G) ld_h = p.G - 1;
    }
  };
  const PkLane<D> at(lane);

  auto role = [&](auto second) __attribute__((always_inline)) {
    constexpr bool B = decltype(second)::value;
    uint4 st[KS];  // K or V rows of this lane's key
    {
      const int64_t t = pt.start + min(key, pt.len - 1);
      const uint16_t* r = (B ? p.v + t * p.vst + (int64_t)hk * p.vsh : p.k + t * p.kst + (int64_t)hk * p.ksh) + half * 8;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) st[ks] = *reinterpret_cast<const uint4*>(r + ks * 16);
    }
    f32x16 acc[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[db][r] = 0.f;
    bool unclean = false;  // the columns (dO, Q) hold inf or NaN in tiles that see some keys only in part
    PkFit fit;  // fp16: dS = P (dP - delta) 2^e, P 2^14
    float dscale = ldexpf(1.f, kFitStart - 14);

    // A tile of 64 queries: rows of rt against the stationary rows, columns of ct into acc.
    auto whole = [&](auto masked, const uint8_t* rt, const uint8_t* ct, const float* start, int i0)
                     __attribute__((always_inline)) {
      constexpr int PRE = 3;
      f32x16 x[2];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const float4 y = *reinterpret_cast<const float4*>(start + 32 * u + 8 * g + 4 * half);
          x[u][4 * g] = y.x;
          x[u][4 * g + 1] = y.y;
          x[u][4 * g + 2] = y.z;
          x[u][4 * g + 3] = y.w;
        }
      uint4 a[PRE], c[PRE];
      auto column = [&](int i) __attribute__((always_inline)) {  // sub-tile, 16 queries, 32 dims
        return at.col(ct, i / (2 * DB), i / DB % 2, i % DB);
      };
#pragma unroll
      for (int i = 0; i < PRE; ++i) a[i] = at.row(rt, 0, i);
#pragma unroll
      for (int i = 0; i < 2 * KS; ++i) {
        x[i / KS] = mma(E{}, a[i % PRE], st[i % KS], x[i / KS]);
        if (i + PRE < 2 * KS)
          a[i % PRE] = at.row(rt, (i + PRE) / KS, (i + PRE) % KS);
        else
          c[i + PRE - 2 * KS] = column(i + PRE - 2 * KS);
        __builtin_amdgcn_sched_barrier(0);
      }
      uint4 b[2][2];
      auto sees = [&](int u, int i, float y) __attribute__((always_inline)) {
        if constexpr (decltype(masked)::value) return 8 * (i / 4) + i % 4 >= key - shift - i0 - 32 * u - 4 * half ? y : 0.f;
        return y;
      };
      if constexpr (!B) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float w[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) w[i] = sees(u, i, fexp2(x[u][i] * sl2));
#pragma unroll
          for (int g = 0; g < 4; ++g) weights[kw][u][g][lane] = make_float4(w[4 * g], w[4 * g + 1], w[4 * g + 2], w[4 * g + 3]);
          b[u][0] = pack_quad<E>(w);
          b[u][1] = pack_quad<E>(w + 8);
        }
      }
      pk_lds_barrier();
      if constexpr (B) {
        float ds[32];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const float4 w = weights[kw][u][g][lane];
            ds[16 * u + 4 * g] = w.x;
            ds[16 * u + 4 * g + 1] = w.y;
            ds[16 * u + 4 * g + 2] = w.z;
            ds[16 * u + 4 * g + 3] = w.w;
          }
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float w = ds[16 * u + i];
            ds[16 * u + i] = sees(u, i, kFp16 ? w * dscale * x[u][i] : w * x[u][i]);
          }
          if constexpr (decltype(masked)::value) {
            const int j0 = i0 + 32 * u;
            if (wkey == 0 && j0 <= -shift && -shift < j0 + 32) {  // the row that sees the first key only has dS = 0
#pragma unroll
              for (int i = 0; i < 16; ++i) ds[16 * u + i] = 8 * (i / 4) + i % 4 + 4 * half == -shift - j0 ? 0.f : ds[16 * u + i];
            }
          }
        }
        if constexpr (kFp16) dscale = ldexpf(dscale, -fit.fit(ds, acc));
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          b[u][0] = pack_quad<E>(ds + 16 * u);
          b[u][1] = pack_quad<E>(ds + 16 * u + 8);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < 4 * DB; ++i) {
        uint4 q[1] = {c[i % PRE]};
        if constexpr (decltype(masked)::value) unclean |= pk_clear_not_finite<E>(q);
        acc[i % DB] = mma(E{}, q[0], b[i / (2 * DB)][i / DB % 2], acc[i % DB]);
        if (i + PRE < 4 * DB) c[i % PRE] = column(i + PRE);
        __builtin_amdgcn_sched_barrier(0);
      }
    };

    int cur = per > 0 ? first + t0 % per : 0;  // the tile that is computed
    // Queries of tiles from `full` on see every key of the workgroup's block.
    const int full = p.causal ? (key0 + BN - 1 - shift + 63) >> 6 : first;
    auto tile = [&](auto buf) __attribute__((always_inline)) {
      constexpr int N = decltype(buf)::value;
      const uint8_t *rc = N ? (B ? gt1 : qt1) : (B ? gt0 : qt0), *cc = N ? (B ? qt1 : gt1) : (B ? qt0 : gt0);
      const float* sc = N ? (B ? nd1 : nl1) : (B ? nd0 : nl0);
      load(N ? qt0 : qt1, N ? gt0 : gt1, N ? nl0 : nl1, N ? nd0 : nd1);
      if (wkey < pt.len && cur >= full)
        whole(PkInt<0>{}, rc, cc, sc, 64 * cur);
      else if (wkey < pt.len && 64 * cur + 63 + shift >= wkey)
        whole(PkInt<1>{}, rc, cc, sc, 64 * cur);
      else
        pk_lds_barrier();
      if (++cur == ntq) cur = first;
      pk_tile_barrier();
    };
    int n = 0;
#pragma unroll 1
    for (; n + 1 < total; n += 2) {
      tile(PkInt<0>{});
      tile(PkInt<1>{});
    }
    if (n < total) tile(PkInt<0>{});
    if (__builtin_expect(unclean, 0)) {
      for (int x = t0; x < t0 + total; ++x) {
        const int h = x / per, i0 = 64 * (first + x % per);
        for (int i = i0; i < min(i0 + 64, min(64 * full, lq)); ++i) {
          const uint16_t* row = B ? qbase + (int64_t)i * p.qst + (int64_t)h * p.qsh : gbase + (int64_t)i * p.gst + (int64_t)h * p.gsh;
          pk_add_not_finite<E, B>(row, half, key <= i + shift, acc);
        }
      }
    }
    // Rows of a sequence of one key all have dS = 0.
    const float f = B ? (pt.len == 1 ? 0.f : kFp16 ? fminf(ldexpf(p.scale, -fit.e), 3e38f) : p.scale) : kFp16 ? ldexpf(1.f, -14) : 1.f;
    const int64_t t = pt.start + (on ? key : 0);
    if (parts > 1) {
      float* dst = p.part_dkv + ((2 * part + (B ? 0 : 1)) * (int64_t)p.Tk + t) * p.Hk * D + (int64_t)hk * D;
#pragma unroll
      for (int db = 0; db < DB; ++db) pk_store_part(dst + 32 * db, acc[db], f, half, on);
      return;
    }
    uint16_t* dst = B ? p.dk + t * p.dkst + (int64_t)hk * p.dksh : p.dv + t * p.dvst + (int64_t)hk * p.dvsh;
#pragma unroll
    for (int db = 0; db < DB; ++db) pk_store_col<E>(dst + 32 * db, acc[db], f, half, on);
  };

  if (total > 0) {
    load(qt0, gt0, nl0, nd0);
    pk_tile_barrier();
  }
  if (wave < 4)
    role(PkInt<0>{});
  else
    role(PkInt<1>{});
}

// Sums the parts of the rows that were cut, in order. KEYS: dk (blockIdx.y = 0) and dv; else dq.
template <typename E, int D, bool KEYS>
__global__ __launch_bounds__(256) void packed_bwd_join_kernel(const PackedBwdParams p) {
  constexpr int LPR = D / 4;
  const int H = KEYS ? p.Hk : p.H, T = KEYS ? p.Tk : p.Tq;
  const int64_t rows = (int64_t)T * H, row = (int64_t)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
  const int c = threadIdx.x % LPR;
  if (row >= rows) return;
  const int t = (int)(row / H), h = (int)(row - (int64_t)t * H);
  const PackedTile pt = pk_token(KEYS ? p.cu_k : p.cu_q, p.n, T, t);
  int other = 0;
  if (pt.seq >= 1 && pt.seq <= p.n) {
    const int32_t* cu = KEYS ? p.cu_q : p.cu_k;
    const int To = KEYS ? p.Tq : p.Tk;
    other = max(0, pk_bound(cu, p.n, To, pt.seq + 1) - pk_bound(cu, p.n, To, pt.seq));
  }
  const int at = t - pt.start;
  const int parts = KEYS ? pk_parts(dkv_work(p, pt.len, other, at / kBwdTile), p.split_dkv, p.per_dkv)
                         : pk_parts(dq_work(p, pt.len, other, (at * p.G + h % p.G) / kBwdTile), p.split_dq, p.per_dq);
  if (parts == 1) return;
  const float* src = KEYS ? p.part_dkv + blockIdx.y * rows * D : p.part_dq;
  const int64_t step = (KEYS ? 2 : 1) * rows * D;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int i = 0; i < parts; ++i) {
    const float4 x = reinterpret_cast<const float4*>(src + i * step + row * D)[c];
    s.x += x.x;
    s.y += x.y;
    s.z += x.z;
    s.w += x.w;
  }
  uint16_t* dst = !KEYS            ? p.dq + (int64_t)t * p.dqst + (int64_t)h * p.dqsh
                  : blockIdx.y == 0 ? p.dk + (int64_t)t * p.dkst + (int64_t)h * p.dksh
                                    : p.dv + (int64_t)t * p.dvst + (int64_t)h * p.dvsh;
  *reinterpret_cast<uint2*>(dst + 4 * c) = make_uint2(pack_pair(E{}, s.x, s.y), pack_pair(E{}, s.z, s.w));
}

// Parts that the keys of a dQ workgroup and the queries of a dK/dV workgroup are cut into, where the tiles
// alone leave workgroup slots empty, or where one long sequence among short ones would run on by itself: at
// most `dq`, one for every `per_dq` tiles of 64, which the kernels find from the lengths. The fewer workgroups there
// are, the shorter the parts: 8 to 64 tiles. The parts' fp32 sums are joined in order by another launch; their
// workspace stays below 512 MiB a pass. 37 causal sequences of 1 to 3,151 tokens, 8 heads over 2: forward and
// backward 381 us with as many parts for every sequence, 249 so; 4 heads, 2 sequences of 3,000 to 6,000: 298, 282.
struct BwdPlan {
  int dq, dkv, per_dq, per_dkv;
  int64_t slots_q, slots_k;  // entries of the lists of tiles (0: no list)
  size_t dq_bytes, dkv_bytes;
};

BwdPlan packed_bwd_plan(int64_t n, int64_t Tq, int64_t Tk, int64_t Hq, int64_t Hk, int64_t D) {
  const int64_t G = Hq / Hk;
  // rows: of the workgroups' own side; other: of the loops'; bytes: of a part; slots: workgroups at once.
  auto parts = [&](int64_t rows, int64_t other, int64_t bytes, int64_t slots, int& per) {
    // Tiles: at least one per sequence that has rows, and the last one of a sequence half full.
    const int64_t wgs = (rows / 128 + (rows < 128 * n ? n : n / 2) + 1) * Hk;
    per = (int)(wgs * 64 / slots < 8 ? 8 : wgs * 64 / slots > 64 ? 64 : wgs * 64 / slots);
    if (other / (n > 0 ? n : 1) / 16 < per) return 1;  // four times the average is no part
    int64_t s = 2 * slots / wgs;
    if (s > (other / 64 + per) / per) s = (other / 64 + per) / per;
    if (s > (512ll << 20) / bytes) s = (512ll << 20) / bytes;
    return (int)(s > 16 ? 16 : s > 1 ? s : 1);
  };
  BwdPlan b = {};
  // A single sequence's tiles are in falling order as they are. 29 training calls of 1 to 171 sequences
  // took 1.06 times as long without the lists (geometric mean; between 0.98 and 1.20).
  b.slots_q = Tq * G / kBwdTile + n + 2;
  b.slots_k = Tk / kBwdTile + n + 2;
  if (n < 2 || Tq == 0 || b.slots_q > kPkOrderMax) b.slots_q = 0;
  if (n < 2 || Tq == 0 || b.slots_k > kPkOrderMax) b.slots_k = 0;
  const int64_t dq_part = Tq * Hq * D * 4, dkv_part = 2 * Tk * Hk * D * 4;
  b.dq = parts(Tq * G, Tk, dq_part > 0 ? dq_part : 1, D == 64 ? 768 : 512, b.per_dq);
  b.dkv = parts(Tk, Tq * G, dkv_part > 0 ? dkv_part : 1, D == 64 ? 512 : 256, b.per_dkv);
  b.dq_bytes = b.dq > 1 ? (size_t)b.dq * dq_part : 0;
  b.dkv_bytes = b.dkv > 1 ? (size_t)b.dkv * dkv_part : 0;
  return b;
}

template <typename E, int D>
int packed_bwd_launch(const PackedBwdParams& p, hipStream_t stream) {
  const int64_t qgrid = (int64_t)dq_slots(p) * p.Hk * p.split_dq, kgrid = (int64_t)dkv_slots(p) * p.Hk * p.split_dkv;
  const int64_t rgrid = 2 + p.Tq / kStatTokens + (int64_t)p.n + 2;
  const int64_t qjoin = ((int64_t)p.Tq * p.H * (D / 4) + 255) / 256, kjoin = ((int64_t)p.Tk * p.Hk * (D / 4) + 255) / 256;
  // All launches fit, or none is made.
  if (p.Tq > 0) {
    GW_CHECK_GRID(rgrid, 256);
    GW_CHECK_GRID(qgrid, 256);
    if (p.split_dq > 1) GW_CHECK_GRID(qjoin, 256);
  }
  if (p.Tk > 0) {
    GW_CHECK_GRID(kgrid, D == 64 ? 256 : 512);
    if (p.split_dkv > 1) GW_CHECK_GRID(kjoin, 256);
  }
  if (p.Tq > 0) {
    hipLaunchKernelGGL((packed_bwd_stats_kernel<E, D>), dim3((uint32_t)rgrid), dim3(256), 0, stream, p);
    GW_HIP_LAUNCH_CHECK("gw_packed_attn_bwd (rows)");
    hipLaunchKernelGGL((packed_bwd_dq_kernel<E, D>), dim3((uint32_t)qgrid), dim3(256), 0, stream, p);
    GW_HIP_LAUNCH_CHECK("gw_packed_attn_bwd (dq)");
    if (p.split_dq > 1) {
      hipLaunchKernelGGL((packed_bwd_join_kernel<E, D, false>), dim3((uint32_t)qjoin), dim3(256), 0, stream, p);
      GW_HIP_LAUNCH_CHECK("gw_packed_attn_bwd (dq join)");
    }
  }
  if (p.Tk > 0) {
    const dim3 tiles((uint32_t)kgrid);
    if constexpr (D == 64) {
      hipLaunchKernelGGL(packed_bwd_dkv_kernel<E>, tiles, dim3(256), 0, stream, p);
    } else {
      hipLaunchKernelGGL(packed_bwd_dkv_pair_kernel<E>, tiles, dim3(512), 0, stream, p);
    }
    GW_HIP_LAUNCH_CHECK("gw_packed_attn_bwd (dk, dv)");
    if (p.split_dkv > 1) {
      hipLaunchKernelGGL((packed_bwd_join_kernel<E, D, true>), dim3((uint32_t)kjoin, 2), dim3(256), 0, stream, p);
      GW_HIP_LAUNCH_CHECK("gw_packed_attn_bwd (dk, dv join)");
    }
  }
  return GW_OK;
}

template <typename E>
int packed_bwd_dim(const PackedBwdParams& p, int64_t D, hipStream_t stream) {
  return D == 64 ? packed_bwd_launch<E, 64>(p, stream) : packed_bwd_launch<E, 128>(p, stream);
}

inline size_t pk_align(size_t n) { return (n + 255) & ~(size_t)255; }

}  // namespace
}  // namespace gw

extern "C" size_t gw_packed_attn_bwd_workspace_size(int64_t n, int64_t Tq, int64_t Tk, int64_t Hq, int64_t Hk, int64_t D) {
  if (n < 0 || Tq < 0 || Tk < 0 || Hk < 1 || Hq < Hk || D < 1) return 0;
  const gw::BwdPlan b = gw::packed_bwd_plan(n, Tq, Tk, Hq, Hk, D);
  return gw::pk_align((size_t)Tq * Hq * 8) + gw::pk_align(b.dq_bytes) + gw::pk_align(b.dkv_bytes) + 8 * (size_t)(b.slots_q + b.slots_k);
}

extern "C" int gw_packed_attn_bwd(int dtype, const void* q, const int64_t* q_strides, const void* k,
                                  const int64_t* k_strides, const void* v, const int64_t* v_strides,
                                  const int32_t* cu_q, const int32_t* cu_k, const void* o, const int64_t* o_strides,
                                  const void* o_rest, const void* dout, const int64_t* do_strides, const float* lse, void* dq,
                                  const int64_t* dq_strides, void* dk, const int64_t* dk_strides, void* dv,
                                  const int64_t* dv_strides, int64_t n, int64_t Tq, int64_t Tk, int64_t Hq, int64_t Hk,
                                  int64_t D, int causal, float softmax_scale, void* workspace, size_t workspace_bytes,
                                  void* stream) {
  using namespace gw;
  clear_error();
  PackedArgs a = {dtype, n, Tq, Tk, Hq, Hk, D, softmax_scale};
  const int rc = pk_check_args(a);
  if (rc != GW_OK) return rc;
  if (Tq == 0 && Tk == 0) return GW_OK;
  GW_CHECK_ARG(cu_q && cu_k && q_strides && k_strides && v_strides && o_strides && do_strides && dq_strides &&
                   dk_strides && dv_strides && (Tq == 0 || (q && o && o_rest && dout && lse && dq)) && (Tk == 0 || (k && v && dk && dv)),
               "a tensor is missing");
  GW_CHECK_ARG(pk_rows_ok(q, q_strides) && pk_rows_ok(k, k_strides) && pk_rows_ok(v, v_strides) &&
                   pk_rows_ok(o, o_strides) && aligned16(o_rest) && pk_rows_ok(dout, do_strides) && pk_rows_ok(dq, dq_strides) &&
                   pk_rows_ok(dk, dk_strides) && pk_rows_ok(dv, dv_strides),
               "q, k, v, o, dO, dq, dk and dv need 16-byte aligned rows, with token strides in [0, 2^24)");
  const size_t need = gw_packed_attn_bwd_workspace_size(n, Tq, Tk, Hq, Hk, D);
  GW_CHECK_ARG(workspace && aligned16(workspace) && workspace_bytes >= need, "workspace of %zu bytes, %zu are needed",
               workspace_bytes, need);
  PackedBwdParams p = {};
  p.q = static_cast<const uint16_t*>(q);
  p.k = static_cast<const uint16_t*>(k);
  p.v = static_cast<const uint16_t*>(v);
  p.o = static_cast<const uint16_t*>(o);
  p.rest = static_cast<const uint16_t*>(o_rest);
  p.dout = static_cast<const uint16_t*>(dout);
  p.lse = lse;
  p.dq = static_cast<uint16_t*>(dq);
  p.dk = static_cast<uint16_t*>(dk);
  p.dv = static_cast<uint16_t*>(dv);
  char* ws = static_cast<char*>(workspace);
  p.nlse = reinterpret_cast<float*>(ws);
  p.ndelta = p.nlse + Tq * Hq;
  const BwdPlan b = packed_bwd_plan(n, Tq, Tk, Hq, Hk, D);
  p.split_dq = b.dq;
  p.split_dkv = b.dkv;
  p.per_dq = b.per_dq;
  p.per_dkv = b.per_dkv;
  p.part_dq = reinterpret_cast<float*>(ws + pk_align((size_t)Tq * Hq * 8));
  p.part_dkv = p.part_dq + pk_align(b.dq_bytes) / sizeof(float);
  int2* lists = reinterpret_cast<int2*>(p.part_dkv + pk_align(b.dkv_bytes) / sizeof(float));
  if (b.slots_q) p.order_q = lists;
  if (b.slots_k) p.order_k = lists + b.slots_q;
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
  p.gst = do_strides[0];
  p.gsh = do_strides[1];
  p.dqst = dq_strides[0];
  p.dqsh = dq_strides[1];
  p.dkst = dk_strides[0];
  p.dksh = dk_strides[1];
  p.dvst = dv_strides[0];
  p.dvsh = dv_strides[1];
  p.scale = softmax_scale;
  p.scale_log2 = softmax_scale * kDLog2e;
  hipStream_t s = static_cast<hipStream_t>(stream);
  return dtype == GW_DTYPE_BF16 ? packed_bwd_dim<BF16>(p, D, s) : packed_bwd_dim<FP16>(p, D, s);
}
