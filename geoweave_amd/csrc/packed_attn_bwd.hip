// Backward of the attention over packed sequences (gfx950): dQ, dK, dV without atomics on the
// gradients, D = 64 or 128.
//
// With P the softmax weights (formed again from the forward's lse) and delta_i = o_i . do_i:
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
// exponents for them: P is scaled by 2^14; dS in the dQ pass by a power of two per row, from the row's
// |do| and the sequence's largest |v| (|dP - delta| <= 2 |do_i| max_j |v_j|), in the dK/dV pass by one per
// sequence and key head, so that |dS| stays below 2^15. The powers are exact and taken out of the fp32
// sums again.
//
// Rows behind a sequence's end arrive as zeros, and rows that see no key have P = 0.
#include <math.h>

#include "gw_packed.h"

namespace gw {
namespace {

struct PackedBwdParams {
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;
  const uint16_t* o;
  const uint16_t* dout;
  const float* lse;
  uint16_t* dq;
  uint16_t* dk;
  uint16_t* dv;
  float2* stats;      // [H][Tq] {lse log2(e), +inf for a row without keys; delta}
  uint32_t* max_do;   // [n + 2][Hk] largest |do_i| of a sequence's rows, as float bits (fp16 only)
  uint32_t* max_v;    // [n + 2][Hk] largest |v_j|
  const int32_t* cu_q;
  const int32_t* cu_k;
  int n, Tq, Tk, H, Hk, G, causal;
  int64_t qst, qsh, kst, ksh, vst, vsh, ost, osh, gst, gsh;
  int64_t dqst, dqsh, dkst, dksh, dvst, dvsh;
  float scale, scale_log2;
};

// Exponent e with 2 bound 2^e <= 2^15 (0 where there is no bound to speak of).
__device__ __forceinline__ int pk_scale_exp(float bound) {
  if (!(bound > 0.f) || !(bound < INFINITY)) return 0;
  int x;
  (void)frexpf(bound, &x);  // bound < 2^x
  return min(max(14 - x, -100), 100);
}

__global__ __launch_bounds__(256) void packed_bwd_clear_kernel(uint32_t* a, int64_t n) {
  for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) a[i] = 0u;
}

// stats of 256 / (D / 8) rows at a time: D / 8 lanes per (token, head) row. MAXIMA: also the
// sequences' largest row norms (the maximum does not depend on the order of the atomics; rows that
// are not finite have no part in it, their gradients are not finite whatever the scale).
constexpr int kStatTokens = 16;

template <typename E, int D, bool MAXIMA>
__global__ __launch_bounds__(256) void packed_bwd_stats_kernel(const PackedBwdParams p) {
  constexpr int LPR = D / 8;
  const PackedTile pt = pk_find_tile(p.cu_q, p.n, p.Tq, 1, kStatTokens, blockIdx.x);
  const int t0 = pt.tile * kStatTokens;
  if (t0 >= pt.len) return;
  const int rows = min(kStatTokens, pt.len - t0) * p.H;
  const int li = threadIdx.x % LPR;
  for (int r = threadIdx.x / LPR; r < rows; r += 256 / LPR) {
    const int t = pt.start + t0 + r / p.H, h = r % p.H;
    float a[8], b[8];
    unpack8<E>(*reinterpret_cast<const uint4*>(p.o + (int64_t)t * p.ost + (int64_t)h * p.osh + li * 8), a);
    unpack8<E>(*reinterpret_cast<const uint4*>(p.dout + (int64_t)t * p.gst + (int64_t)h * p.gsh + li * 8), b);
    float s = 0.f, nn = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      s = fmaf(a[i], b[i], s);
      nn = fmaf(b[i], b[i], nn);
    }
    s = group_sum<LPR>(s);
    if (MAXIMA) nn = group_sum<LPR>(nn);
    if (li == 0) {
      const float l = p.lse[(int64_t)t * p.H + h];
      p.stats[(int64_t)h * p.Tq + t] = make_float2(l == -INFINITY ? INFINITY : l * kDLog2e, s);
      if (MAXIMA && nn < INFINITY) atomicMax(p.max_do + (int64_t)pt.seq * p.Hk + h / p.G, __float_as_uint(sqrtf(nn)));
    }
  }
}

template <typename E, int D>
__global__ __launch_bounds__(256) void packed_bwd_vmax_kernel(const PackedBwdParams p) {
  constexpr int LPR = D / 8;
  const PackedTile pt = pk_find_tile(p.cu_k, p.n, p.Tk, 1, kStatTokens, blockIdx.x);
  const int t0 = pt.tile * kStatTokens;
  if (t0 >= pt.len) return;
  const int rows = min(kStatTokens, pt.len - t0) * p.Hk;
  const int li = threadIdx.x % LPR;
  for (int r = threadIdx.x / LPR; r < rows; r += 256 / LPR) {
    const int t = pt.start + t0 + r / p.Hk, h = r % p.Hk;
    float a[8], nn = 0.f;
    unpack8<E>(*reinterpret_cast<const uint4*>(p.v + (int64_t)t * p.vst + (int64_t)h * p.vsh + li * 8), a);
#pragma unroll
    for (int i = 0; i < 8; ++i) nn = fmaf(a[i], a[i], nn);
    nn = group_sum<LPR>(nn);
    if (li == 0 && nn < INFINITY) atomicMax(p.max_v + (int64_t)pt.seq * p.Hk + h, __float_as_uint(sqrtf(nn)));
  }
}

// ---------------------------------------------------------------------------------------
// dQ: the forward's decomposition.
// ---------------------------------------------------------------------------------------
template <typename E, int D, int QPW>
__global__ __launch_bounds__(256, 2) void packed_bwd_dq_kernel(const PackedBwdParams p) {
  constexpr int KS = D / 16, DB = D / 32, BM = 128 * QPW;
  constexpr int kTileBytes = 64 * 2 * D;
  constexpr bool kFp16 = __is_same(E, FP16);
  __shared__ __align__(16) uint8_t kt0[kTileBytes], kt1[kTileBytes], vt0[kTileBytes], vt1[kTileBytes];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, half = lane >> 5;
  const int hk = blockIdx.x % p.Hk;
  const PackedTile pt = pk_find_tile(p.cu_q, p.n, p.Tq, p.G, BM, blockIdx.x / p.Hk);
  const int rows = pt.len * p.G;
  const int ntile = (rows + BM - 1) / BM;
  if (pt.tile >= ntile) return;
  const int row0 = (p.causal ? ntile - 1 - pt.tile : pt.tile) * BM;
  int k0, lk;
  pk_other(p.cu_k, p.n, p.Tk, pt.seq, k0, lk);
  const int shift = lk - pt.len;
  const float sl2 = p.scale_log2;

  int lim[QPW], lim_lo[QPW], tok[QPW], head[QPW];
  bool on[QPW];
  uint4 qa[QPW][KS], ga[QPW][KS];
  float nlse[QPW], delta[QPW], unscale[QPW];
#pragma unroll
  for (int a = 0; a < QPW; ++a) {
    const int base = row0 + (wave * QPW + a) * 32;
    const int r = min(base + col, rows - 1);
    on[a] = base + col < rows;
    tok[a] = r / p.G;
    head[a] = hk * p.G + (r - tok[a] * p.G);
    lim[a] = p.causal ? min(tok[a] + shift, lk - 1) : lk - 1;
    lim_lo[a] = __builtin_amdgcn_readfirstlane(lim[a]);
    const int64_t t = pt.start + tok[a];
    const uint16_t* qr = p.q + t * p.qst + (int64_t)head[a] * p.qsh + half * 8;
    const uint16_t* gr = p.dout + t * p.gst + (int64_t)head[a] * p.gsh + half * 8;
    float nn = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      qa[a][ks] = *reinterpret_cast<const uint4*>(qr + ks * 16);
      ga[a][ks] = *reinterpret_cast<const uint4*>(gr + ks * 16);
      if (kFp16) nn = dot2(E{}, ga[a][ks].x, ga[a][ks].x, dot2(E{}, ga[a][ks].y, ga[a][ks].y,
                      dot2(E{}, ga[a][ks].z, ga[a][ks].z, dot2(E{}, ga[a][ks].w, ga[a][ks].w, nn))));
    }
    const float2 st = p.stats[(int64_t)head[a] * p.Tq + t];
    int e = 0;
    if (kFp16) e = pk_scale_exp(sqrtf(pair_sum(nn)) * __uint_as_float(p.max_v[(int64_t)pt.seq * p.Hk + hk]));
    nlse[a] = (float)e - st.x;  // p 2^e = 2^(s - lse + e)
    delta[a] = st.y;
    unscale[a] = ldexpf(p.scale, -e);
  }
  auto last_key = [&](int r) { return p.causal ? min(min(r, rows - 1) / p.G + shift, lk - 1) : lk - 1; };
  const int lim_wave = row0 + wave * QPW * 32 < rows ? last_key(row0 + (wave + 1) * QPW * 32 - 1) : -1;
  const int keys = last_key(row0 + BM - 1) + 1;
  const int ntk = keys > 0 ? (keys + 63) >> 6 : 0;

  f32x16 acc[QPW][DB];
#pragma unroll
  for (int a = 0; a < QPW; ++a)
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[a][db][r] = 0.f;

  PkRows<D, 256> krows, vrows;
  krows.init(p.k + (int64_t)k0 * p.kst + (int64_t)hk * p.ksh, p.kst, lk, tid);
  vrows.init(p.v + (int64_t)k0 * p.vst + (int64_t)hk * p.vsh, p.vst, lk, tid);

  auto sub = [&](const uint8_t* kt, const uint8_t* vt, int st, int j0) __attribute__((always_inline)) {
    f32x16 s[QPW], dp[QPW];
#pragma unroll
    for (int a = 0; a < QPW; ++a)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[a][r] = 0.f;
        dp[a][r] = -delta[a];
      }
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const uint4 ka = pk_row_quad<D>(kt, st, ks, lane);
      const uint4 va = pk_row_quad<D>(vt, st, ks, lane);
#pragma unroll
      for (int a = 0; a < QPW; ++a) s[a] = mma(E{}, ka, qa[a][ks], s[a]);
#pragma unroll
      for (int a = 0; a < QPW; ++a) dp[a] = mma(E{}, va, ga[a][ks], dp[a]);
    }
    uint4 kc[DB][2];
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) kc[db][ks] = pk_col_quad<D>(kt, st, ks, db, lane);
#pragma unroll
    for (int a = 0; a < QPW; ++a) {
      float ds[16];
#pragma unroll
      for (int r = 0; r < 16; ++r) ds[r] = fexp2(fmaf(s[a][r], sl2, nlse[a])) * dp[a][r];
      if (j0 + 31 > lim_lo[a]) {
        const int room = lim[a] - j0 - 4 * half;
#pragma unroll
        for (int r = 0; r < 16; ++r) ds[r] = 8 * (r / 4) + r % 4 <= room ? ds[r] : 0.f;
      }
      const uint4 b0 = pack_quad<E>(ds), b1 = pack_quad<E>(ds + 8);
#pragma unroll
      for (int db = 0; db < DB; ++db) acc[a][db] = mma(E{}, kc[db][0], b0, acc[a][db]);
#pragma unroll
      for (int db = 0; db < DB; ++db) acc[a][db] = mma(E{}, kc[db][1], b1, acc[a][db]);
    }
  };

  if (ntk > 0) {
    krows.load(0, kt0);
    vrows.load(0, vt0);
    pk_tile_barrier();
    auto tile = [&](int n, const uint8_t* kc, const uint8_t* vc, uint8_t* kn, uint8_t* vn) __attribute__((always_inline)) {
      krows.load(min(n + 1, ntk - 1), kn);
      vrows.load(min(n + 1, ntk - 1), vn);
      if (64 * n <= lim_wave) {
        sub(kc, vc, 0, 64 * n);
        sub(kc, vc, 1, 64 * n + 32);
      }
      pk_tile_barrier();
    };
    int n = 0;
#pragma unroll 1
    for (; n + 1 < ntk; n += 2) {
      tile(n, kt0, vt0, kt1, vt1);
      tile(n + 1, kt1, vt1, kt0, vt0);
    }
    if (n < ntk) tile(n, kt0, vt0, kt1, vt1);
  }
#pragma unroll
  for (int a = 0; a < QPW; ++a) {
    uint16_t* row = p.dq + (int64_t)(pt.start + tok[a]) * p.dqst + (int64_t)head[a] * p.dqsh;
#pragma unroll
    for (int db = 0; db < DB; ++db) pk_store_col<E>(row + 32 * db, acc[a][db], unscale[a], half, on[a]);
  }
}

// ---------------------------------------------------------------------------------------
// dK and dV: 4 waves x 32 keys of one key head; tiles of 64 query tokens of each head of the group.
// A lane holds one key and 16 queries of S = Q K^T and dP = dO V^T.
// ---------------------------------------------------------------------------------------
constexpr int kBwdKeys = 128;

template <typename E, int D>
__global__ __launch_bounds__(256, D == 64 ? 2 : 1) void packed_bwd_dkv_kernel(const PackedBwdParams p) {
  constexpr int KS = D / 16, DB = D / 32;
  constexpr int kTileBytes = 64 * 2 * D;
  constexpr bool kFp16 = __is_same(E, FP16);
  __shared__ __align__(16) uint8_t qt0[kTileBytes], qt1[kTileBytes], gt0[kTileBytes], gt1[kTileBytes];
  __shared__ __align__(16) float2 st0[64], st1[64];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 31, half = lane >> 5;
  const int hk = blockIdx.x % p.Hk;
  const PackedTile pt = pk_find_tile(p.cu_k, p.n, p.Tk, 1, kBwdKeys, blockIdx.x / p.Hk);
  const int key0 = pt.tile * kBwdKeys;
  if (key0 >= pt.len) return;
  int q0, lq;
  pk_other(p.cu_q, p.n, p.Tq, pt.seq, q0, lq);
  const int shift = pt.len - lq;  // causal: key j is seen by tokens i >= j - shift
  const float sl2 = p.scale_log2;
  const int wkey = key0 + wave * 32;
  const int key = wkey + col;
  const bool on = key < pt.len;

  // Stationary operands: K and V rows of this lane's key.
  uint4 kb[KS], vb[KS];
  {
    const int64_t t = pt.start + (on ? key : pt.len - 1);
    const uint16_t* kr = p.k + t * p.kst + (int64_t)hk * p.ksh + half * 8;
    const uint16_t* vr = p.v + t * p.vst + (int64_t)hk * p.vsh + half * 8;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      kb[ks] = *reinterpret_cast<const uint4*>(kr + ks * 16);
      vb[ks] = *reinterpret_cast<const uint4*>(vr + ks * 16);
    }
  }
  // fp16: dS = P (dP - delta) 2^e, P 2^14.
  int e = 0;
  if (kFp16) {
    const int64_t at = (int64_t)pt.seq * p.Hk + hk;
    e = pk_scale_exp(__uint_as_float(p.max_do[at]) * __uint_as_float(p.max_v[at]));
  }
  const float dscale = kFp16 ? ldexpf(1.f, e - 14) : 1.f;

  f32x16 ak[DB], av[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) ak[db][r] = av[db][r] = 0.f;

  const int first = p.causal ? max(0, key0 - shift) >> 6 : 0;  // first tile with a query that sees a key
  const int ntq = (lq + 63) >> 6;
  const int per = ntq > first ? ntq - first : 0;
  const int total = per * p.G;

  PkRows<D, 256> qrows, grows;
  const uint16_t* qbase = p.q + (int64_t)q0 * p.qst + (int64_t)hk * p.G * p.qsh;
  const uint16_t* gbase = p.dout + (int64_t)q0 * p.gst + (int64_t)hk * p.G * p.gsh;
  const float2* sbase = p.stats + (int64_t)hk * p.G * p.Tq + q0;
  qrows.init(qbase, p.qst, lq, tid);
  grows.init(gbase, p.gst, lq, tid);
  // The tile that is loaded next: head of the group and tile of its queries.
  int ld_h = 0, ld_t = first;
  auto load = [&](uint8_t* qd, uint8_t* gd, float2* sd) __attribute__((always_inline)) {
    qrows.base = uniform_ptr(reinterpret_cast<const char*>(qbase + (int64_t)ld_h * p.qsh));
    grows.base = uniform_ptr(reinterpret_cast<const char*>(gbase + (int64_t)ld_h * p.gsh));
    qrows.load(ld_t, qd);
    grows.load(ld_t, gd);
    const char* sp = reinterpret_cast<const char*>(sbase + (int64_t)ld_h * p.Tq + ld_t * 64);
    const __amdgpu_buffer_rsrc_t rs = pk_rsrc(sp, (int64_t)(lq - ld_t * 64) * 8);
    // 64 {lse, delta} pairs, 4 bytes a lane (their start is only 8-byte aligned): waves 0 and 1.
    if (wave < 2)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rs, (__attribute__((address_space(3))) void*)(reinterpret_cast<char*>(sd) + wave * 256), 4,
          wave * 256 + lane * 4, 0, 0, 0);
    if (++ld_t == ntq) {
      ld_t = first;
      if (++ld_h == p.G) ld_h = p.G - 1;  // past the end: a tile again that no wave uses
    }
  };

  auto sub = [&](const uint8_t* qt, const uint8_t* gt, const float2* sd, int st, int i0) __attribute__((always_inline)) {
    f32x16 s, dp;
    float nl[16];
    // Entry r of this lane is query i0 + 8 (r / 4) + 4 half + r % 4.
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const float4* sp = reinterpret_cast<const float4*>(sd + 32 * st + 8 * g + 4 * half);
      const float4 a = sp[0], b = sp[1];
      nl[4 * g] = a.x;
      nl[4 * g + 1] = a.z;
      nl[4 * g + 2] = b.x;
      nl[4 * g + 3] = b.z;
      dp[4 * g] = -a.y;
      dp[4 * g + 1] = -a.w;
      dp[4 * g + 2] = -b.y;
      dp[4 * g + 3] = -b.w;
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      s = mma(E{}, pk_row_quad<D>(qt, st, ks, lane), kb[ks], s);
      dp = mma(E{}, pk_row_quad<D>(gt, st, ks, lane), vb[ks], dp);
    }
    float w[16], ds[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) w[r] = fexp2(fmaf(s[r], sl2, (kFp16 ? 14.f : 0.f) - nl[r]));
    if (p.causal && i0 < wkey + 31 - shift) {
      const int need = key - shift - i0 - 4 * half;
#pragma unroll
      for (int r = 0; r < 16; ++r) w[r] = 8 * (r / 4) + r % 4 >= need ? w[r] : 0.f;
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) ds[r] = kFp16 ? w[r] * dscale * dp[r] : w[r] * dp[r];
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      const uint4 pb = pack_quad<E>(w + 8 * ks), db_ = pack_quad<E>(ds + 8 * ks);
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        av[db] = mma(E{}, pk_col_quad<D>(gt, st, ks, db, lane), pb, av[db]);
        ak[db] = mma(E{}, pk_col_quad<D>(qt, st, ks, db, lane), db_, ak[db]);
      }
    }
  };

  if (total > 0) {
    load(qt0, gt0, st0);
    pk_tile_barrier();
    int cur = first;  // the tile that is computed
    auto tile = [&](const uint8_t* qc, const uint8_t* gc, const float2* sc, uint8_t* qn, uint8_t* gn, float2* sn)
                    __attribute__((always_inline)) {
      load(qn, gn, sn);
      if (wkey < pt.len && (!p.causal || 64 * cur + 63 + shift >= wkey)) {
        sub(qc, gc, sc, 0, 64 * cur);
        sub(qc, gc, sc, 1, 64 * cur + 32);
      }
      if (++cur == ntq) cur = first;
      pk_tile_barrier();
    };
    int n = 0;
#pragma unroll 1
    for (; n + 1 < total; n += 2) {
      tile(qt0, gt0, st0, qt1, gt1, st1);
      tile(qt1, gt1, st1, qt0, gt0, st0);
    }
    if (n < total) tile(qt0, gt0, st0, qt1, gt1, st1);
  }
  const int64_t t = pt.start + (on ? key : 0);
  uint16_t* dkr = p.dk + t * p.dkst + (int64_t)hk * p.dksh;
  uint16_t* dvr = p.dv + t * p.dvst + (int64_t)hk * p.dvsh;
  const float fk = kFp16 ? ldexpf(p.scale, -e) : p.scale, fv = kFp16 ? ldexpf(1.f, -14) : 1.f;
#pragma unroll
  for (int db = 0; db < DB; ++db) {
    pk_store_col<E>(dkr + 32 * db, ak[db], fk, half, on);
    pk_store_col<E>(dvr + 32 * db, av[db], fv, half, on);
  }
}

template <typename E, int D, int QPW>
int packed_bwd_launch(const PackedBwdParams& p, hipStream_t stream) {
  constexpr bool kFp16 = __is_same(E, FP16);
  const int64_t qslots = (int64_t)p.Tq * p.G / (128 * QPW) + p.n + 2, kslots = (int64_t)p.Tk / kBwdKeys + p.n + 2;
  GW_CHECK_ARG(qslots * p.Hk < (1ll << 31) && kslots * p.Hk < (1ll << 31), "the grid is too large");
  if (kFp16) {
    const int64_t words = 2 * (int64_t)(p.n + 2) * p.Hk;  // max_do and max_v, one behind the other
    hipLaunchKernelGGL(packed_bwd_clear_kernel, dim3((uint32_t)((words + 255) / 256 > 1024 ? 1024 : (words + 255) / 256)),
                       dim3(256), 0, stream, p.max_do, words);
    GW_HIP_LAUNCH_CHECK("gw_packed_attn_bwd (clear)");
    if (p.Tk > 0) {
      hipLaunchKernelGGL((packed_bwd_vmax_kernel<E, D>), dim3((uint32_t)(p.Tk / kStatTokens + p.n + 2)), dim3(256), 0, stream, p);
      GW_HIP_LAUNCH_CHECK("gw_packed_attn_bwd (v)");
    }
  }
  if (p.Tq > 0) {
    hipLaunchKernelGGL((packed_bwd_stats_kernel<E, D, kFp16>), dim3((uint32_t)(p.Tq / kStatTokens + p.n + 2)), dim3(256), 0,
                       stream, p);
    GW_HIP_LAUNCH_CHECK("gw_packed_attn_bwd (rows)");
    hipLaunchKernelGGL((packed_bwd_dq_kernel<E, D, QPW>), dim3((uint32_t)(qslots * p.Hk)), dim3(256), 0, stream, p);
    GW_HIP_LAUNCH_CHECK("gw_packed_attn_bwd (dq)");
  }
  if (p.Tk > 0) {
    hipLaunchKernelGGL((packed_bwd_dkv_kernel<E, D>), dim3((uint32_t)(kslots * p.Hk)), dim3(256), 0, stream, p);
    GW_HIP_LAUNCH_CHECK("gw_packed_attn_bwd (dk, dv)");
  }
  return GW_OK;
}

template <typename E>
int packed_bwd_dim(const PackedBwdParams& p, int64_t D, hipStream_t stream) {
  return D == 64 ? packed_bwd_launch<E, 64, 2>(p, stream) : packed_bwd_launch<E, 128, 1>(p, stream);
}

inline size_t pk_align(size_t n) { return (n + 255) & ~(size_t)255; }

}  // namespace
}  // namespace gw

extern "C" size_t gw_packed_attn_bwd_workspace_size(int64_t n, int64_t Tq, int64_t Tk, int64_t Hq, int64_t Hk, int64_t D) {
  (void)Tk;
  (void)D;
  if (n < 0 || Tq < 0 || Hq < 1 || Hk < 1) return 0;
  return gw::pk_align((size_t)Tq * Hq * 8) + gw::pk_align((size_t)(n + 2) * Hk * 8);
}

extern "C" int gw_packed_attn_bwd(int dtype, const void* q, const int64_t* q_strides, const void* k,
                                  const int64_t* k_strides, const void* v, const int64_t* v_strides,
                                  const int32_t* cu_q, const int32_t* cu_k, const void* o, const int64_t* o_strides,
                                  const void* dout, const int64_t* do_strides, const float* lse, void* dq,
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
                   dk_strides && dv_strides && (Tq == 0 || (q && o && dout && lse && dq)) && (Tk == 0 || (k && v && dk && dv)),
               "a tensor is missing");
  GW_CHECK_ARG(pk_rows_ok(q, q_strides) && pk_rows_ok(k, k_strides) && pk_rows_ok(v, v_strides) &&
                   pk_rows_ok(o, o_strides) && pk_rows_ok(dout, do_strides) && pk_rows_ok(dq, dq_strides) &&
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
  p.dout = static_cast<const uint16_t*>(dout);
  p.lse = lse;
  p.dq = static_cast<uint16_t*>(dq);
  p.dk = static_cast<uint16_t*>(dk);
  p.dv = static_cast<uint16_t*>(dv);
  char* ws = static_cast<char*>(workspace);
  p.stats = reinterpret_cast<float2*>(ws);
  p.max_do = reinterpret_cast<uint32_t*>(ws + pk_align((size_t)Tq * Hq * 8));
  p.max_v = p.max_do + (n + 2) * Hk;
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
