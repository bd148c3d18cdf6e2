// Pieces shared by the packed and paged attention passes: where a workgroup's tile lies among
// sequences of different lengths, LDS tiles that are read by rows and by columns, and loads that end at a
// sequence's last row.
#pragma once

#include "gw_common.h"
#include "gw_mma.h"

namespace gw {
namespace {

typedef __fp16 pk_fp16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) pk_fp16x4 lds_pk_h4;

// ---------------------------------------------------------------------------------------
// Host checks that the packed entry points share.
// ---------------------------------------------------------------------------------------
struct PackedArgs {
  int dtype;
  int64_t n, Tq, Tk, Hq, Hk, D;
  float scale;
};

inline int pk_check_args(const PackedArgs& a) {
  GW_CHECK_ARG(a.dtype == GW_DTYPE_BF16 || a.dtype == GW_DTYPE_FP16, "unknown dtype %d", a.dtype);
  if (a.D != 64 && a.D != 128) return set_error(GW_ERR_UNSUPPORTED, "head dim %lld is not 64 or 128", (long long)a.D);
  GW_CHECK_ARG(a.n >= 0 && a.Tq >= 0 && a.Tk >= 0, "negative size");
  GW_CHECK_ARG(a.Hk >= 1 && a.Hq >= a.Hk && a.Hq % a.Hk == 0, "%lld query heads are no multiple of %lld key heads",
               (long long)a.Hq, (long long)a.Hk);
  GW_CHECK_ARG(a.scale > 0.f && a.scale <= 3.0e38f, "the softmax scale must be positive and finite");
  if (a.n >= (1ll << 30) || a.Tq > 0x7FFFF000ll / a.Hq || a.Tk > 0x7FFFF000ll / a.Hq)
    return set_error(GW_ERR_UNSUPPORTED, "tokens x heads must stay below 2^31 - 2^12, sequences below 2^30");
  return GW_OK;
}

// Strides {token, head} of a [T, H, D] tensor whose rows are read 16 bytes at a time; 64 rows lie
// within a load's 32-bit offset.
inline bool pk_rows_ok(const void* p, const int64_t* s) {
  return aligned16(p) && s[0] % 8 == 0 && s[1] % 8 == 0 && s[0] >= 0 && s[0] < (1ll << 24);
}

// ---------------------------------------------------------------------------------------
// Sequences. cu[0..n] bounds the n sequences of T packed tokens. Tokens before cu[0] and behind
// cu[n] belong to none: they are treated as sequences 0 and n + 1 without keys (or queries), so that
// their outputs are written (as zeros) like all others. Bounds are clamped to [0, T], so whatever the
// device array holds, no access leaves the tensors.
//
// Tiles without a list: sequence i, whose rows are tokens x g heads, may use the slots from
// floor(start_i g / BM) + i on; the next sequence's first slot is at least ceil(rows_i / BM) later, and
// there are floor(T g / BM) + n + 2 slots in all, a number that the host knows without the lengths. A
// workgroup finds the sequence of its slot by a search with 64 probes at a time (a wave's lanes),
// two rounds for up to 4,094 sequences; slots without a tile end at once.
// ---------------------------------------------------------------------------------------
__device__ __forceinline__ int pk_bound(const int32_t* cu, int n, int T, int i) {
  if (i <= 0) return 0;
  if (i > n + 1) return T;
  return min(max(cu[i - 1], 0), T);
}

struct PackedTile {
  int seq;       // 0..n+1 (0 and n + 1: tokens of no sequence)
  int start;     // first token
  int len;       // tokens
  int tile;      // tile of the sequence
};

__device__ __forceinline__ PackedTile pk_find_tile(const int32_t* cu, int n, int T, int g, int bm, int slot) {
  const int lane = threadIdx.x & 63;
  auto first_slot = [&](int i) { return (int)((uint64_t)((uint32_t)pk_bound(cu, n, T, i) * (uint64_t)g) / (uint32_t)bm) + i; };
  int lo = 0, cnt = n + 2;
  while (cnt > 1) {
    const int step = (cnt + 63) >> 6;
    const int i = lo + lane * step;
    const bool below = lane * step < cnt && first_slot(i) <= slot;
    const uint64_t bal = __builtin_amdgcn_ballot_w64(below);
    const int top = bal ? 63 - __builtin_clzll(bal) : 0;
    lo += top * step;
    cnt = min(step, cnt - top * step);
  }
  PackedTile r;
  r.seq = __builtin_amdgcn_readfirstlane(lo);
  r.start = __builtin_amdgcn_readfirstlane(pk_bound(cu, n, T, r.seq));
  r.len = max(0, __builtin_amdgcn_readfirstlane(pk_bound(cu, n, T, r.seq + 1)) - r.start);
  r.tile = slot - __builtin_amdgcn_readfirstlane(first_slot(r.seq));
  return r;
}

// Longest first. In the order of the slots the workgroups of a long sequence may start last, and the chip
// waits for them. A list of the tiles by falling work (64-row tiles of the other side that a tile meets), in
// classes of an eighth of a power of two, is formed by one workgroup; empty slots come last. Only when a
// tile is computed depends on it, no result does.
constexpr int kPkOrderMax = 4096;  // slots of a list; longer calls have rounds of workgroups enough
constexpr int kPkClasses = 128;

// KEYS: tiles of bm keys that meet queries; else tiles of bm rows (token, head of g) that meet keys, the causal
// ones counted from the sequence's end. order: [slots]; count: LDS, kPkClasses + 1 words;
// parts: how many workgroups share such a tile. A wave takes 64
// sequences at a time.
template <bool KEYS, typename Parts>
__device__ __forceinline__ void pk_order(const int32_t* cu, int T, const int32_t* cu_other, int T_other, int n, int g,
                                         int bm, int causal, int slots, int2* order, uint32_t* count, Parts&& parts) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  auto tiles = [&](auto&& take) {
    auto one = [&](int seq, int len, int other, int ntile, int t) {
      int work;
      if (KEYS) {
        work = ((other + 63) >> 6) - (causal ? max(0, t * bm - (len - other)) >> 6 : 0);
      } else {
        const int last = (min((ntile - t) * bm, len * g) - 1) / g;
        work = ((causal ? min(last + other - len, other - 1) + 1 : other) + 63) >> 6;
      }
      const float share = (float)work / (float)parts(work);
      take(seq, t, work > 0 ? max(0, kPkClasses - 2 - (int)(8.f * flog2(fmaxf(share, 1.f)))) : kPkClasses - 1);
    };
    for (int i0 = 64 * wave; i0 < n + 2; i0 += 256) {
      const int i = i0 + lane;
      int len = 0, other = 0;
      if (i < n + 2) len = max(0, pk_bound(cu, n, T, i + 1) - pk_bound(cu, n, T, i));
      if (i >= 1 && i <= n) other = max(0, pk_bound(cu_other, n, T_other, i + 1) - pk_bound(cu_other, n, T_other, i));
      const int ntile = (len * g + bm - 1) / bm;
      // Sequences of a few tiles: a sequence per lane. The longer ones one by one, a tile per lane.
      const bool few = ntile <= 16;
      for (int t = 0; t < 16 && __builtin_amdgcn_ballot_w64(few && t < ntile); ++t)
        if (few && t < ntile) one(i, len, other, ntile, t);
      for (uint64_t left = __builtin_amdgcn_ballot_w64(!few); left; left &= left - 1) {
        const int l = __builtin_ctzll(left);
        const int ln = __builtin_amdgcn_readlane(len, l), lo = __builtin_amdgcn_readlane(other, l);
        const int nt = __builtin_amdgcn_readlane(ntile, l);
        for (int t = lane; t < nt; t += 64) one(i0 + l, ln, lo, nt, t);
      }
    }
  };
  if (tid < kPkClasses) count[tid] = 0u;
  __syncthreads();
  tiles([&](int, int, int cls) { atomicAdd(count + cls, 1u); });
  __syncthreads();
  if (tid < 64) {  // where each class starts
    const uint32_t a = count[2 * tid], b = count[2 * tid + 1];
    uint32_t x = a + b;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t y = __shfl_up(x, d);
      if (tid >= d) x += y;
    }
    count[2 * tid] = x - a - b;
    count[2 * tid + 1] = x - b;
    if (tid == 63) count[kPkClasses] = x;
  }
  __syncthreads();
  tiles([&](int seq, int t, int cls) {
    const uint32_t at = atomicAdd(count + cls, 1u);
    if (at < (uint32_t)slots) order[at] = make_int2(seq, t);  // bounds out of order may name more tiles
  });
  for (int s = (int)min(count[kPkClasses], (uint32_t)slots) + tid; s < slots; s += 256) order[s] = make_int2(0, -1);
}

// The tile of workgroup slot `slot`, by the list where there is one (tile -1: nothing to do).
__device__ __forceinline__ PackedTile pk_tile(const int2* order, const int32_t* cu, int n, int T, int g, int bm, int slot) {
  if (!order) return pk_find_tile(cu, n, T, g, bm, slot);
  PackedTile r;
  r.seq = __builtin_amdgcn_readfirstlane(order[slot].x);
  r.tile = __builtin_amdgcn_readfirstlane(order[slot].y);
  r.start = __builtin_amdgcn_readfirstlane(pk_bound(cu, n, T, r.seq));
  r.len = max(0, __builtin_amdgcn_readfirstlane(pk_bound(cu, n, T, r.seq + 1)) - r.start);
  return r;
}

// The sequence of token t (a search per lane).
__device__ __forceinline__ PackedTile pk_token(const int32_t* cu, int n, int T, int t) {
  int lo = 0, hi = n + 2;  // the sequence lies in [lo, hi)
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (pk_bound(cu, n, T, mid) <= t)
      lo = mid;
    else
      hi = mid;
  }
  PackedTile r;
  r.seq = lo;
  r.start = pk_bound(cu, n, T, lo);
  r.len = max(0, pk_bound(cu, n, T, lo + 1) - r.start);
  r.tile = 0;
  return r;
}

// The other side's tokens of sequence seq (none for 0 and n + 1).
__device__ __forceinline__ void pk_other(const int32_t* cu, int n, int T, int seq, int& start, int& len) {
  start = len = 0;
  if (seq >= 1 && seq <= n) {
    start = __builtin_amdgcn_readfirstlane(pk_bound(cu, n, T, seq));
    len = max(0, __builtin_amdgcn_readfirstlane(pk_bound(cu, n, T, seq + 1)) - start);
  }
}

// ---------------------------------------------------------------------------------------
// LDS tiles of rows of 2 D bytes: the 16-byte chunk c of row R sits at c ^ pk_swz(R). Sixteen
// consecutive rows at one chunk (row operands) touch all banks evenly, and so do four rows,
// starting at a multiple of four, at four consecutive chunks (column operands).
// ---------------------------------------------------------------------------------------
template <int D>
__device__ __forceinline__ int pk_swz(int R) {
  if constexpr (D == 64)
    return (((R >> 1) & 1) << 2) | (((R >> 2) & 1) << 1) | ((R & 1) ^ ((R >> 3) & 1));
  else
    return ((R & 3) << 2) | ((R >> 2) & 3);
}

template <int V>
struct PkInt {
  static constexpr int value = V;
};

// A descriptor of `bytes` bytes at a wave-uniform base: loads past them, and at kPkNowhere, give zeros.
constexpr uint32_t kPkNowhere = 0xFFFF8000u;
__device__ __forceinline__ __amdgpu_buffer_rsrc_t pk_rsrc(const char* base, int64_t bytes) {
  const uint32_t n = (uint32_t)min(max(bytes, (int64_t)0), (int64_t)0xFFFF0000);
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(uniform_ptr(base)), (short)0,
                                           (int)__builtin_amdgcn_readfirstlane(n), 0x00020000);
}

// Row tiles of one head of one sequence: 64 rows at a time from memory straight to LDS. Lane i of a
// wave writes 16 bytes at the wave's segment + 16 i, so it reads the chunk that the swizzle keeps there.
// Rows past the sequence's end arrive as zeros, whatever the strides (a broadcast row has stride 0), or as the last
// row again (LAST; 64 n < rows).
template <int D, int THREADS>
struct PkRows {
  static constexpr int kRowBytes = 2 * D;
  static constexpr int kChunks = D / 8;                       // 16-byte chunks of a row
  static constexpr int kRowsPerPass = THREADS / kChunks;      // rows of one 16-byte load per thread
  static constexpr int kPasses = 64 / kRowsPerPass;
  const char* base;
  int64_t bytes;       // from base to the end of the last row
  int rows;
  int row;             // this lane's row in pass 0
  uint32_t stride;     // bytes
  uint32_t off;        // this lane's offset in pass 0,
  uint32_t chunk;      // and within its row
  uint32_t seg;        // this wave's segment of the tile in pass 0

  __device__ __forceinline__ void init(const void* p, int64_t stride_elems, int n, int tid) {
    base = uniform_ptr(static_cast<const char*>(p));
    rows = n;
    stride = (uint32_t)stride_elems * 2u;
    bytes = rows > 0 ? (int64_t)(rows - 1) * stride + kRowBytes : 0;
    row = tid / kChunks;
    const int c = tid % kChunks;
    static_assert(kRowsPerPass % 16 == 0, "the swizzle repeats every 16 rows");
    chunk = (uint32_t)((c ^ pk_swz<D>(row)) * 16);
    off = (uint32_t)row * stride + chunk;
    seg = (uint32_t)(tid >> 6) * 1024u;
  }
  // Rows [64 n, 64 n + 64) to lds.
  template <bool LAST = false>
  __device__ __forceinline__ void load(int n, uint8_t* lds) const {
    const int64_t at = (int64_t)n * 64 * stride;
    const __amdgpu_buffer_rsrc_t rs = pk_rsrc(base + at, bytes - at);
    const uint32_t end = LAST ? chunk + (uint32_t)(rows - 1 - 64 * n) * stride : kPkNowhere;
#pragma unroll
    for (int i = 0; i < kPasses; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rs, (__attribute__((address_space(3))) void*)(lds + seg + i * kRowsPerPass * kRowBytes), 16,
          (int)(64 * n + row + i * kRowsPerPass < rows ? off + (uint32_t)(i * kRowsPerPass) * stride : end), 0, 0, 0);
  }
};

// Operand quads of a tile in LDS for the 32x32x16 products, at byte offsets that a lane forms once (the
// empty asm keeps the compiler from forming them again at every read). D = 128 keeps one offset of each
// kind and flips its chunk bits per read.
template <int D>
struct PkLane {
  static constexpr bool kKeep = D == 64;
  static constexpr int kRowOffs = kKeep ? D / 16 : 1, kColOffs = kKeep ? D / 32 * 2 : 1;
  static constexpr uint32_t kNext8 = D == 64 ? 16u : 32u;  // the swizzle of a row eight further on
  uint32_t row_[kRowOffs], col_[kColOffs];

  __device__ __forceinline__ explicit PkLane(int lane) {
    const int col = lane & 31, half = lane >> 5;
    const uint32_t r0 = (uint32_t)(col * 2 * D + ((half ^ pk_swz<D>(col)) << 4));
    const int i = lane & 15, dh = (lane >> 4) & 1, r = 4 * half + (i >> 2);
    const uint32_t c0 = (uint32_t)(r * 2 * D + (((2 * dh + ((i & 3) >> 1)) ^ pk_swz<D>(r)) << 4) + 8 * (i & 1));
#pragma unroll
    for (int ks = 0; ks < kRowOffs; ++ks) {
      row_[ks] = r0 ^ (uint32_t)(ks << 5);
      asm("" : "+v"(row_[ks]));
    }
#pragma unroll
    for (int x = 0; x < kColOffs; ++x) {
      col_[x] = c0 ^ (uint32_t)((x >> 1) << 6) ^ ((x & 1) ? kNext8 : 0u);
      asm("" : "+v"(col_[x]));
    }
  }
  // Rows: lane l supplies row 32 st + l % 32, elements 16 ks + 8 (l / 32) + 0..7.
  __device__ __forceinline__ uint4 row(const uint8_t* tile, int st, int ks) const {
    const uint32_t o = kKeep ? row_[kKeep ? ks : 0] : row_[0] ^ (uint32_t)(ks << 5);
    return *reinterpret_cast<const uint4*>(tile + st * 64 * D + o);
  }
  // Columns: lane l supplies column 32 db + l % 32 of rows 32 st + 16 ks + 4 (l / 32) + {0..3, 8..11}: the
  // rows that the accumulator entries 8 ks + 0..7 of lane l stand for, so that those, packed to 16
  // bits, are the other operand as they are. Two transposing reads (16 lanes read 4 rows of 32 bytes
  // and receive a column each).
  __device__ __forceinline__ uint4 col(const uint8_t* tile, int st, int ks, int db) const {
    uint2 q[2];
#pragma unroll
    for (int jj = 0; jj < 2; ++jj) {
      const uint32_t o = kKeep ? col_[kKeep ? 2 * db + jj : 0] : col_[0] ^ (uint32_t)(db << 6) ^ (jj ? kNext8 : 0u);
      q[jj] = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4f16(
                                            (lds_pk_h4*)(tile + (32 * st + 16 * ks + 8 * jj) * 2 * D + o)));
    }
    return make_uint4(q[0].x, q[0].y, q[1].x, q[1].y);
  }
};

// Runs tiles 0..ntk - 1 in turn, the first nfull of them as tile(integral_constant 0, ...), the others as
// (1, ...) (their entries need a mask), alternating between two buffers (an even tile in buffer 0).
template <typename F>
__device__ __forceinline__ void pk_tiles(int ntk, int nfull, F&& tile) {
  int n = 0;
#pragma unroll 1
  for (; n + 1 < nfull; n += 2) {
    tile(PkInt<0>{}, PkInt<0>{}, n);
    tile(PkInt<0>{}, PkInt<1>{}, n + 1);
  }
#pragma unroll 1
  for (; n + 1 < ntk; n += 2) {
    tile(PkInt<1>{}, PkInt<0>{}, n);
    tile(PkInt<1>{}, PkInt<1>{}, n + 1);
  }
  if (n < ntk) tile(PkInt<1>{}, PkInt<0>{}, n);
}

// A running reference m of the softmax: weights are 2^(s - m), rounded to the 16-bit type for the second
// product. fp16's smallest step is 2^-24, so with the largest score as the reference what lies 25 octaves below it
// would be 0 in the product while the sum keeps it (43,968 keys that far below one with v = 0: o = 0 for
// 1.2e-3). Its reference lies 10 octaves below the largest score: a weight keeps all its bits down to 2^-24 of the
// largest, and a smaller one is off by at most 2^-35 of the largest. bf16 has the exponents of fp32. A lane whose
// weights of a step (8 or 16) sum past the cap raises m, so no weight leaves fp16's range.
template <typename E>
constexpr float kPkBelow = __is_same(E, FP16) ? 10.f : 0.f;
template <typename E>
constexpr float kPkSumCap = __is_same(E, FP16) ? 60000.f : 32768.f;

// inf and NaN in places that a row does not see. A masked weight is 0, but 0 * inf is NaN: in tiles
// that some rows see only in part, inf and NaN among the second operand's entries are cleared before the
// product, and once it is known that there were any (never, in healthy data), a pass over those tiles
// adds them to the rows that do see them. Entries of V and dO meet weights (ZERO false: the entries are added); K
// and Q meet dS, where a row or key that sees such an entry has a NaN dS or, its score -inf, a dS of 0, and 0 * inf
// is NaN (ZERO true: NaN is added).
template <typename E>
constexpr uint32_t kPkExp = __is_same(E, FP16) ? 0x7C00u : 0x7F80u;

template <typename E>
__device__ __forceinline__ bool pk_not_finite(uint32_t half) { return (half & kPkExp<E>) == kPkExp<E>; }

// Bits 15 and 31 tell whether the low and the high half are not finite: a full exponent and one more of its
// units carry into the sign's place.
template <typename E>
__device__ __forceinline__ uint32_t pk_not_finite_bits(uint32_t w) {
  return (w & 0x7FFF7FFFu) + (__is_same(E, FP16) ? 0x04000400u : 0x00800080u);
}
template <typename E>
__device__ __forceinline__ uint32_t pk_finite_word(uint32_t w) {
  return (pk_not_finite<E>(w) ? 0u : w & 0xFFFFu) | (pk_not_finite<E>(w >> 16) ? 0u : w & 0xFFFF0000u);
}
// Clears the entries that are not finite; whether there were any in the wave.
template <typename E, int N>
__device__ __forceinline__ bool pk_clear_not_finite(uint4 (&q)[N]) {
  uint32_t any = 0u;
#pragma unroll
  for (int i = 0; i < N; ++i)
    any |= pk_not_finite_bits<E>(q[i].x) | pk_not_finite_bits<E>(q[i].y) | pk_not_finite_bits<E>(q[i].z) |
           pk_not_finite_bits<E>(q[i].w);
  if (__builtin_expect(__builtin_amdgcn_ballot_w64((any & 0x80008000u) != 0u) == 0ull, 1)) return false;
#pragma unroll
  for (int i = 0; i < N; ++i)
    q[i] = make_uint4(pk_finite_word<E>(q[i].x), pk_finite_word<E>(q[i].y), pk_finite_word<E>(q[i].z),
                      pk_finite_word<E>(q[i].w));
  return true;
}
// Adds the entries of a memory row that are not finite to a lane's accumulator entries (dims 32 db + 8 g + 4 half
// + 0..3), where `seen`.
template <typename E, bool ZERO = false, int DB>
__device__ __forceinline__ void pk_add_not_finite(const uint16_t* row, int half, bool seen, f32x16 (&acc)[DB]) {
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const uint2 w = *reinterpret_cast<const uint2*>(row + 32 * db + 8 * g + 4 * half);
      const uint32_t h[4] = {w.x & 0xFFFFu, w.x >> 16, w.y & 0xFFFFu, w.y >> 16};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (seen && pk_not_finite<E>(h[i])) acc[db][4 * g + i] += ZERO ? NAN : in_to_float(__is_same(E, FP16), h[i]);
    }
}

// What rounding a pair of floats to the 16-bit type leaves, in that type again.
template <typename E>
__device__ __forceinline__ uint32_t pk_pair_rest(float a, float b, uint32_t rounded) {
  return pack_pair(E{}, a - in_to_float(__is_same(E, FP16), rounded & 0xFFFFu),
                   b - in_to_float(__is_same(E, FP16), rounded >> 16));
}

// Stores a lane's column of a transposed accumulator (32 dims of one row) scaled by f: lanes l and
// l ^ 32 exchange quads so that each stores eight consecutive dims. REST: what the rounding left goes to
// rest.
template <typename E, bool REST = false>
__device__ __forceinline__ void pk_store_col(uint16_t* row, const f32x16& acc, float f, int half, bool on,
                                             uint16_t* rest = nullptr) {
#pragma unroll
  for (int gp = 0; gp < 2; ++gp) {
    uint32_t w[2][2], l[2][2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int r = 4 * (2 * gp + u);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float x = acc[r + 2 * i] * f, y = acc[r + 2 * i + 1] * f;
        w[u][i] = pack_pair(E{}, x, y);
        if (REST) l[u][i] = pk_pair_rest<E>(x, y, w[u][i]);
      }
    }
    const auto x = __builtin_amdgcn_permlane32_swap(w[0][0], w[1][0], false, false);
    const auto y = __builtin_amdgcn_permlane32_swap(w[0][1], w[1][1], false, false);
    if (on) *reinterpret_cast<uint4*>(row + 8 * (2 * gp + half)) = make_uint4(x[0], y[0], x[1], y[1]);
    if constexpr (REST) {
      const auto z = __builtin_amdgcn_permlane32_swap(l[0][0], l[1][0], false, false);
      const auto t = __builtin_amdgcn_permlane32_swap(l[0][1], l[1][1], false, false);
      if (on) *reinterpret_cast<uint4*>(rest + 8 * (2 * gp + half)) = make_uint4(z[0], t[0], z[1], t[1]);
    }
  }
}

// Four dims of an output row, and what their rounding left (rest, nullable).
template <typename E>
__device__ __forceinline__ void pk_store4(uint16_t* row, uint16_t* rest, float a, float b, float c, float d) {
  const uint32_t x = pack_pair(E{}, a, b), y = pack_pair(E{}, c, d);
  *reinterpret_cast<uint2*>(row) = make_uint2(x, y);
  if (rest) *reinterpret_cast<uint2*>(rest) = make_uint2(pk_pair_rest<E>(a, b, x), pk_pair_rest<E>(c, d, y));
}

// Waits for this wave's LDS accesses only (loads stay in flight), then for the other waves.
__device__ __forceinline__ void pk_lds_barrier() {
  __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Waits for this wave's loads and LDS accesses, then for the other waves.
__device__ __forceinline__ void pk_tile_barrier() {
  __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

}  // namespace
}  // namespace gw
