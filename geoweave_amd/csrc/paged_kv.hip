// Writing new tokens' keys and values into a paged cache, k (and q) rotated on the way, and reading sequences back as
// packed rows (gfx950). The cache holds 16-bit rows or 4-bit ones (gw_fp4.h). D = 64 or 128.
//
// New token i of a sequence's N is key lens - N + i; key j lies in slot j % page of page table[j / page]. A token
// whose key has no slot (negative, behind the table, a page outside the pool) is written nowhere; its q is turned.
// The rotation is that of rotary_axes.hip: angles in 64 bits, products and sums in fp32, each rounded once (no fused
// multiply-add: so the 4-bit codes of k are those of the same steps taken one by one).
//
// Bound by memory: rows are read and written once, 16 bytes (eight dims) per thread. A workgroup takes TT tokens, a power
// of two. A thread keeps one token and eight dims of a row and walks over the heads, so that its slot, its
// cosines and sines (formed once for all heads, in LDS) and its addresses stay in registers; a wave's rows are
// neighbouring tokens of one head, which lie one behind the other in a head-major cache (4 bits: 32 bytes a row). The partners of
// its dims come from the wave's own copy of its rows in LDS, W at a time (W: the widest of 8, 4, 2, 1 that divides every half
// block). 4 bits: the 32 values of a power of two lie in four neighbouring lanes, which exchange their largest
// within the vector unit.
//
// Measured (kernels alone): 19,000 tokens of 24 scenes, q, k and v of 16 heads of 64, into 16 bits 30 us, 5.2 TB/s, what a
// large copy reaches; 28,980 tokens, 16 + 4 + 4 heads of 128, four axes of odd halves (W = 1) 80 to 83 us, 4.4 TB/s; 50,160
// tokens, 16 heads of 64, into 4 bits 74 to 80 us, 3.4 TB/s, the vector unit 75 % busy. The rows of all heads one
// behind the other (token by token), with selects that the compiler made loads of: 159 us. Reading back: 41 us from 4 bits (5.8 TB/s, part
// of it from the last-level cache), 88,036 tokens of 4 heads of 128 from 16 bits 61 to 65 us.
// Moving addresses instead of one product per row: 128.5 for 131 us of the 4-bit pass with its reading, but 5.2 for 4.8 us of
// 64 single tokens.
#include <math.h>
#include <string.h>

#include "gw_fp4.h"
#include "gw_mma.h"
#include "gw_rotary.h"

namespace gw {
namespace {

constexpr int kKvThreads = 256;
constexpr int kKvLogTokens = 3;   // tokens of a workgroup: up to 8
constexpr int kKvMaxTokens = 1 << kKvLogTokens;
constexpr int kKvUnroll = 4;     // rows of a thread whose loads are in flight together
constexpr int kKvMaxPairs = 64;

struct KvCache {
  uint8_t* rows;    // 16-bit rows or codes
  uint8_t* scales;  // 4 bits: a byte per 32 dims
  int64_t page, slot, head;     // strides in bytes
  int64_t spage, sslot, shead;  // of the scales
};

struct KvTable {
  const int32_t* table;
  const int32_t* lens;
  const int32_t* cu;  // nullable: packed tokens
  int64_t stride;
  int width, pages, page;
  int n, N, T;  // sequences, tokens of each (not packed), tokens in all
};

struct KvIn {
  const uint16_t* x;
  int64_t sb, st, sh;
};

struct KvAppendParams {
  KvIn in[3];  // q, k, v
  uint16_t* q_out;
  KvCache cache[2];
  KvTable t;
  const void* pos;
  int64_t pb, pt, pa;
  int pos_type;
  int Hq, Hk, D, pairs;
  int TT;  // log2 of a workgroup's tokens
  double freq[kKvMaxPairs];
  uint8_t axis[kKvMaxPairs];
  int8_t dim_pair[2 * kKvMaxPairs], dim_other[2 * kKvMaxPairs];  // a dim's pair, distance to its partner (0: not turned)
};

struct KvReadParams {
  KvCache cache[2];
  uint16_t* out[2];  // k, v: [T][Hk][D]
  KvTable t;
  int Hk, D, TT;  // TT: as above
};

// The sequence of packed token t: the last whose bound is not above t (64 bounds a step), by one wave.
__device__ __forceinline__ int kv_sequence(const int32_t* cu, int n, int t, int lane) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int step = (hi - lo + 63) / 64;
    const int at = lo + lane * step;
    const uint64_t le = __builtin_amdgcn_ballot_w64(at < hi && cu[min(at, n)] <= t);
    const int l = le ? 63 - __builtin_clzll(le) : 0;
    lo += l * step;
    hi = min(hi, lo + step);
  }
  return lo;
}

// (page, slot) of key `key` of sequence seq; page -1: none.
__device__ __forceinline__ int2 kv_slot(const KvTable& t, int seq, int64_t key) {
  if (key < 0 || key >= (int64_t)t.width * t.page) return make_int2(-1, 0);
  const int pg = (int)key / t.page;
  const int id = t.table[(int64_t)seq * t.stride + pg];
  return make_int2((uint32_t)id < (uint32_t)t.pages ? id : -1, (int)key - pg * t.page);
}

// A token's rows in a cache.
struct KvRows {
  uint8_t* rows;
  uint8_t* scales;
};
template <bool FP4>
__device__ __forceinline__ KvRows kv_rows(const KvCache& c, int2 at) {
  return KvRows{c.rows + at.x * c.page + at.y * c.slot, FP4 ? c.scales + at.x * c.spage + at.y * c.sslot : nullptr};
}

// W consecutive 16-bit values as floats.
template <typename E, int W>
__device__ __forceinline__ void kv_floats(const uint8_t* at, float* f) {
  if constexpr (W == 8) {
    unpack8<E>(*reinterpret_cast<const uint4*>(at), f);
  } else if constexpr (W == 4) {
    const uint2 x = *reinterpret_cast<const uint2*>(at);
    unpack2(E{}, x.x, f[0], f[1]);
    unpack2(E{}, x.y, f[2], f[3]);
  } else if constexpr (W == 2) {
    unpack2(E{}, *reinterpret_cast<const uint32_t*>(at), f[0], f[1]);
  } else {
    f[0] = ld_f32(E{}, at, 0);
  }
}

__device__ __forceinline__ uint32_t kv_quad_max(uint32_t x) {
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, kDppXor1, 0xF, 0xF, true));
  return max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, kDppXor2, 0xF, 0xF, true));
}

// First token of a workgroup. Workgroups go to the eight XCDs in turn; in 4 bits each XCD takes a run of neighbouring
// tokens, so that lines which several workgroups write in part (the scales of 64 slots are one) are put together in one
// L2 (six scenes of 16 heads of 64 into 4 bits and back: 134 -> 131 us; whole lines of 16 bits lose 1 % by it).
template <bool FP4>
__device__ __forceinline__ int kv_first_token(int TT) {
  return (FP4 ? (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3) : blockIdx.x) << TT;
}

template <typename E, bool FP4, int W>
__global__ __launch_bounds__(kKvThreads) void kv_append_kernel(const KvAppendParams p) {
  __shared__ float2 cs[kKvMaxTokens * kKvMaxPairs];
  __shared__ int2 where[kKvMaxTokens];
  __shared__ __align__(16) uint8_t rows_s[kKvThreads / 64][kKvUnroll * 64 * 16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int t0 = kv_first_token<FP4>(p.TT), nt = min(1 << p.TT, p.t.T - t0);
  if (nt <= 0) return;
  const int H0 = p.Hq, H1 = p.Hq + p.Hk, HT = p.Hq + 2 * p.Hk;
  const int C = p.D >> 3, shift = p.D == 64 ? 3 : 4;
  const int c = threadIdx.x & (C - 1), r0 = threadIdx.x >> shift;
  const int tok = r0 & ((1 << p.TT) - 1);  // this thread's token
  const int R = (kKvThreads >> shift) >> p.TT;  // heads of a round
  const int step = R * gridDim.y;
  int head = (r0 >> p.TT) + R * blockIdx.y;
  if (tok >= nt) head = HT;  // nothing to do

  const int t = t0 + min(tok, nt - 1);
  const int b = p.t.N ? t / p.t.N : 0, i_in_b = t - b * p.t.N;
  // What differs between q, k and v is held in registers and selected: an index into the arguments would be a load.
  auto row_of = [&](const KvIn& in) __attribute__((always_inline)) { return in.x + b * in.sb + i_in_b * in.st + c * 8; };
  const uint16_t *const q_row = row_of(p.in[0]), *const k_row = row_of(p.in[1]), *const v_row = row_of(p.in[2]);
  const uint64_t q_head = p.in[0].sh, k_head = p.in[1].sh, v_head = p.in[2].sh;
  uint4 x[kKvUnroll];
  auto load = [&](uint4(&to)[kKvUnroll], int first) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < kKvUnroll; ++u) {
      const int h = first + u * step;
      const uint16_t* base = h < H0 ? q_row : h < H1 ? k_row : v_row;
      const uint64_t sh = h < H0 ? q_head : h < H1 ? k_head : v_head;
      if (h < HT) to[u] = *reinterpret_cast<const uint4*>(base + (uint32_t)(h - (h < H0 ? 0 : h < H1 ? H0 : H1)) * sh);
    }
  };
  load(x, head);

  // Slots of the tokens, a wave each; angles by all threads.
  for (int i = wave; i < nt; i += kKvThreads / 64) {
    int2 at = make_int2(-1, 0);
    if (p.t.n > 0) {
      int seq;
      int64_t first, count = p.t.N;
      if (p.t.cu) {
        seq = kv_sequence(p.t.cu, p.t.n, t0 + i, lane);
        first = p.t.cu[seq];
        count = p.t.cu[seq + 1] - first;
      } else {
        seq = (t0 + i) / p.t.N;
        first = (int64_t)seq * p.t.N;
      }
      const int64_t in = t0 + i - first;
      if (in >= 0 && in < count) at = kv_slot(p.t, seq, p.t.lens[seq] - count + in);
    }
    if (lane == 0) where[i] = at;
  }
  for (int i = threadIdx.x; i < nt * p.pairs; i += kKvThreads) {
    const int tk = i / p.pairs, pr = i - tk * p.pairs;
    const int tt = t0 + tk, bb = p.t.N ? tt / p.t.N : 0;
    const double pos = rot_position(p.pos, p.pos_type, bb * p.pb + (int64_t)(tt - bb * p.t.N) * p.pt + p.axis[pr] * p.pa);
    cs[tk * p.pairs + pr] = rot_cos_sin(pos * p.freq[pr], 1.0);
  }
  __syncthreads();

  const int2 at = where[tok < nt ? tok : 0];
  const KvRows k_to = kv_rows<FP4>(p.cache[0], at), v_to = kv_rows<FP4>(p.cache[1], at);
  const uint64_t k_step = p.cache[0].head, v_step = p.cache[1].head, ks_step = p.cache[0].shead, vs_step = p.cache[1].shead;
  // This thread's dims by W: where the partners lie (0: not turned), cosines, and sines with the partner's sign.
  int other[8 / W];
  float co[8], si[8];
#pragma unroll
  for (int i = 0; i < 8 / W; ++i) {
    other[i] = p.dim_other[c * 8 + i * W];
    const int pair = p.dim_pair[c * 8 + i * W];
#pragma unroll
    for (int j = 0; j < W; ++j) {
      const float2 a = other[i] ? cs[(tok < nt ? tok : 0) * p.pairs + pair + j] : make_float2(1.f, 0.f);
      co[i * W + j] = a.x;
      si[i * W + j] = other[i] > 0 ? -a.y : a.y;
    }
  }

  uint8_t* const mine = rows_s[wave];
  const int turns = (HT + step * kKvUnroll - 1) / (step * kKvUnroll);  // the same for every thread
  for (int n = 0; n < turns; ++n) {
    uint4 next[kKvUnroll];
    load(next, head + step * kKvUnroll);
#pragma unroll
    for (int u = 0; u < kKvUnroll; ++u) *reinterpret_cast<uint4*>(mine + (u * 64 + lane) * 16) = x[u];
    lds_fence();
#pragma unroll
    for (int u = 0; u < kKvUnroll; ++u) {
      const int h = head + u * step;
      if (h >= HT) continue;
      float y[8];
      unpack8<E>(x[u], y);
      if (h < H1) {
#pragma unroll
        for (int i = 0; i < 8 / W; ++i) {
          if (other[i] == 0) continue;
          float o[W];
          kv_floats<E, W>(mine + (u * 64 + lane) * 16 + (i * W + other[i]) * 2, o);
#pragma unroll
          for (int j = 0; j < W; ++j) {
#pragma clang fp contract(off)
            const float a = y[i * W + j] * co[i * W + j], d = o[j] * si[i * W + j];
            y[i * W + j] = a + d;
          }
        }
      }
      if (h < H0) {
        *reinterpret_cast<uint4*>(p.q_out + ((int64_t)t * H0 + h) * p.D + c * 8) = pack_quad<E>(y);
        continue;
      }
      if (at.x < 0) continue;
      const bool is_v = h >= H1;
      const uint32_t hk = h - (is_v ? H1 : H0);
      uint8_t* dst = (is_v ? v_to.rows : k_to.rows) + hk * (is_v ? v_step : k_step);
      if constexpr (FP4) {
        uint32_t top = 0u;
#pragma unroll
        for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(y[j]) & 0x7fffffffu);
        const uint32_t scale = fp4_scale(kv_quad_max(top));
        reinterpret_cast<uint32_t*>(dst)[c] = scale == kFp4NaN ? 0u : fp4_pack8(y, scale);
        if ((c & 3) == 0) ((is_v ? v_to.scales : k_to.scales) + hk * (is_v ? vs_step : ks_step))[c >> 2] = (uint8_t)scale;
      } else {
        reinterpret_cast<uint4*>(dst)[c] = is_v ? x[u] : pack_quad<E>(y);
      }
    }
    lds_fence();
    head += step * kKvUnroll;
#pragma unroll
    for (int u = 0; u < kKvUnroll; ++u) x[u] = next[u];
  }
}

// Sequence b's keys 0 .. cu[b + 1] - cu[b] - 1 to rows cu[b] .. of k and v; rows without a slot are zeros.
template <typename E, bool FP4>
__global__ __launch_bounds__(kKvThreads) void kv_read_kernel(const KvReadParams p) {
  __shared__ int2 where[kKvMaxTokens];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int t0 = kv_first_token<FP4>(p.TT), nt = min(1 << p.TT, p.t.T - t0);
  if (nt <= 0) return;
  const int HT = 2 * p.Hk, shift = p.D == 64 ? 3 : 4;
  const int c = threadIdx.x & ((p.D >> 3) - 1), r0 = threadIdx.x >> shift;
  const int tok = r0 & ((1 << p.TT) - 1);
  const int R = (kKvThreads >> shift) >> p.TT, step = R * gridDim.y;
  for (int i = wave; i < nt; i += kKvThreads / 64) {
    int2 at = make_int2(-1, 0);
    if (p.t.n > 0) {
      const int t = t0 + i, seq = kv_sequence(p.t.cu, p.t.n, t, lane);
      const int first = p.t.cu[seq], end = p.t.cu[seq + 1];
      if (t >= first && t < end) at = kv_slot(p.t, seq, (int64_t)t - first);
    }
    if (lane == 0) where[i] = at;
  }
  __syncthreads();
  if (tok >= nt) return;
  const int2 at = where[tok];
  const KvRows k_from = kv_rows<FP4>(p.cache[0], at), v_from = kv_rows<FP4>(p.cache[1], at);
  const uint64_t k_step = p.cache[0].head, v_step = p.cache[1].head, ks_step = p.cache[0].shead, vs_step = p.cache[1].shead;
  uint16_t *const k_out = p.out[0], *const v_out = p.out[1];
  const int64_t to = (int64_t)(t0 + tok) * p.Hk * p.D + c * 8;
  for (int head = (r0 >> p.TT) + R * blockIdx.y; head < HT; head += step * kKvUnroll) {
    uint4 x[kKvUnroll];
    uint32_t s[kKvUnroll];
#pragma unroll
    for (int u = 0; u < kKvUnroll; ++u) {
      const int h = head + u * step;
      const bool is_v = h >= p.Hk;
      x[u] = make_uint4(0u, 0u, 0u, 0u);
      s[u] = 0u;
      if (h < HT && at.x >= 0) {
        const uint32_t hk = h - (is_v ? p.Hk : 0);
        const uint8_t* src = (is_v ? v_from.rows : k_from.rows) + hk * (is_v ? v_step : k_step);
        if constexpr (FP4) {
          x[u].x = reinterpret_cast<const uint32_t*>(src)[c];
          s[u] = ((is_v ? v_from.scales : k_from.scales) + hk * (is_v ? vs_step : ks_step))[c >> 2];
        } else {
          x[u] = reinterpret_cast<const uint4*>(src)[c];
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kKvUnroll; ++u) {
      const int h = head + u * step;
      if (h >= HT) continue;
      uint16_t* dst = (h >= p.Hk ? v_out + (h - p.Hk) * p.D : k_out + h * p.D) + to;
      *reinterpret_cast<uint4*>(dst) = FP4 ? fp4_operand<E>(x[u].x, fp4_unit(s[u])) : x[u];
    }
  }
}

// ---------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------

// Workgroups along x and y, and the logarithm of a workgroup's tokens: few tokens a workgroup until the chip has four
// workgroups per CU, and where the tokens are too few for that, a token's heads over several (each forms the angles again).
dim3 kv_grid(int64_t T, int64_t heads, int64_t D, int* TT) {
  *TT = kKvLogTokens;
  while (*TT > 0 && ((T - 1) >> *TT) + 1 < 1024) --*TT;
  const int64_t x = ((((T - 1) >> *TT) >> 3) + 1) * 8, per = (kKvThreads / (D / 8) >> *TT) * kKvUnroll;  // a multiple of 8
  int64_t y = (heads + per - 1) / per;
  if (y > 1024 / x) y = 1024 / x > 0 ? 1024 / x : 1;
  return dim3((uint32_t)x, (uint32_t)y);
}

int kv_check_cache(const char* what, int format, int64_t D, const void* rows, const int64_t* strides, const void* scales,
                   const int64_t* scale_strides, int64_t pages, KvCache* out) {
  const int64_t per = D / 32;  // bytes of a row's scales
  GW_CHECK_ARG(strides && (rows || pages == 0), "the %s cache is missing", what);
  const int64_t unit = format == GW_CACHE_FP4 ? 1 : 2;
  GW_CHECK_ARG(aligned16(rows) && strides[0] * unit % 16 == 0 && strides[1] * unit % 16 == 0 && strides[2] * unit % 16 == 0,
               "the %s cache needs 16-byte aligned rows", what);
  *out = KvCache{const_cast<uint8_t*>(static_cast<const uint8_t*>(rows)), nullptr, strides[0] * unit, strides[1] * unit,
                 strides[2] * unit, 0, 0, 0};
  if (format != GW_CACHE_FP4) return GW_OK;
  GW_CHECK_ARG(scale_strides && (scales || pages == 0), "the %s cache's scales are missing", what);
  GW_CHECK_ARG(reinterpret_cast<uintptr_t>(scales) % per == 0 && scale_strides[0] % per == 0 &&
                   scale_strides[1] % per == 0 && scale_strides[2] % per == 0,
               "the %s cache's scales need rows aligned to their %lld bytes", what, (long long)per);
  out->scales = const_cast<uint8_t*>(static_cast<const uint8_t*>(scales));
  out->spage = scale_strides[0];
  out->sslot = scale_strides[1];
  out->shead = scale_strides[2];
  return GW_OK;
}

int kv_check_sizes(int format, int64_t D, int64_t n, int64_t T, int64_t heads, int64_t Hk, int64_t pages,
                   int64_t page_size, int64_t table_width, const int32_t* block_table) {
  GW_CHECK_ARG(format == GW_CACHE_16BIT || format == GW_CACHE_FP4, "unknown cache format %d", format);
  if (D != 64 && D != 128) return set_error(GW_ERR_UNSUPPORTED, "head dim %lld is not 64 or 128", (long long)D);
  GW_CHECK_ARG(n >= 0 && T >= 0 && pages >= 0 && table_width >= 0, "negative size");
  GW_CHECK_ARG(Hk >= 1, "%lld key heads", (long long)Hk);
  GW_CHECK_ARG(page_size >= 1 && page_size < (1ll << 31) && pages < (1ll << 31), "page size %lld, pages %lld",
               (long long)page_size, (long long)pages);
  if (heads > (1ll << 20) || T > 0x7FFFF000ll / heads || n >= (1ll << 30) || table_width > 0x7FFFF000ll / page_size)
    return set_error(GW_ERR_UNSUPPORTED, "tokens x heads and keys of a sequence must stay below 2^31 - 2^12, heads below 2^20");
  GW_CHECK_ARG(block_table || table_width == 0 || n == 0, "the block table is missing");
  return GW_OK;
}

template <typename E, bool FP4>
int kv_append_launch(const KvAppendParams& p, int W, dim3 grid, hipStream_t s) {
  switch (W) {
    case 8: hipLaunchKernelGGL((kv_append_kernel<E, FP4, 8>), grid, dim3(kKvThreads), 0, s, p); break;
    case 4: hipLaunchKernelGGL((kv_append_kernel<E, FP4, 4>), grid, dim3(kKvThreads), 0, s, p); break;
    case 2: hipLaunchKernelGGL((kv_append_kernel<E, FP4, 2>), grid, dim3(kKvThreads), 0, s, p); break;
    default: hipLaunchKernelGGL((kv_append_kernel<E, FP4, 1>), grid, dim3(kKvThreads), 0, s, p); break;
  }
  GW_HIP_LAUNCH_CHECK("gw_paged_kv_append");
  return GW_OK;
}

}  // namespace
}  // namespace gw

extern "C" int gw_paged_kv_append(int dtype, const void* q, const int64_t* q_strides, void* q_out, int64_t Hq,
                                  const void* k, const int64_t* k_strides, const void* v, const int64_t* v_strides,
                                  int64_t Hk, int64_t D, int cache_format, void* k_cache, const int64_t* k_cache_strides,
                                  void* k_scales, const int64_t* k_scale_strides, void* v_cache,
                                  const int64_t* v_cache_strides, void* v_scales, const int64_t* v_scale_strides,
                                  const int32_t* block_table, int64_t table_stride, const int32_t* lens,
                                  const int32_t* cu_new, int64_t n, int64_t N, int64_t pages, int64_t page_size,
                                  int64_t table_width, int pos_type, const void* pos, const int64_t* pos_strides,
                                  int n_axes, const int32_t* axis_dims, const double* bases, void* stream) {
  using namespace gw;
  clear_error();
  GW_CHECK_ARG(dtype == GW_DTYPE_BF16 || dtype == GW_DTYPE_FP16, "unknown dtype %d", dtype);
  GW_CHECK_ARG(N >= 0 && n >= 0 && Hq >= 0, "negative size");
  GW_CHECK_ARG(Hk >= 1 && Hq <= (1ll << 20) && Hk <= (1ll << 19), "%lld query heads, %lld key heads", (long long)Hq, (long long)Hk);
  if (!cu_new && N > 0 && n > 0x7FFFF000ll / N)
    return set_error(GW_ERR_UNSUPPORTED, "%lld sequences of %lld tokens", (long long)n, (long long)N);
  const int64_t T = cu_new ? N : n * N;
  int rc = kv_check_sizes(cache_format, D, n, T, Hq + 2 * Hk, Hk, pages, page_size, table_width, block_table);
  if (rc != GW_OK) return rc;
  GW_CHECK_ARG(n_axes >= 0 && n_axes <= kRotMaxAxes && (n_axes == 0 || (axis_dims && bases)), "0 to %d axes, got %d",
               kRotMaxAxes, n_axes);
  KvAppendParams p = {};
  int turned = 0, W = 8;
  for (int a = 0; a < n_axes; ++a) {
    GW_CHECK_ARG(axis_dims[a] >= 0 && axis_dims[a] % 2 == 0, "axis %d has %d dims: an even number is needed", a, axis_dims[a]);
    GW_CHECK_ARG(bases[a] > 0 && isfinite(bases[a]), "axis %d: the base must be positive and finite", a);
    GW_CHECK_ARG(axis_dims[a] <= D - turned, "the axes' dims exceed the head dim %lld", (long long)D);
    const int half = axis_dims[a] / 2;
    while (half % W) W >>= 1;
    for (int i = 0; i < axis_dims[a]; ++i) {
      p.dim_pair[turned + i] = (int8_t)(turned / 2 + (i < half ? i : i - half));
      p.dim_other[turned + i] = (int8_t)(i < half ? half : -half);
    }
    for (int i = 0; i < half; ++i) p.axis[turned / 2 + i] = (uint8_t)a;
    turned += axis_dims[a];
  }
  if (T == 0) return GW_OK;
  GW_CHECK_ARG(k && v && k_strides && v_strides && (Hq == 0 || (q && q_out && q_strides)), "a tensor is missing");
  GW_CHECK_ARG(lens || n == 0, "the lengths are missing");
  GW_CHECK_ARG(turned == 0 || (pos && pos_strides), "positions are missing");
  GW_CHECK_ARG(pos_type == GW_POS_INT32 || pos_type == GW_POS_INT64 || pos_type == GW_POS_FP32,
               "unknown position type %d", pos_type);
  const void* in[3] = {q, k, v};
  const int64_t* st[3] = {q_strides, k_strides, v_strides};
  for (int i = Hq == 0 ? 1 : 0; i < 3; ++i) {
    GW_CHECK_ARG(aligned16(in[i]) && st[i][0] % 8 == 0 && st[i][1] % 8 == 0 && st[i][2] % 8 == 0,
                 "q, k and v need 16-byte aligned rows");
    p.in[i] = KvIn{static_cast<const uint16_t*>(in[i]), st[i][0], st[i][1], st[i][2]};
  }
  GW_CHECK_ARG(aligned16(q_out), "the turned q needs 16-byte aligned rows");
  rc = kv_check_cache("key", cache_format, D, k_cache, k_cache_strides, k_scales, k_scale_strides, pages, &p.cache[0]);
  if (rc == GW_OK)
    rc = kv_check_cache("value", cache_format, D, v_cache, v_cache_strides, v_scales, v_scale_strides, pages, &p.cache[1]);
  if (rc != GW_OK) return rc;
  p.q_out = static_cast<uint16_t*>(q_out);
  p.t = KvTable{block_table, lens, cu_new, table_stride, pages == 0 ? 0 : (int)table_width, (int)pages, (int)page_size, (int)n, cu_new ? 0 : (int)N,
                (int)T};
  p.pos = pos;
  p.pos_type = pos_type;
  if (turned) {
    p.pb = pos_strides[0];
    p.pt = pos_strides[1];
    p.pa = pos_strides[2];
    memcpy(p.freq, rot_freqs(n_axes, axis_dims, bases), turned / 2 * sizeof(double));
  }
  p.Hq = (int)Hq;
  p.Hk = (int)Hk;
  p.D = (int)D;
  p.pairs = turned / 2;
  const dim3 grid = kv_grid(T, Hq + 2 * Hk, D, &p.TT);
  GW_CHECK_GRID(grid.x, kKvThreads);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool fp4 = cache_format == GW_CACHE_FP4;
  if (dtype == GW_DTYPE_BF16) return fp4 ? kv_append_launch<BF16, true>(p, W, grid, s) : kv_append_launch<BF16, false>(p, W, grid, s);
  return fp4 ? kv_append_launch<FP16, true>(p, W, grid, s) : kv_append_launch<FP16, false>(p, W, grid, s);
}

extern "C" int gw_paged_kv_read(int dtype, int cache_format, const void* k_cache, const int64_t* k_cache_strides,
                                const void* k_scales, const int64_t* k_scale_strides, const void* v_cache,
                                const int64_t* v_cache_strides, const void* v_scales, const int64_t* v_scale_strides,
                                const int32_t* block_table, int64_t table_stride, const int32_t* cu, int64_t n,
                                int64_t tokens, int64_t Hk, int64_t D, int64_t pages, int64_t page_size,
                                int64_t table_width, void* k_out, void* v_out, void* stream) {
  using namespace gw;
  clear_error();
  GW_CHECK_ARG(dtype == GW_DTYPE_BF16 || dtype == GW_DTYPE_FP16, "unknown dtype %d", dtype);
  GW_CHECK_ARG(Hk >= 1 && Hk <= (1ll << 19), "%lld key heads", (long long)Hk);
  int rc = kv_check_sizes(cache_format, D, n, tokens, 2 * Hk, Hk, pages, page_size, table_width, block_table);
  if (rc != GW_OK) return rc;
  if (tokens == 0) return GW_OK;
  GW_CHECK_ARG(k_out && v_out, "a tensor is missing");
  GW_CHECK_ARG(cu || n == 0, "the bounds are missing");
  GW_CHECK_ARG(aligned16(k_out) && aligned16(v_out), "k and v need 16-byte aligned rows");
  KvReadParams p = {};
  rc = kv_check_cache("key", cache_format, D, k_cache, k_cache_strides, k_scales, k_scale_strides, pages, &p.cache[0]);
  if (rc == GW_OK)
    rc = kv_check_cache("value", cache_format, D, v_cache, v_cache_strides, v_scales, v_scale_strides, pages, &p.cache[1]);
  if (rc != GW_OK) return rc;
  p.out[0] = static_cast<uint16_t*>(k_out);
  p.out[1] = static_cast<uint16_t*>(v_out);
  p.t = KvTable{block_table, nullptr, cu, table_stride, pages == 0 ? 0 : (int)table_width, (int)pages, (int)page_size, (int)n, 0, (int)tokens};
  p.Hk = (int)Hk;
  p.D = (int)D;
  const dim3 grid = kv_grid(tokens, 2 * Hk, D, &p.TT);
  GW_CHECK_GRID(grid.x, kKvThreads);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (cache_format != GW_CACHE_FP4) {
    hipLaunchKernelGGL((kv_read_kernel<BF16, false>), grid, dim3(kKvThreads), 0, s, p);
  } else if (dtype == GW_DTYPE_BF16) {
    hipLaunchKernelGGL((kv_read_kernel<BF16, true>), grid, dim3(kKvThreads), 0, s, p);
  } else {
    hipLaunchKernelGGL((kv_read_kernel<FP16, true>), grid, dim3(kKvThreads), 0, s, p);
  }
  GW_HIP_LAUNCH_CHECK("gw_paged_kv_read");
  return GW_OK;
}
