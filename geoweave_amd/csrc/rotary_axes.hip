// Rotary positions with several axes (gfx950): query and key heads turned in one pass.
//
// The first sum(axis_dims) dims of a head are blocks, one per axis a, of d_a dims (even); dims i
// and i + d_a / 2 of a block (i < d_a / 2) are a point turned by the angle
// pos_a * base_a^(-2 i / d_a):  y1 = x1 cos - x2 sin,  y2 = x2 cos + x1 sin. Dims behind the last
// block are copied. The backward is the rotation by the negative angle (inverse = 1).
//
// Angles: turns = pos * base^(-2 i / d) / (2 pi) in 64 bits, less the nearest quarter turn, so a
// position of a million keeps its angle to 1e-10; sine and cosine of the remainder (at most an
// eighth of a turn) by their Taylor series in 64 bits (the first term left out is below 1e-11),
// rounded once to fp32. They are formed once per token and pair, into LDS, and used by all heads of
// q and k. Products and sums are fp32, rounded once to the output's type.
//
// Bound by memory: each element is read and written once. A workgroup takes TT tokens x all
// heads of q and k; a thread keeps one pair group (V pairs: V elements of the first half and V of
// the second) and walks over (token, head) rows, two rows' loads in flight, the first of them issued
// before the angles are formed (the angles cost 1 to 2 us of a pass of 48 views). Eight tokens and two rows in
// flight: 65,952 tokens x 20 heads of 128 in bf16 140 us (4.9 TB/s, what a large copy reaches), 16 tokens and
// four rows 161, four tokens and one row 135; 9,973 tokens x 24 heads of 80 in fp32 53, 70 and 61 us. V is the
// widest of 8, 4, 2, 1 elements that divides every half block and every stride.
#include <math.h>
#include <string.h>

#include "gw_common.h"

namespace gw {
namespace {

constexpr int kRotMaxAxes = 8;
constexpr int kRotMaxPairs = 128;  // D <= 256
constexpr int kRotThreads = 256;
constexpr int kRotMaxTokens = 8;  // tokens of a workgroup
constexpr int kRotUnroll = 2;     // rows of a thread whose loads are in flight together

struct RotTensor {
  const void* x;
  void* y;
  int64_t xb, xt, xh, yb, yt, yh;
  int H;
};

struct RotParams {
  RotTensor t[2];  // the second with H = 0 when there is one tensor only
  const void* pos;
  int64_t pb, pt, pa;
  int pos_type;
  int B, T, TT, D;
  int pairs;   // rotated pairs
  int groups;  // pair groups of a head, the copied tail's included
  double sign;
  double freq[kRotMaxPairs];   // turns per unit of position
  uint8_t axis[kRotMaxPairs];
  // Start of the group's first half, distance to its second, first pair (>= pairs: copied)
  int16_t lo[kRotMaxPairs], half[kRotMaxPairs], pair[kRotMaxPairs];
  // Per dim (staged form): its pair (-1: copied), distance to its partner
  int16_t dim_pair[2 * kRotMaxPairs], dim_other[2 * kRotMaxPairs];
};

template <int BYTES>
struct RotRaw;
template <>
struct RotRaw<2> { typedef uint16_t type; };
template <>
struct RotRaw<4> { typedef uint32_t type; };
template <>
struct RotRaw<8> { typedef uint2 type; };
template <>
struct RotRaw<16> { typedef uint4 type; };

template <typename E, int V>
struct RotVec {
  typename RotRaw<V * ElemBytes<E>::value>::type raw;
  __device__ __forceinline__ float get(int i) const { return ld_f32(E{}, &raw, i); }
  __device__ __forceinline__ void set(int i, float f) { st_f32(E{}, &raw, i, f); }
};

__device__ __forceinline__ double rot_position(const void* pos, int type, int64_t at) {
  if (type == GW_POS_INT32) return (double)static_cast<const int32_t*>(pos)[at];
  if (type == GW_POS_INT64) return (double)static_cast<const int64_t*>(pos)[at];
  return (double)static_cast<const float*>(pos)[at];
}

__device__ __forceinline__ float2 rot_cos_sin(double turns, double sign) {
  const double quarter = rint(turns * 4.0);
  const double t = (turns - quarter * 0.25) * 6.283185307179586476925;  // within +- pi / 4
  const double u = t * t;
  double s = -1.0 / 39916800.0, c = 1.0 / 479001600.0;
  s = fma(s, u, 1.0 / 362880.0);
  s = fma(s, u, -1.0 / 5040.0);
  s = fma(s, u, 1.0 / 120.0);
  s = fma(s, u, -1.0 / 6.0);
  s = fma(s * u, t, t);
  c = fma(c, u, -1.0 / 3628800.0);
  c = fma(c, u, 1.0 / 40320.0);
  c = fma(c, u, -1.0 / 720.0);
  c = fma(c, u, 1.0 / 24.0);
  c = fma(c, u, -0.5);
  c = fma(c, u, 1.0);
  const int k = (int)(quarter - 4.0 * floor(quarter * 0.25));  // 0..3
  double cc = (k & 1) ? s : c, ss = (k & 1) ? c : s;
  if (k == 1 || k == 2) cc = -cc;
  if (k >= 2) ss = -ss;
  return make_float2((float)cc, (float)(sign * ss));
}

// Cosines and sines of nt tokens' pairs into LDS.
__device__ __forceinline__ void rot_angles(const RotParams& p, int b, int t0, int nt, float2* cs) {
  for (int i = threadIdx.x; i < nt * p.pairs; i += kRotThreads) {
    const int tk = i / p.pairs, pr = i - tk * p.pairs;
    const double pos = rot_position(p.pos, p.pos_type, b * p.pb + (int64_t)(t0 + tk) * p.pt + p.axis[pr] * p.pa);
    cs[tk * p.pairs + pr] = rot_cos_sin(pos * p.freq[pr], p.sign);
  }
}

template <typename E, int V>
__global__ __launch_bounds__(kRotThreads) void rotary_axes_kernel(const RotParams p) {
  __shared__ float2 cs[kRotMaxTokens * kRotMaxPairs];
  const int b = blockIdx.y;
  const int t0 = blockIdx.x * p.TT;
  const int nt = min(p.TT, p.T - t0);
  const int H0 = p.t[0].H, HT = H0 + p.t[1].H;
  const int R = kRotThreads / p.groups;  // rows of an iteration
  const int r0 = threadIdx.x / p.groups, g = threadIdx.x - r0 * p.groups;
  const bool on = r0 < R;
  const int lo = p.lo[g], half = p.half[g], pair = p.pair[g];
  const int rows = nt * HT;
  const int step_t = R / HT, step_h = R - step_t * HT;

  int row = r0, tok = r0 / HT, head = r0 - tok * HT;
  RotVec<E, V> x1[kRotUnroll], x2[kRotUnroll];
  int at_tok[kRotUnroll], at_head[kRotUnroll];
  auto addr = [&](const RotTensor& t, int tk, int hd) {
    return static_cast<const typename RotRaw<ElemBytes<E>::value>::type*>(t.x) + b * t.xb + (int64_t)(t0 + tk) * t.xt +
           (int64_t)hd * t.xh + lo;
  };
  auto load = [&](int u) {
    at_tok[u] = tok;
    at_head[u] = head;
    if (on && row < rows) {
      const bool first = head < H0;
      const auto* src = first ? addr(p.t[0], tok, head) : addr(p.t[1], tok, head - H0);
      x1[u] = *reinterpret_cast<const RotVec<E, V>*>(src);
      x2[u] = *reinterpret_cast<const RotVec<E, V>*>(src + half);
    } else {
      at_tok[u] = -1;
    }
    row += R;
    tok += step_t;
    head += step_h;
    if (head >= HT) {
      head -= HT;
      ++tok;
    }
  };
#pragma unroll
  for (int u = 0; u < kRotUnroll; ++u) load(u);

  rot_angles(p, b, t0, nt, cs);
  __syncthreads();

  while (true) {
    bool any = false;
#pragma unroll
    for (int u = 0; u < kRotUnroll; ++u) {
      if (at_tok[u] < 0) continue;
      any = true;
      const bool first = at_head[u] < H0;
      const RotTensor& t = first ? p.t[0] : p.t[1];
      auto* dst = static_cast<typename RotRaw<ElemBytes<E>::value>::type*>(t.y) + b * t.yb +
                  (int64_t)(t0 + at_tok[u]) * t.yt + (int64_t)(at_head[u] - (first ? 0 : H0)) * t.yh + lo;
      RotVec<E, V> y1 = x1[u], y2 = x2[u];
      if (pair < p.pairs) {
        const float2* c = cs + at_tok[u] * p.pairs + pair;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float a = x1[u].get(i), d = x2[u].get(i);
          const float co = c[i].x, si = c[i].y;
          y1.set(i, a * co - d * si);
          y2.set(i, d * co + a * si);
        }
      }
      *reinterpret_cast<RotVec<E, V>*>(dst) = y1;
      *reinterpret_cast<RotVec<E, V>*>(dst + half) = y2;
    }
    if (!any || row >= rows) break;
#pragma unroll
    for (int u = 0; u < kRotUnroll; ++u) load(u);
  }
}

// ---------------------------------------------------------------------------------------
// Blocks whose halves are not whole 16-byte (8-byte for the 16-bit types) groups: a wave reads whole
// rows 16 bytes at a time, keeps them in its own LDS rows, and each thread fetches the partners of its
// elements from there, wherever they lie. No barrier: a wave's LDS accesses are in order. 9,973 tokens x
// 24 heads of 80 in fp32 by blocks of 18, 14, 20, 20: 53 to 60 us (2.6 to 2.9 TB/s; 39 where the last-level cache
// still holds the inputs), bound by the reads of single partners, pairs and angles from LDS; pairs of single elements
// took 78 us where rows through LDS took 70 (both with four rows in flight).
// ---------------------------------------------------------------------------------------
template <typename E>
__global__ __launch_bounds__(kRotThreads) void rotary_staged_kernel(const RotParams p) {
  constexpr int V = 16 / ElemBytes<E>::value;
  typedef typename RotRaw<ElemBytes<E>::value>::type Elem;
  __shared__ float2 cs[kRotMaxTokens * kRotMaxPairs];
  __shared__ __align__(16) uint8_t rows_s[kRotThreads / 64][kRotUnroll * 64 * 16];
  const int b = blockIdx.y, t0 = blockIdx.x * p.TT;
  const int nt = min(p.TT, p.T - t0);
  const int H0 = p.t[0].H, HT = H0 + p.t[1].H;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int C = p.D / V;       // 16-byte chunks of a row, at most 64
  const int RW = 64 / C;       // rows of a wave's load
  const int r0 = lane / C, c = lane - r0 * C;
  const bool on = r0 < RW;
  const int rows = nt * HT;
  const int R = RW * (kRotThreads / 64);
  const int step_t = R / HT, step_h = R - step_t * HT;

  // This thread's elements: where the partner lies in the row, the pair, and the sign of the partner's term.
  int16_t partner[V], pair[V];
  uint32_t minus = 0u;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int d = min(c * V + i, p.D - 1);
    const int pr = p.dim_pair[d];
    pair[i] = (int16_t)pr;
    partner[i] = (int16_t)(pr < 0 ? d : d + p.dim_other[d]);
    if (pr >= 0 && p.dim_other[d] > 0) minus |= 1u << i;
  }

  int row = wave * RW + r0, tok = row / HT, head = row - tok * HT;
  uint4 x[kRotUnroll];
  int at_tok[kRotUnroll], at_head[kRotUnroll];
  auto load = [&](int u) __attribute__((always_inline)) {
    at_tok[u] = on && row < rows ? tok : -1;
    at_head[u] = head;
    if (at_tok[u] >= 0) {
      const bool first = head < H0;
      const RotTensor& t = first ? p.t[0] : p.t[1];
      x[u] = *reinterpret_cast<const uint4*>(static_cast<const Elem*>(t.x) + b * t.xb + (int64_t)(t0 + tok) * t.xt +
                                             (int64_t)(head - (first ? 0 : H0)) * t.xh + c * V);
    }
    row += R;
    tok += step_t;
    head += step_h;
    if (head >= HT) {
      head -= HT;
      ++tok;
    }
  };
#pragma unroll
  for (int u = 0; u < kRotUnroll; ++u) load(u);
  rot_angles(p, b, t0, nt, cs);
  __syncthreads();

  const int turns = (rows + R * kRotUnroll - 1) / (R * kRotUnroll);  // the same for every thread
  for (int n = 0; n < turns; ++n) {
    uint4 y[kRotUnroll];
    uint8_t* const mine = rows_s[wave];
#pragma unroll
    for (int u = 0; u < kRotUnroll; ++u)
      if (on) *reinterpret_cast<uint4*>(mine + (u * RW * C + lane) * 16) = x[u];
    asm volatile("" ::: "memory");
#pragma unroll
    for (int u = 0; u < kRotUnroll; ++u) {
      if (at_tok[u] < 0) continue;
      const Elem* src = reinterpret_cast<const Elem*>(mine + (u * RW * C + r0 * C) * 16);
      const float2* tc = cs + at_tok[u] * p.pairs;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float a = ld_f32(E{}, &x[u], i), o = ld_f32(E{}, src, partner[i]);
        const float2 k = tc[max((int)pair[i], 0)];
        const float term = o * k.y;
        const float r = a * k.x + ((minus >> i) & 1u ? -term : term);
        st_f32(E{}, &y[u], i, r);
        if (pair[i] < 0) reinterpret_cast<Elem*>(&y[u])[i] = reinterpret_cast<const Elem*>(&x[u])[i];
      }
      const bool first = at_head[u] < H0;
      const RotTensor& t = first ? p.t[0] : p.t[1];
      *reinterpret_cast<uint4*>(static_cast<Elem*>(t.y) + b * t.yb + (int64_t)(t0 + at_tok[u]) * t.yt +
                                (int64_t)(at_head[u] - (first ? 0 : H0)) * t.yh + c * V) = y[u];
    }
    asm volatile("" ::: "memory");
    if (n + 1 < turns) {
#pragma unroll
      for (int u = 0; u < kRotUnroll; ++u) load(u);
    }
  }
}

// The angles' factors of the calling thread's last axes (64 powers cost more host time than the rest of a
// call; a layer stack turns by the same axes throughout).
struct RotFreqs {
  int n_axes = -1;
  int32_t dims[kRotMaxAxes];
  double bases[kRotMaxAxes];
  double freq[kRotMaxPairs];
};

const double* rot_freqs(int n_axes, const int32_t* dims, const double* bases) {
  static thread_local RotFreqs t;
  if (t.n_axes == n_axes && memcmp(t.dims, dims, n_axes * sizeof(int32_t)) == 0 &&
      memcmp(t.bases, bases, n_axes * sizeof(double)) == 0)
    return t.freq;
  t.n_axes = n_axes;
  int pair = 0;
  for (int a = 0; a < n_axes; ++a) {
    t.dims[a] = dims[a];
    t.bases[a] = bases[a];
    for (int i = 0; i < dims[a] / 2; ++i) t.freq[pair++] = pow(bases[a], -2.0 * i / dims[a]) / 6.283185307179586476925;
  }
  return t.freq;
}

template <typename E>
int rot_launch(const RotParams& p, int V, bool staged, hipStream_t stream) {
  const dim3 grid((p.T + p.TT - 1) / p.TT, p.B);
  if (staged) {
    hipLaunchKernelGGL(rotary_staged_kernel<E>, grid, dim3(kRotThreads), 0, stream, p);
    GW_HIP_LAUNCH_CHECK("gw_rotary_axes");
    return GW_OK;
  }
  switch (V) {
    case 8:
      if constexpr (ElemBytes<E>::value == 2) {
        hipLaunchKernelGGL((rotary_axes_kernel<E, 8>), grid, dim3(kRotThreads), 0, stream, p);
      }
      break;
    case 4: hipLaunchKernelGGL((rotary_axes_kernel<E, 4>), grid, dim3(kRotThreads), 0, stream, p); break;
    case 2: hipLaunchKernelGGL((rotary_axes_kernel<E, 2>), grid, dim3(kRotThreads), 0, stream, p); break;
    default: hipLaunchKernelGGL((rotary_axes_kernel<E, 1>), grid, dim3(kRotThreads), 0, stream, p); break;
  }
  GW_HIP_LAUNCH_CHECK("gw_rotary_axes");
  return GW_OK;
}

}  // namespace
}  // namespace gw

extern "C" int gw_rotary_axes(int dtype, const void* x0, const int64_t* x0_strides, void* y0, const int64_t* y0_strides,
                              int64_t H0, const void* x1, const int64_t* x1_strides, void* y1,
                              const int64_t* y1_strides, int64_t H1, int pos_type, const void* pos,
                              const int64_t* pos_strides, int64_t B, int64_t T, int64_t D, int n_axes,
                              const int32_t* axis_dims, const double* bases, int inverse, void* stream) {
  using namespace gw;
  clear_error();
  GW_CHECK_ARG(dtype == GW_DTYPE_BF16 || dtype == GW_DTYPE_FP16 || dtype == GW_DTYPE_FP32, "unknown dtype %d", dtype);
  GW_CHECK_ARG(pos_type == GW_POS_INT32 || pos_type == GW_POS_INT64 || pos_type == GW_POS_FP32,
               "unknown position type %d", pos_type);
  GW_CHECK_ARG(B >= 0 && T >= 0 && H0 >= 0 && H1 >= 0, "negative size");
  GW_CHECK_ARG(D >= 1, "head dim must be positive, got %lld", (long long)D);
  if (D > 2 * kRotMaxPairs) return set_error(GW_ERR_UNSUPPORTED, "head dim %lld is above %d", (long long)D, 2 * kRotMaxPairs);
  GW_CHECK_ARG(n_axes >= 1 && n_axes <= kRotMaxAxes && axis_dims && bases, "1 to %d axes, got %d", kRotMaxAxes, n_axes);
  if (B == 0 || T == 0 || H0 + H1 == 0) return GW_OK;
  if (B > 65535 || T > (1ll << 30) || H0 + H1 > (1ll << 20))
    return set_error(GW_ERR_UNSUPPORTED, "sizes B %lld, T %lld, heads %lld are above 65535, 2^30, 2^20", (long long)B,
                     (long long)T, (long long)(H0 + H1));
  GW_CHECK_ARG(pos && pos_strides, "positions are missing");
  GW_CHECK_ARG((H0 == 0 || (x0 && y0 && x0_strides && y0_strides)) && (H1 == 0 || (x1 && y1 && x1_strides && y1_strides)),
               "a tensor is missing");

  RotParams p = {};
  int turned = 0;
  for (int a = 0; a < n_axes; ++a) {
    GW_CHECK_ARG(axis_dims[a] >= 0 && axis_dims[a] % 2 == 0, "axis %d has %d dims: an even number is needed", a, axis_dims[a]);
    GW_CHECK_ARG(bases[a] > 0 && isfinite(bases[a]), "axis %d: the base must be positive and finite", a);
    GW_CHECK_ARG(axis_dims[a] <= D - turned, "the axes' dims exceed the head dim %lld", (long long)D);
    turned += axis_dims[a];
  }
  GW_CHECK_ARG((D - turned) % 2 == 0, "the %lld dims behind the axes must be an even number", (long long)(D - turned));

  const int elem = dtype == GW_DTYPE_FP32 ? 4 : 2;
  const RotTensor in[2] = {
      {x0, y0, H0 ? x0_strides[0] : 0, H0 ? x0_strides[1] : 0, H0 ? x0_strides[2] : 0, H0 ? y0_strides[0] : 0,
       H0 ? y0_strides[1] : 0, H0 ? y0_strides[2] : 0, (int)H0},
      {x1, y1, H1 ? x1_strides[0] : 0, H1 ? x1_strides[1] : 0, H1 ? x1_strides[2] : 0, H1 ? y1_strides[0] : 0,
       H1 ? y1_strides[1] : 0, H1 ? y1_strides[2] : 0, (int)H1}};
  p.t[0] = in[0];
  p.t[1] = in[1];
  int V = elem == 4 ? 4 : 8;
  auto fits = [&](int v) {
    for (int a = 0; a < n_axes; ++a)
      if (axis_dims[a] / 2 % v) return false;
    if ((D - turned) / 2 % v) return false;
    for (const RotTensor& t : in) {
      if (t.H == 0) continue;
      const int64_t all[6] = {t.xb, t.xt, t.xh, t.yb, t.yt, t.yh};
      for (int64_t s : all)
        if (s % v) return false;
      if ((reinterpret_cast<uintptr_t>(t.x) | reinterpret_cast<uintptr_t>(t.y)) % ((size_t)v * elem)) return false;
    }
    return true;
  };
  const int wide = V;
  while (V > 1 && !fits(V)) V >>= 1;
  // Whole rows 16 bytes at a time, whatever the blocks are?
  bool staged = V < 4 && D % wide == 0 && D / wide <= 64;
  for (const RotTensor& t : in) {
    if (t.H == 0) continue;
    const int64_t all[6] = {t.xb, t.xt, t.xh, t.yb, t.yt, t.yh};
    for (int64_t x : all) staged = staged && x % wide == 0;
    staged = staged && aligned16(t.x) && aligned16(t.y);
  }
  GW_CHECK_ARG(fits(V), "a tensor is not aligned to its element type");

  int dim = 0, pair = 0, group = 0;
  for (int a = 0; a <= n_axes; ++a) {
    const int n = a < n_axes ? axis_dims[a] : (int)D - turned;
    const int half = n / 2;
    for (int i = 0; i < half; i += V, ++group) {
      p.lo[group] = (int16_t)(dim + i);
      p.half[group] = (int16_t)half;
      p.pair[group] = (int16_t)(a < n_axes ? pair + i : kRotMaxPairs);
    }
    for (int i = 0; i < n; ++i) {
      p.dim_pair[dim + i] = (int16_t)(a < n_axes ? pair + (i < half ? i : i - half) : -1);
      p.dim_other[dim + i] = (int16_t)(i < half ? half : -half);
    }
    if (a < n_axes) {
      for (int i = 0; i < half; ++i) p.axis[pair + i] = (uint8_t)a;
      pair += half;
    }
    dim += n;
  }
  p.pairs = pair;
  memcpy(p.freq, rot_freqs(n_axes, axis_dims, bases), pair * sizeof(double));
  p.groups = group;
  p.pos = pos;
  p.pos_type = pos_type;
  p.pb = pos_strides[0];
  p.pt = pos_strides[1];
  p.pa = pos_strides[2];
  p.B = (int)B;
  p.T = (int)T;
  p.D = (int)D;
  p.sign = inverse ? -1.0 : 1.0;
  // Few tokens a workgroup until the chip has four workgroups per CU, then up to 8.
  p.TT = kRotMaxTokens;
  while (p.TT > 1 && B * ((T + p.TT - 1) / p.TT) < 1024) p.TT >>= 1;
  GW_CHECK_GRID((T + p.TT - 1) / p.TT, kRotThreads);
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case GW_DTYPE_BF16: return rot_launch<BF16>(p, V, staged, s);
    case GW_DTYPE_FP16: return rot_launch<FP16>(p, V, staged, s);
    default: return rot_launch<FP32>(p, V, staged, s);
  }
}
