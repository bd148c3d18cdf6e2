// Angles of rotary positions with several axes, shared by the passes that turn heads.
#pragma once

#include <math.h>
#include <string.h>

#include "gw_common.h"

namespace gw {
namespace {

constexpr int kRotMaxAxes = 8;
constexpr int kRotMaxPairs = 128;  // D <= 256

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

}  // namespace
}  // namespace gw
