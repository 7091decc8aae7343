// Rotary angles, shared by the kernels that turn activations.
#pragma once

#include "qs_values.h"

namespace qs {

// cos and sin of pos * freq, scaled by mag and rounded to fp32 once.  The angle of a far position
// needs fp64 (position 10^6 leaves fp32 an error of 0.03 rad), and so does its reduction: k quarter
// turns are taken off with a two-term pi/2 in fused operations (Cody and Waite's scheme), then the
// Taylor series of both on |r| <= pi/4, whose first term left out is below 2^-57.  A token's angles
// are computed once and used by all of its heads.
__device__ __forceinline__ float2 rotary_cos_sin(int pos, double freq, double mag) {
  const double a = (double)pos * freq;
  const double k = __builtin_rint(a * 0.63661977236758134308);  // 2 / pi
  double r = __builtin_fma(-k, 1.57079632679489661923, a);
  r = __builtin_fma(-k, 6.12323399573676603587e-17, r);
  const double z = r * r;
  double s = -1.0 / 1307674368000.0;  // 1 / 15!
  s = __builtin_fma(s, z, 1.0 / 6227020800.0);
  s = __builtin_fma(s, z, -1.0 / 39916800.0);
  s = __builtin_fma(s, z, 1.0 / 362880.0);
  s = __builtin_fma(s, z, -1.0 / 5040.0);
  s = __builtin_fma(s, z, 1.0 / 120.0);
  s = __builtin_fma(s, z, -1.0 / 6.0);
  s = __builtin_fma(s * z, r, r);
  double c = 1.0 / 20922789888000.0;  // 1 / 16!
  c = __builtin_fma(c, z, -1.0 / 87178291200.0);
  c = __builtin_fma(c, z, 1.0 / 479001600.0);
  c = __builtin_fma(c, z, -1.0 / 3628800.0);
  c = __builtin_fma(c, z, 1.0 / 40320.0);
  c = __builtin_fma(c, z, -1.0 / 720.0);
  c = __builtin_fma(c, z, 1.0 / 24.0);
  c = __builtin_fma(c, z, -0.5);
  c = __builtin_fma(c, z, 1.0);
  const int quarter = (int)((long long)k & 3);
  const double sw = quarter & 1 ? c : s, cw = quarter & 1 ? s : c;
  const double cs = quarter == 1 || quarter == 2 ? -cw : cw;
  const double sn = quarter >= 2 ? -sw : sw;
  return {(float)(cs * mag), (float)(sn * mag)};
}

// Sixteen bytes of a head's turned values, with the halves' layout their partners' sixteen, or of the
// values behind them: item c of `turned` + (D - rot) / V.  Heads aligned to 16 bytes, sizes that divide.
template <class T>
struct TurnItem {
  static constexpr int V = 16 / sizeof(T);
  float a[V], b[V];
  static __device__ __forceinline__ int turned(int rot, int interleaved) { return interleaved ? rot / V : rot / 2 / V; }
  static __host__ __device__ __forceinline__ bool fits(int D, int rot, int interleaved) {
    return D % V == 0 && rot % (interleaved ? V : 2 * V) == 0;
  }
  __device__ __forceinline__ void load(const T* x, int c, int turned, int rot, int interleaved) {
    load_values<T, V>(x + (c < turned ? c * V : rot + (c - turned) * V), a);
    if (c < turned && !interleaved) load_values<T, V>(x + rot / 2 + c * V, b);
  }
  // cs: cos and sin of the token's pairs
  __device__ __forceinline__ void store(T* y, int c, int turned, int rot, int interleaved, const float2* cs) {
    if (c >= turned) {
      store_values<T, V>(y + rot + (c - turned) * V, a);
    } else if (interleaved) {
      const float2* w = cs + c * (V / 2);
#pragma unroll
      for (int e = 0; e < V; e += 2) {
        const float x1 = a[e], x2 = a[e + 1];
        a[e] = x1 * w[e / 2].x - x2 * w[e / 2].y;
        a[e + 1] = x2 * w[e / 2].x + x1 * w[e / 2].y;
      }
      store_values<T, V>(y + c * V, a);
    } else {
      const float2* w = cs + c * V;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float x1 = a[e], x2 = b[e];
        a[e] = x1 * w[e].x - x2 * w[e].y;
        b[e] = x2 * w[e].x + x1 * w[e].y;
      }
      store_values<T, V>(y + c * V, a);
      store_values<T, V>(y + rot / 2 + c * V, b);
    }
  }
};

}  // namespace qs
