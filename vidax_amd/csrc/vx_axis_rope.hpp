// Turning pairs of channels by a token's positions on several axes.
//
// Pair j of a head turns by position[axis[j]] * turns[j], turns[j] a fraction of a
// turn in units of 2^-64. The product modulo 2^64 is the angle with its whole turns
// left out, exact for any 32-bit position: two integer multiplications take the
// place of a range reduction, and its top 32 bits are off by less than 2^-32 of a
// turn (and by half a unit of turns[j], 2^-65, times the position). The nearest
// quarter turn is the top bits' own; what is left, r in [-pi/4, pi/4), goes through
// the Taylor polynomials of sine and cosine to r^9 and r^8, whose remainders,
// r^11 / 11! and r^10 / 10!, are below 1.8e-9 and 2.5e-8. With their roundings (three
// half steps in r, one in the result) a sine or cosine is off by less than 2^-21. A pair
// that does not turn keeps its values.
//
// Lanes: D / 16 to a head's row, each with eight pairs: channels 16 c .. 16 c + 15
// (adjacent pairs) or 8 c .. 8 c + 7 of both halves (pairs (j, j + D / 2)).
#pragma once

#include "vx_fp8_cache.hpp"
#include "vx_kernels.h"

namespace vx {

enum RopePairs : int { kNoRope = 0, kAdjacent = 1, kHalves = 2 };

template <int D, int PAIRS>
struct RopeRow {
  static constexpr int kLanes = D / 16;
  // first channels of the lane's two groups of eight
  static __device__ __forceinline__ int first(int c) { return PAIRS == kHalves ? 8 * c : 16 * c; }
  static __device__ __forceinline__ int second(int c) { return PAIRS == kHalves ? D / 2 + 8 * c : 16 * c + 8; }
};

__device__ __forceinline__ void sincos_turns(uint32_t a, float& s, float& c) {
  const uint32_t q = (a + 0x20000000u) >> 30;  // nearest quarter turn
  const float r = (float)(int32_t)(a - (q << 30)) * 1.46291807926715968105e-9f;  // 2 pi / 2^32
  const float z = r * r;
  float u = __builtin_fmaf(z, 2.75573192239858906526e-6f, -1.98412698412698412698e-4f);
  u = __builtin_fmaf(z, u, 8.33333333333333333333e-3f);
  u = __builtin_fmaf(z, u, -1.66666666666666666667e-1f);
  u = __builtin_fmaf(z * r, u, r);
  float v = __builtin_fmaf(z, 2.48015873015873015873e-5f, -1.38888888888888888889e-3f);
  v = __builtin_fmaf(z, v, 4.16666666666666666667e-2f);
  v = __builtin_fmaf(z, v, -0.5f);
  v = __builtin_fmaf(z, v, 1.0f);
  const float x = q & 1 ? v : u, y = q & 1 ? u : v;
  s = __uint_as_float(__float_as_uint(x) ^ ((q & 2) << 30));
  c = __uint_as_float(__float_as_uint(y) ^ (((q + 1) & 2) << 30));
}

// N pairs, from `first` on.
template <int N>
struct RopeTable {
  uint64_t turns[N];
  int32_t axis[N];
};

template <int N>
__device__ __forceinline__ RopeTable<N> rope_table(const AxisRope& r, int first) {
  RopeTable<N> t;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    t.turns[e] = r.turns[first + e];
    t.axis[e] = r.axis[first + e];
  }
  return t;
}

// Positions of a token, at `at` (elements of r.positions); axes that there are not are 0.
struct RopePlace {
  int32_t p[kRopeAxes];
};
__device__ __forceinline__ RopePlace rope_place(const AxisRope& r, int64_t at) {
  RopePlace p;
#pragma unroll
  for (int x = 0; x < kRopeAxes; ++x) p.p[x] = x < r.axes ? r.positions[at + x * r.ps[2]] : 0;
  return p;
}

// Their sines and cosines at a token's positions.
template <int N>
__device__ __forceinline__ void rope_angles(const RopeTable<N>& t, const RopePlace& at, bool back, float (&s)[N],
                                            float (&c)[N]) {
#pragma unroll
  for (int e = 0; e < N; ++e) {
    int32_t p = 0;  // (a pair of an axis that there is not does not turn)
#pragma unroll
    for (int x = 0; x < kRopeAxes; ++x) p = t.axis[e] == x ? at.p[x] : p;
    sincos_turns((uint32_t)(((uint64_t)(int64_t)p * t.turns[e]) >> 32), s[e], c[e]);
    if (back) s[e] = -s[e];
  }
}

// The lane's 16 channels (two groups of eight, as bf16 pairs), turned, in fp32.
template <int PAIRS>
__device__ __forceinline__ void rope_turn(const u32x4 (&x)[2], const float (&s)[8], const float (&c)[8],
                                          float (&y)[2][8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int g0 = PAIRS == kHalves ? 0 : e >> 2, i0 = PAIRS == kHalves ? e : 2 * (e & 3);
    const int g1 = PAIRS == kHalves ? 1 : g0, i1 = PAIRS == kHalves ? e : i0 + 1;
    auto value = [&](int g, int i) {
      const uint32_t w = x[g][i >> 1];
      return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
    };
    const float a = value(g0, i0), b = value(g1, i1);
    // (without a turn neither channel takes the other's infinity or NaN, nor loses the
    // sign of a zero)
    const bool still = s[e] == 0.0f && c[e] > 0.0f;
    y[g0][i0] = still ? a : __builtin_fmaf(a, c[e], -(b * s[e]));
    y[g1][i1] = still ? b : __builtin_fmaf(a, s[e], b * c[e]);
  }
}

}  // namespace vx
