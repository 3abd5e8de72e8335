// Rotary positions on several axes from integer positions per token (gfx950): the
// turn of vx_axis_rope.hpp on rows (B, S, H, D) of bf16, in fp32, rounded once.
//
// Bound by its bytes, 4 per value. A wave takes one token and up to 64 / (D / 16)
// heads a pass, whole lines on both sides, in up to kPasses passes whose loads are
// all in flight before the angles are formed: they are formed once for all of the
// wave's heads, and their cost hides behind the loads. Measured: 32760 tokens of 40
// heads of 128 in 119 us (5.6 TB/s; a copy of 1 GiB 5.1), 2 x 5003 of 16 heads of 64 in
// 12, eight single tokens of 32 heads in 4.2. Not kept: several tokens of few heads per
// wave (11.5 -> 12.5).
#include "vx_axis_rope.hpp"

#include <algorithm>

namespace vx {
namespace {

constexpr int kWaves = 4;
constexpr int kPasses = 4;

template <int D, int PAIRS>
__global__ __launch_bounds__(kWaves * 64) void axis_rope_kernel(const AxisRopeArgs a, const int parts,
                                                              const int passes) {
  using R = RopeRow<D, PAIRS>;
  constexpr int kHeads = 64 / R::kLanes;  // per pass
  const int lane = threadIdx.x & 63;
  const uint32_t w = blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t t = w / (uint32_t)parts;
  const int b = blockIdx.y, part = (int)(w - t * (uint32_t)parts);
  if (t >= (uint32_t)a.S) return;
  const int c = lane % R::kLanes, h0 = part * passes * kHeads + lane / R::kLanes;
  const bf16* const x = (const bf16*)a.x + b * a.xs[0] + (int64_t)t * a.xs[1];
  bf16* const o = (bf16*)a.o + ((int64_t)b * a.S + t) * a.H * D;
  u32x4 v[kPasses][2];
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const int h = h0 + p * kHeads;
    if (p < passes && h < a.H) {
      v[p][0] = *(const u32x4*)(x + h * a.xs[2] + R::first(c));
      v[p][1] = *(const u32x4*)(x + h * a.xs[2] + R::second(c));
    }
  }
  float s[8], co[8];
  rope_angles(rope_table<8>(a.rope, 8 * c), rope_place(a.rope, b * a.rope.ps[0] + (int64_t)t * a.rope.ps[1]),
              a.inverse != 0, s, co);
#pragma unroll
  for (int p = 0; p < kPasses; ++p) {
    const int h = h0 + p * kHeads;
    if (p < passes && h < a.H) {
      float y[2][8];
      rope_turn<PAIRS>(v[p], s, co, y);
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        bf16x8 r;
#pragma unroll
        for (int e = 0; e < 8; ++e) r[e] = (bf16)y[g][e];
        *(bf16x8*)(o + (int64_t)h * D + (g ? R::second(c) : R::first(c))) = r;
      }
    }
  }
}

template <int D, int PAIRS>
void run(const AxisRopeArgs& a, hipStream_t st) {
  constexpr int kHeads = 64 / RopeRow<D, PAIRS>::kLanes;
  const int all = (a.H + kHeads - 1) / kHeads, parts = (all + kPasses - 1) / kPasses;
  const int passes = (all + parts - 1) / parts;
  const int64_t waves = (int64_t)a.S * parts;  // (below 2^26: checked by the C ABI)
  hipLaunchKernelGGL((axis_rope_kernel<D, PAIRS>), dim3((unsigned)((waves + kWaves - 1) / kWaves), (unsigned)a.B),
                     dim3(kWaves * 64), 0, st, a, parts, passes);
}

}  // namespace

int launch_axis_rope(const AxisRopeArgs& a, void* stream, const char** launched) {
  const hipStream_t st = (hipStream_t)stream;
  if (a.D == 128) {
    a.rope.halves ? run<128, kHalves>(a, st) : run<128, kAdjacent>(a, st);
    *launched = a.rope.halves ? "axis_rope_kernel<128, halves>" : "axis_rope_kernel<128, adjacent>";
  } else {
    a.rope.halves ? run<64, kHalves>(a, st) : run<64, kAdjacent>(a, st);
    *launched = a.rope.halves ? "axis_rope_kernel<64, halves>" : "axis_rope_kernel<64, adjacent>";
  }
  return (int)hipGetLastError();
}

}  // namespace vx
