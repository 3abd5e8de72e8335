// Writing and reading the 8-bit key/value cache (gfx950).
//
// write: a row x of D bf16 values becomes e4m3(x * 2^-e) with 2^e the smallest
// power of two for which max|x| * 2^-e <= 448 = 1.75 * 2^8. The magnitudes of
// bf16 values order as the integers of their bits, so the maximum is an integer
// one and e comes from its exponent field E and mantissa: e + 127 = E - 8, one
// more where the mantissa is above 1.75 (never below 1: rows smaller than that
// lose their lowest bits). The product by a power of two is exact, so each
// value is rounded once, to nearest even.
// read: the same back, exact in bf16 (subnormal values of it rounded to nearest).
//
// Both are bound by their bytes: 2 D + D + 1 per row. A row takes D / 16 lanes,
// 16 values each: whole 256-byte lines on the bf16 side, 128-byte ones on the
// cache's. A wave takes 16 positions of one head, keys and values (all its loads
// in flight before the first is used), and neighbouring waves neighbouring
// heads, whose bf16 rows lie side by side.
// Measured: 32760 positions of 40 heads of 128 read in 214 to 257 us (3.9 to 4.7 TB/s;
// a copy of 1 GiB runs at 5.2), 7800 of 12 heads written in 13 us and read back in 16
// (partly from cache). Not kept: non-temporal stores (32760 positions 248 -> 363
// us), 32 or 64 positions per wave (40 heads of 128: 512 positions 8.5, 9.1 and 9.1 us,
// 8192 41, 42 and 39, 32768 249, 236 and 238; 16 heads of 64, 32768 33.6, 34.7 and 41.7).
#include "vx_axis_rope.hpp"
#include "vx_kernels.h"

#include <algorithm>

namespace vx {
namespace {

constexpr int kWaves = 4;
constexpr int kTokens = kKvTokensPerWave;  // positions per wave

template <int D>
struct Rows {
  static constexpr int kLanes = D / 16;          // lanes per row
  static constexpr int kPerPass = 64 / kLanes;   // rows per pass of a wave
  static constexpr int kPasses = kTokens / kPerPass;
};

// Largest magnitude of 16 bf16 values, over the lanes of their row, as bits.
template <int D>
__device__ __forceinline__ uint32_t row_amax(const u32x4 (&x)[2]) {
  u16x2 m = {0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, x[i >> 2][i & 3] & 0x7fff7fffu));
  uint32_t r = max((uint32_t)m[0], (uint32_t)m[1]);
#pragma unroll
  for (int off = 1; off < Rows<D>::kLanes; off <<= 1) r = max(r, (uint32_t)__shfl_xor((int)r, off, 64));
  return r;
}

// Scale byte of a row with this largest magnitude (bf16 bits).
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax) {
  const int e = (int)(amax >> 7);
  return e == 255 ? 255u : (uint32_t)max(e - 8 + ((amax & 0x7fu) > 0x60u ? 1 : 0), 1);
}

// 16 bf16 values times 2^(127 - s), rounded to e4m3 (zeros for a row of scale NaN).
__device__ __forceinline__ u32x4 quantise(const u32x4 (&x)[2], uint32_t s) {
  const float f = __uint_as_float((254u - s) << 23);
  u32x4 y;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t a = x[i >> 1][2 * (i & 1)], b = x[i >> 1][2 * (i & 1) + 1];
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(__uint_as_float(a << 16) * f, __uint_as_float(a & 0xffff0000u) * f, 0, false);
    r = __builtin_amdgcn_cvt_pk_fp8_f32(__uint_as_float(b << 16) * f, __uint_as_float(b & 0xffff0000u) * f, r, true);
    y[i] = s == 255u ? 0u : (uint32_t)r;
  }
  return y;
}

// Largest magnitude of 16 fp32 values, over the lanes of their row, as bits.
template <int D>
__device__ __forceinline__ uint32_t row_amax(const float (&x)[2][8]) {
  uint32_t r = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) r = max(r, __float_as_uint(x[i >> 3][i & 7]) & 0x7fffffffu);
#pragma unroll
  for (int off = 1; off < Rows<D>::kLanes; off <<= 1) r = max(r, (uint32_t)__shfl_xor((int)r, off, 64));
  return r;
}

// Scale byte of a row with this largest magnitude (fp32 bits).
__device__ __forceinline__ uint32_t scale_byte32(uint32_t amax) {
  const int e = (int)(amax >> 23);
  return e == 255 ? 255u : (uint32_t)max(e - 8 + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0), 1);
}

// 16 fp32 values times 2^(127 - s), rounded to e4m3 (zeros for a row of scale NaN).
__device__ __forceinline__ u32x4 quantise(const float (&x)[2][8], uint32_t s) {
  const float f = __uint_as_float((254u - s) << 23);
  u32x4 y;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float* v = &x[i >> 1][4 * (i & 1)];
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * f, v[1] * f, 0, false);
    r = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * f, v[3] * f, r, true);
    y[i] = s == 255u ? 0u : (uint32_t)r;
  }
  return y;
}

// PAIRS: keys are turned (kNoRope: as they are) on the way, in fp32, and rounded once.
// (2 x 4680 positions of 12 heads of 128 in 18.5 us, 21.2 where each wave forms all of
// its angles; the bytes alone 16.9.)
// Then lanes take their channels as the pairs lie (see vx_axis_rope.hpp). SHARED: the
// workgroup's waves have four heads of the same tokens, and form a quarter of a token's
// angles each for all four, by way of LDS.
template <int D, int PAIRS, bool SHARED = false>
__device__ __forceinline__ void write_rows(const KvWriteArgs& a, const AxisRope& rope) {
  using R = Rows<D>;
  const int lane = threadIdx.x & 63;
  const uint32_t w = blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t hk = (uint32_t)a.c.Hk;
  const uint32_t head = w % hk;
  const int64_t t0 = (int64_t)(w / hk) * kTokens;
  const int b = blockIdx.y;
  const int slot = a.slots != nullptr ? a.slots[b] : b;
  const int n = a.num != nullptr ? min(max(a.num[b], 0), a.S) : a.S;
  const int64_t first = a.start != nullptr ? a.start[b] : 0;
  if (t0 >= n || (uint32_t)slot >= (uint32_t)a.c.slots) return;  // (uniform in the wave)
  const int r = lane / R::kLanes, c = lane % R::kLanes;
  bool keep[R::kPasses];
  u32x4 xk[R::kPasses][2], xv[R::kPasses][2];
  RopePlace place[R::kPasses];
#pragma unroll
  for (int p = 0; p < R::kPasses; ++p) {
    const int64_t t = t0 + p * R::kPerPass + r, pos = first + t;
    keep[p] = t < n && pos >= 0 && pos < a.c.cap;
    const int64_t ti = min(t, (int64_t)n - 1);  // (rows past the end load the last one)
    if constexpr (PAIRS == kHalves) {
      const bf16* pk = (const bf16*)a.k + b * a.ks[0] + ti * a.ks[1] + head * a.ks[2] + c * 8;
      const bf16* pv = (const bf16*)a.v + b * a.vs[0] + ti * a.vs[1] + head * a.vs[2] + c * 8;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        xk[p][i] = *(const u32x4*)(pk + D / 2 * i);
        xv[p][i] = *(const u32x4*)(pv + D / 2 * i);
      }
    } else {
      const bf16* pk = (const bf16*)a.k + b * a.ks[0] + ti * a.ks[1] + head * a.ks[2] + c * 16;
      const bf16* pv = (const bf16*)a.v + b * a.vs[0] + ti * a.vs[1] + head * a.vs[2] + c * 16;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        xk[p][i] = *(const u32x4*)(pk + 8 * i);
        xv[p][i] = *(const u32x4*)(pv + 8 * i);
      }
    }
    if constexpr (PAIRS != kNoRope) place[p] = rope_place(rope, b * rope.ps[0] + ti * rope.ps[1]);
  }
  // Positions that a later batch item writes in the same slot are left to it,
  // so that no row mixes two tokens' values and scales.
  if (a.slots != nullptr) {
    for (int b0 = b + 1; b0 < a.B; b0 += 64) {
      const int o = b0 + lane;
      int64_t lo = 0, hi = 0;
      if (o < a.B && a.slots[o] == slot) {
        lo = a.start != nullptr ? a.start[o] : 0;
        hi = lo + (a.num != nullptr ? min(max(a.num[o], 0), a.S) : a.S);
      }
      uint64_t same = __builtin_amdgcn_ballot_w64(lo < hi && lo < first + t0 + kTokens && hi > first + t0);
      for (; same != 0; same &= same - 1) {
        const int j = __builtin_ctzll(same);
        const int64_t jlo = __shfl(lo, j, 64), jhi = __shfl(hi, j, 64);
#pragma unroll
        for (int p = 0; p < R::kPasses; ++p) {
          const int64_t pos = first + t0 + p * R::kPerPass + r;
          keep[p] = keep[p] && !(pos >= jlo && pos < jhi);
        }
      }
    }
  }
  const int64_t row0 = ((int64_t)slot * hk + head) * a.c.cap;
  __shared__ f32x4 angles[SHARED ? R::kPasses : 1][4][SHARED ? 64 : 1];  // a lane's eight sines, then cosines
  if constexpr (SHARED) {
    static_assert(kWaves == 4, "two of a lane's pairs each");
    const int mine = 2 * (threadIdx.x >> 6);
    const RopeTable<2> table = rope_table<2>(rope, 8 * c + mine);
#pragma unroll
    for (int p = 0; p < R::kPasses; ++p) {
      float s[2], co[2];
      rope_angles(table, place[p], false, s, co);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        ((float*)&angles[p][mine >> 2][lane])[(mine & 2) + e] = s[e];
        ((float*)&angles[p][2 + (mine >> 2)][lane])[(mine & 2) + e] = co[e];
      }
    }
    __syncthreads();  // (whole workgroups are here: their waves' tokens are the same)
  }
#pragma unroll
  for (int p = 0; p < R::kPasses; ++p) {
    uint32_t sk;
    float y[2][8];  // keys, turned
    if constexpr (PAIRS == kNoRope) {
      sk = scale_byte(row_amax<D>(xk[p]));
    } else {
      float s[8], co[8];
      if constexpr (SHARED) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          s[e] = angles[p][e >> 2][lane][e & 3];
          co[e] = angles[p][2 + (e >> 2)][lane][e & 3];
        }
      } else {
        rope_angles(rope_table<8>(rope, 8 * c), place[p], false, s, co);
      }
      rope_turn<PAIRS>(xk[p], s, co, y);
      sk = scale_byte32(row_amax<D>(y));
    }
    const uint32_t sv = scale_byte(row_amax<D>(xv[p]));
    u32x4 yk;
    if constexpr (PAIRS == kNoRope)
      yk = quantise(xk[p], sk);
    else
      yk = quantise(y, sk);
    const u32x4 yv = quantise(xv[p], sv);
    if (keep[p]) {
      const int64_t row = row0 + first + t0 + p * R::kPerPass + r;
      if constexpr (PAIRS == kHalves) {
        *(u32x2*)(a.c.k + row * D + c * 8) = u32x2{yk[0], yk[1]};
        *(u32x2*)(a.c.k + row * D + D / 2 + c * 8) = u32x2{yk[2], yk[3]};
        *(u32x2*)(a.c.v + row * D + c * 8) = u32x2{yv[0], yv[1]};
        *(u32x2*)(a.c.v + row * D + D / 2 + c * 8) = u32x2{yv[2], yv[3]};
      } else {
        *(u32x4*)(a.c.k + row * D + c * 16) = yk;
        *(u32x4*)(a.c.v + row * D + c * 16) = yv;
      }
      if (c == 0) {
        a.c.ks[row] = (uint8_t)sk;
        a.c.vs[row] = (uint8_t)sv;
      }
    }
  }
}

template <int D>
__global__ __launch_bounds__(kWaves * 64) void kv_write_kernel(const KvWriteArgs a) {
  write_rows<D, kNoRope>(a, AxisRope{});
}

template <int D, int PAIRS, bool SHARED>
__global__ __launch_bounds__(kWaves * 64) void kv_write_rope_kernel(const KvWriteArgs a, const AxisRope rope) {
  write_rows<D, PAIRS, SHARED>(a, rope);
}

template <int D>
__global__ __launch_bounds__(kWaves * 64) void kv_read_kernel(const KvReadArgs a) {
  using R = Rows<D>;
  const int lane = threadIdx.x & 63;
  const uint32_t w = blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t hk = (uint32_t)a.c.Hk;
  const uint32_t head = w % hk;
  const int64_t t0 = (int64_t)(w / hk) * kTokens;
  const int b = blockIdx.y;
  if (t0 >= a.S) return;
  const int slot = a.slots != nullptr ? a.slots[b] : b;
  const int64_t first = a.start != nullptr ? a.start[b] : 0;
  const int r = lane / R::kLanes, c = lane % R::kLanes;
  const int64_t row0 = ((int64_t)slot * hk + head) * a.c.cap;
  u32x4 yk[R::kPasses], yv[R::kPasses];
  uint32_t sk[R::kPasses], sv[R::kPasses];
#pragma unroll
  for (int p = 0; p < R::kPasses; ++p) {
    const int64_t t = t0 + p * R::kPerPass + r, pos = first + t;
    yk[p] = yv[p] = u32x4{0, 0, 0, 0};
    sk[p] = sv[p] = 127;
    if (t < a.S && (uint32_t)slot < (uint32_t)a.c.slots && pos >= 0 && pos < a.c.cap) {
      yk[p] = *(const u32x4*)(a.c.k + (row0 + pos) * D + c * 16);
      yv[p] = *(const u32x4*)(a.c.v + (row0 + pos) * D + c * 16);
      sk[p] = a.c.ks[row0 + pos];
      sv[p] = a.c.vs[row0 + pos];
    }
  }
#pragma unroll
  for (int p = 0; p < R::kPasses; ++p) {
    const int64_t t = t0 + p * R::kPerPass + r;
    if (t >= a.S) continue;
    const int64_t o = (((int64_t)b * a.S + t) * hk + head) * D + c * 16;
    const float fk = e8m0_scale(sk[p]), fv = e8m0_scale(sv[p]);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      *(bf16x8*)((bf16*)a.k_out + o + 8 * i) = e4m3x8_bf16(u32x2{yk[p][2 * i], yk[p][2 * i + 1]}, fk);
      *(bf16x8*)((bf16*)a.v_out + o + 8 * i) = e4m3x8_bf16(u32x2{yv[p][2 * i], yv[p][2 * i + 1]}, fv);
    }
  }
}

// The first limit[b] positions of each item's slot to contiguous (B, Hk, cap, D) rows
// for the flash kernels, and those lengths, held to the cache, to len_out. A
// token whose key or value row has scale NaN becomes a zero key with a NaN value:
// NaN for every query, whatever weight it gets. Positions lie side by side in
// both forms, so neighbouring waves take neighbouring positions of one head.
template <int D>
__global__ __launch_bounds__(kWaves * 64) void kv_expand_kernel(const KvReadArgs a) {
  using R = Rows<D>;
  const int lane = threadIdx.x & 63;
  const uint32_t w = blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t blocks = ((uint32_t)a.c.cap + kTokens - 1) / kTokens;
  const uint32_t head = w / blocks, t0 = (w % blocks) * kTokens;
  const int b = blockIdx.y;
  const int slot = a.slots != nullptr ? a.slots[b] : b;
  int n = a.limit != nullptr ? min(max(a.limit[b], 0), a.c.cap) : a.c.cap;
  if ((uint32_t)slot >= (uint32_t)a.c.slots) n = 0;
  if (w == 0 && lane == 0) a.len_out[b] = n;
  if (head >= (uint32_t)a.c.Hk || t0 >= (uint32_t)n) return;
  const int r = lane / R::kLanes, c = lane % R::kLanes;
  const int64_t from = ((int64_t)slot * a.c.Hk + head) * a.c.cap + t0 + r;
  const int64_t to = ((int64_t)b * a.c.Hk + head) * a.c.cap + t0 + r;
  u32x4 yk[R::kPasses], yv[R::kPasses];
  uint32_t sk[R::kPasses], sv[R::kPasses];
#pragma unroll
  for (int p = 0; p < R::kPasses; ++p) {  // (the capacity is a multiple of kTokens)
    const int64_t row = from + p * R::kPerPass;
    yk[p] = *(const u32x4*)(a.c.k + row * D + c * 16);
    yv[p] = *(const u32x4*)(a.c.v + row * D + c * 16);
    sk[p] = a.c.ks[row];
    sv[p] = a.c.vs[row];
  }
#pragma unroll
  for (int p = 0; p < R::kPasses; ++p) {
    const int64_t o = (to + p * R::kPerPass) * D + c * 16;
    const bool bad = max(sk[p], sv[p]) == 255u;
    const u32x4 k = bad ? u32x4{0, 0, 0, 0} : yk[p];
    const float fk = e8m0_scale(bad ? 127u : sk[p]), fv = e8m0_scale(bad ? 255u : sv[p]);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      *(bf16x8*)((bf16*)a.k_out + o + 8 * i) = e4m3x8_bf16(u32x2{k[2 * i], k[2 * i + 1]}, fk);
      *(bf16x8*)((bf16*)a.v_out + o + 8 * i) = e4m3x8_bf16(u32x2{yv[p][2 * i], yv[p][2 * i + 1]}, fv);
    }
  }
}

static_assert(64 % kTokens == 0, "a capacity, a multiple of 64, is one of kTokens");

dim3 grid_of(int B, int S, int Hk) {
  const int64_t waves = ((int64_t)S + kTokens - 1) / kTokens * Hk;  // < 2^26 (checked by the C ABI)
  return dim3((unsigned)((waves + kWaves - 1) / kWaves), (unsigned)B);
}

// (Waves go by head, then by tokens: with heads in fours a workgroup has whole tokens.)
template <int D, int PAIRS>
void write_rope(const KvWriteArgs& a, const AxisRope& rope, hipStream_t st) {
  const dim3 grid = grid_of(a.B, a.S, a.c.Hk), threads(kWaves * 64);
  if (a.c.Hk % kWaves == 0)
    hipLaunchKernelGGL((kv_write_rope_kernel<D, PAIRS, true>), grid, threads, 0, st, a, rope);
  else
    hipLaunchKernelGGL((kv_write_rope_kernel<D, PAIRS, false>), grid, threads, 0, st, a, rope);
}

}  // namespace

int launch_kv_write(const KvWriteArgs& a, void* stream, const char** launched) {
  const dim3 grid = grid_of(a.B, a.S, a.c.Hk);
  if (a.c.D == 128)
    hipLaunchKernelGGL(kv_write_kernel<128>, grid, dim3(kWaves * 64), 0, (hipStream_t)stream, a);
  else
    hipLaunchKernelGGL(kv_write_kernel<64>, grid, dim3(kWaves * 64), 0, (hipStream_t)stream, a);
  *launched = a.c.D == 128 ? "kv_write_kernel<128>" : "kv_write_kernel<64>";
  return (int)hipGetLastError();
}

int launch_kv_write_rope(const KvWriteArgs& a, const AxisRope& rope, void* stream, const char** launched) {
  const hipStream_t st = (hipStream_t)stream;
  if (a.c.D == 128)
    rope.halves ? write_rope<128, kHalves>(a, rope, st) : write_rope<128, kAdjacent>(a, rope, st);
  else
    rope.halves ? write_rope<64, kHalves>(a, rope, st) : write_rope<64, kAdjacent>(a, rope, st);
  *launched = a.c.D == 128 ? (rope.halves ? "kv_write_rope_kernel<128, halves>" : "kv_write_rope_kernel<128, adjacent>")
                           : (rope.halves ? "kv_write_rope_kernel<64, halves>" : "kv_write_rope_kernel<64, adjacent>");
  return (int)hipGetLastError();
}

int launch_kv_read(const KvReadArgs& a, void* stream, const char** launched) {
  const dim3 grid = grid_of(a.B, a.S, a.c.Hk);
  if (a.c.D == 128)
    hipLaunchKernelGGL(kv_read_kernel<128>, grid, dim3(kWaves * 64), 0, (hipStream_t)stream, a);
  else
    hipLaunchKernelGGL(kv_read_kernel<64>, grid, dim3(kWaves * 64), 0, (hipStream_t)stream, a);
  *launched = a.c.D == 128 ? "kv_read_kernel<128>" : "kv_read_kernel<64>";
  return (int)hipGetLastError();
}

int launch_kv_expand(const KvReadArgs& a, void* stream, const char** launched) {
  const dim3 grid = grid_of(a.B, a.c.cap, a.c.Hk);
  if (a.c.D == 128)
    hipLaunchKernelGGL(kv_expand_kernel<128>, grid, dim3(kWaves * 64), 0, (hipStream_t)stream, a);
  else
    hipLaunchKernelGGL(kv_expand_kernel<64>, grid, dim3(kWaves * 64), 0, (hipStream_t)stream, a);
  *launched = a.c.D == 128 ? "kv_expand_kernel<128>" : "kv_expand_kernel<64>";
  return (int)hipGetLastError();
}

}  // namespace vx
