// Attention over the 8-bit key/value cache for gfx950.
//
// One wave per query row (batch item, query, head): a lane takes a key of each
// 64-key tile, its dot product with the query in fp32, and the wave's softmax
// runs over the tiles with one maximum and one sum; then each lane takes D / 64
// dims of the values. Cached rows are read as they lie.
#include "vx_fp8_cache.hpp"
#include "vx_kernels.h"

namespace vx {
namespace {

constexpr int kWaves = 4;

template <int D>
__global__ __launch_bounds__(kWaves * 64) void cached_attn_rows_kernel(const CachedAttnArgs a) {
  __shared__ float q_lds[kWaves][D];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t rows = (int64_t)a.B * a.Sq * a.H;
  const int64_t w = min((int64_t)blockIdx.x * kWaves + wave, rows - 1);
  const int h = (int)(w % a.H);
  const int64_t bi = w / a.H;
  const int i = (int)(bi % a.Sq), b = (int)(bi / a.Sq);
  const int kvh = h / (a.H / a.c.Hk);
  const bf16* q = (const bf16*)a.q + b * a.qs[0] + i * a.qs[1] + h * a.qs[2];
  bf16* o = (bf16*)a.o + b * a.os[0] + i * a.os[1] + h * a.os[2];
  for (int d = lane; d < D; d += 64) q_lds[wave][d] = (float)q[d] * (a.scale * kLog2e);
  __syncthreads();
  const int m = a.q_len != nullptr ? min(max(a.q_len[b], 0), a.Sq) : a.Sq;
  const int len = a.kv_len != nullptr ? min(max(a.kv_len[b], 0), a.c.cap) : a.c.cap;
  const int slot = a.slots != nullptr ? a.slots[b] : b;
  int own = (uint32_t)slot < (uint32_t)a.c.slots ? len : 0;
  if (a.causal) own = min(own, max(len - m + i + 1, 0));
  float top = -1.0e30f, sum = 0.f, acc[D / 64] = {};
  for (int part = 0; part < 2; ++part) {
    if (part == 0 && a.prefix.k == nullptr) continue;
    const KvCache& c = part == 0 ? a.prefix : a.c;
    int n = own;
    int64_t row0 = ((int64_t)slot * c.Hk + kvh) * c.cap;
    if (part == 0) {
      const int g = b / (a.B / c.slots);
      n = a.prefix_len != nullptr ? min(max(a.prefix_len[g], 0), c.cap) : c.cap;
      row0 = ((int64_t)g * c.Hk + kvh) * c.cap;
    }
    if (i >= m) n = 0;
    for (int j0 = 0; j0 < n; j0 += 64) {
      const int j = j0 + lane;
      float s = -__builtin_inff();
      if (j < n) {
        const uint8_t* k = c.k + (row0 + j) * D;
        float dot = 0.f;
        for (int d = 0; d < D; d += 4) {
          const uint32_t x = *(const uint32_t*)(k + d);
          const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(x, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(x, true);
          dot += lo[0] * q_lds[wave][d] + lo[1] * q_lds[wave][d + 1] + hi[0] * q_lds[wave][d + 2] + hi[1] * q_lds[wave][d + 3];
        }
        s = dot * e8m0_scale(c.ks[row0 + j]);
      }
      float mx = s;
      for (int off = 32; off >= 1; off >>= 1) mx = fmaxf(mx, __shfl_xor(mx, off, 64));
      const float m_new = fmaxf(top, mx), alpha = fast_exp2(top - m_new);
      const float p = j < n ? fast_exp2(s - m_new) : 0.f;
      float ps = p;
      for (int off = 32; off >= 1; off >>= 1) ps += __shfl_xor(ps, off, 64);
      top = m_new;
      sum = sum * alpha + ps;
      const float pv = j < n ? p * e8m0_scale(c.vs[row0 + j]) : 0.f;
      for (int e = 0; e < D / 64; ++e) acc[e] *= alpha;
      for (int jj = 0; jj < min(64, n - j0); ++jj) {
        const float pj = __shfl(pv, jj, 64);
        const uint8_t* v = c.v + (row0 + j0 + jj) * D;
        for (int e = 0; e < D / 64; ++e) acc[e] += pj * __builtin_amdgcn_cvt_f32_fp8((int)v[e * 64 + lane], 0);
      }
    }
  }
  if ((int64_t)blockIdx.x * kWaves + wave >= rows) return;
  const bool empty = __float_as_uint(sum) == 0;  // (by its bits: the build takes comparisons to be of numbers)
  for (int e = 0; e < D / 64; ++e) o[e * 64 + lane] = (bf16)(empty ? 0.f : acc[e] / sum);
}

}  // namespace

int launch_cached_attn(const CachedAttnArgs& a, void* stream, const char** launched) {
  const int64_t rows = (int64_t)a.B * a.Sq * a.H;
  const dim3 grid((unsigned)((rows + kWaves - 1) / kWaves));
  if (a.c.D == 128)
    hipLaunchKernelGGL(cached_attn_rows_kernel<128>, grid, dim3(kWaves * 64), 0, (hipStream_t)stream, a);
  else
    hipLaunchKernelGGL(cached_attn_rows_kernel<64>, grid, dim3(kWaves * 64), 0, (hipStream_t)stream, a);
  *launched = a.c.D == 128 ? "cached_attn_rows_kernel<128>" : "cached_attn_rows_kernel<64>";
  return (int)hipGetLastError();
}

}  // namespace vx
