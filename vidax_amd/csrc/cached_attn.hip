// The launches of attention over the 8-bit key/value cache, with and without a
// shared prefix; the kernels, and what they measured, are in cached_attn.hpp.
#include "cached_attn.hpp"

namespace vx {
namespace {

template <int D>
int launch(const CachedAttnArgs& a, hipStream_t st, const char** launched) {
  const int n_prefix = a.prefix.k != nullptr ? a.prefix.slots : 0;
  Plan pl = plan_of(a.c.cap, n_prefix, a.prefix.cap, a.B, a.Sq, a.H, a.c.Hk, D);
  Part& own = pl.own.p;
  Part& pre = pl.pre.p;
  own.s = Streams{a.c, a.kv_len, a.slots, a.B};
  own.ws = a.ws;
  pre.s = Streams{a.prefix, a.prefix_len, nullptr, n_prefix};
  pre.ws = a.ws + pl.own.floats;
  const dim3 grid((unsigned)(pl.pre.blocks + pl.own.blocks)), threads(kThreads);
  const int pre_blocks = (int)pl.pre.blocks;
  const bool wide = pl.wide;
  const dim3 few_threads(wide ? 512 : 256);
  if (pl.both) {
    if (wide)
      hipLaunchKernelGGL((few_kernel<D, 8, true>), grid, few_threads, 0, st, a, own, pre);
    else
      hipLaunchKernelGGL((few_kernel<D, 4, true>), grid, few_threads, 0, st, a, own, pre);
    *launched = wide ? (D == 128 ? "few_kernel<128, 8, true>" : "few_kernel<64, 8, true>")
                     : (D == 128 ? "few_kernel<128, 4, true>" : "few_kernel<64, 4, true>");
  } else if (n_prefix == 0 && own.few) {
    if (wide)
      hipLaunchKernelGGL((few_kernel<D, 8, false>), grid, few_threads, 0, st, a, own, pre);
    else
      hipLaunchKernelGGL((few_kernel<D, 4, false>), grid, few_threads, 0, st, a, own, pre);
    *launched = wide ? (D == 128 ? "few_kernel<128, 8, false>" : "few_kernel<64, 8, false>")
                     : (D == 128 ? "few_kernel<128, 4, false>" : "few_kernel<64, 4, false>");
  } else if (n_prefix == 0) {
    hipLaunchKernelGGL(many_kernel<D>, grid, threads, 0, st, a, own);
    *launched = D == 128 ? "many_kernel<128>" : "many_kernel<64>";
  } else if (pre.few && own.few) {
    hipLaunchKernelGGL((prefix_kernel<D, true, true>), grid, threads, 0, st, a, pre, own, pre_blocks);
    *launched = D == 128 ? "prefix_kernel<128, true, true>" : "prefix_kernel<64, true, true>";
  } else if (pre.few) {
    hipLaunchKernelGGL((prefix_kernel<D, true, false>), grid, threads, 0, st, a, pre, own, pre_blocks);
    *launched = D == 128 ? "prefix_kernel<128, true, false>" : "prefix_kernel<64, true, false>";
  } else if (own.few) {
    hipLaunchKernelGGL((prefix_kernel<D, false, true>), grid, threads, 0, st, a, pre, own, pre_blocks);
    *launched = D == 128 ? "prefix_kernel<128, false, true>" : "prefix_kernel<64, false, true>";
  } else {
    hipLaunchKernelGGL((prefix_kernel<D, false, false>), grid, threads, 0, st, a, pre, own, pre_blocks);
    *launched = D == 128 ? "prefix_kernel<128, false, false>" : "prefix_kernel<64, false, false>";
  }
  int err = (int)hipGetLastError();
  if (err == 0 && !pl.both && (n_prefix > 0 || own.budget > 0)) {
    const int split = merge_split(pl.own.usual_parts + (n_prefix > 0 ? pl.pre.usual_parts : 0), D);
    const int64_t per_wg = kThreads / (D / 4) / split;
    hipLaunchKernelGGL(merge_kernel<D>, dim3((unsigned)(((int64_t)a.c.Hk * own.rows + per_wg - 1) / per_wg), a.B),
                       threads, 0, st, a, own, pre, split);
    err = (int)hipGetLastError();
  }
  return err;
}

}  // namespace

int64_t cached_attn_workspace(int32_t cap, int32_t n_prefix, int32_t p_cap, int32_t B, int32_t Sq, int32_t H,
                              int32_t Hk, int32_t D) {
  const Plan p = plan_of(cap, n_prefix, p_cap, B, Sq, H, Hk, D);
  return (p.own.floats + p.pre.floats) * (int64_t)sizeof(float);
}

int launch_cached_attn(const CachedAttnArgs& a, void* stream, const char** launched) {
  return a.c.D == 128 ? launch<128>(a, (hipStream_t)stream, launched) : launch<64>(a, (hipStream_t)stream, launched);
}

}  // namespace vx
