// Attention over the 8-bit key/value cache whose queries see less than all tokens
// up to theirs: a sliding window behind a few first tokens, or a tree of drafted
// tokens. The kernels are those of cached_attn.hpp (few_part, many_part, merge),
// which mask by a row's own rule in the tiles where its rows differ:
//
//   window  keys j < e with j >= e - window or j < sinks, e one past the query's
//           position (causal) or past the last token. A stream's tiles are those
//           of its sinks and of the union of its rows' windows, so the ranges that
//           workgroups take hold no tile that nobody sees, and each tile of rows
//           skips what its own rows do not see; only tiles at a row's border, at
//           either end, are masked key by key. What lies in such a tile at keys that none
//           of its rows sees (Unseen) is kept out of the products: another key's bytes
//           are copied in their place, or zeros stored.
//   tree    keys in front of the drafted ones as ever; of those, the query's
//           ancestors and itself, as bits in LDS that each row walks out from the
//           parents once per part (fill_tree): a tile takes 32 of a row's bits from
//           two words of them, one VALU instruction.
//
// Measured (kernels): one query of 12 heads in a window of 256 of 700 tokens 8.1 us,
// latency of 9 tiles on eight waves; 64 sequences of 150 to 8192 tokens, 32 heads on 8,
// window 2048, 53 us (245 MB, 4.6 TB/s); 1000 and 777 queries of 32 heads, window 1500,
// 65 us (51 GFLOP), and 4680 of 12 heads on 20280 keys 544 us (583 GFLOP, 1.07 PFLOP/s),
// both bound by many_part's loop; trees of 30 to 61 tokens of 32 heads on 150 to 8192
// keys, 16 items, 95 us and the merge of 48 MB of partial rows 15.
#include "cached_attn.hpp"

namespace vx {
namespace {

// Positions that a tile of rows sees at most, for the plan: of a cache of `cap`.
int seen_most(int cap, int Sq, int G, int window, int sinks, bool causal) {
  if (window == 0) return cap;
  const int64_t queries = causal ? std::min(Sq, kManyRows / G + 1) : 1;
  const int64_t most = ((int64_t)sinks + 63) / 64 * 64 + ((int64_t)window + queries + 63) / 64 * 64 + 64;
  return (int)std::min<int64_t>(cap, most);
}

// Ranges of few rows go over streams, with a launch that merges. Where most streams are
// longer than the window it makes them alike, so often each is one workgroup's. Measured,
// streams whole / in ranges, where the rule takes them whole (us a call; 32 heads on 8,
// capacity 8192, lengths spread evenly over 150 to 8192):
//   window       1100           2048           4096           8192
//   8 items      12.9 / 17.1    19.6 / 18.7
//   32           17.3 / 24.8    24.9 / 31.8    39.1 / 46.2    74.0 / 57.6
//   64           28.2 / 38.2    48.8 / 57.8    77.7 / 83.6    131 / 121
//   100          42.6 / 50.4
// The rule has the capacity, not the lengths, which are on the device. A stream of 8192
// among ones of 200 takes its time alone, and a window of the capacity bounds nothing:
//   8            12.9 / 16.1    19.2 / 15.4
//   32           13.1 / 17.6    19.7 / 18.6    33.1 / 21.3    60.2 / 22.7
//   64           17.0 / 19.4    26.3 / 19.6    48.2 / 24.6    92.2 / 27.1
//   100          19.1 / 25.5
// A 32-key tile takes a wave 1.65 us, and ranges cost 11 more.
bool whole_streams(int64_t groups, int64_t tiles, int D, int64_t cus) {
  const int64_t slots = 2 * cus, rounds = (groups + slots - 1) / slots, waves = groups <= cus ? 8 : 4;
  const double t = 1.65 * (double)tiles * D / 128;
  return t * (double)rounds / (double)waves <= t * (double)groups / (double)(slots * kWaves) + 11;
}

// us that many_part takes about (head dim 128). Two workgroups of four waves on a CU take
// 1.83 a tile, one alone 1.3; one of eight, which converts a tile's keys and values once
// for 256 rows, takes 1.7, but leaves less to fill an uneven round with. Measured, 4 / 8
// waves:
//   4680 rows of 12 heads on 20280 keys, one block       570 / 543 us
//   9360                                                 1159 / 1071
//   7800 on 17160 (372 workgroups of eight waves)        826 / 897 (not taken)
//   2 x 1000 queries of 32 heads on 8, window 1500       66 / 62
//   1 x 1000                                             46.3 / 54.5 (not taken)
//   trees: 16 x 61 on 150 .. 8192 keys                   118 / 111
// Whole streams that no window bounds (of a tree, or seen to the capacity) stay with two
// workgroups, a long one beside a short one (queries on 3000 to 8192 keys: 189 / 211).
// Those of a window count as alike, though a wide one leaves them their lengths: window
// 8000 of 8192, 256 queries of 32 heads on 8, lengths of 3000 to 8192, 4 items 117 / 114,
// 8 items 193 / 210, 16 items 418 / 419; 8 items of which one has 8192 keys and the
// others 1100, 160 / 196.
double many_time(const Planned& h, int streams, int64_t tiles, bool wide, int64_t cus) {
  const int64_t k = h.p.budget > 0 ? h.p.budget / streams : 1, full = h.blocks / (2 * cus), rest = h.blocks % (2 * cus);
  const double rounds = wide ? 1.7 * (double)((h.blocks + cus - 1) / cus)
                             : 1.83 * (double)full + (rest == 0 ? 0 : rest <= cus ? 1.3 : 1.83);
  const double rows = (double)h.blocks * (wide ? 2 * kManyRows : kManyRows);
  return rounds * (double)((tiles + k - 1) / k) + (k > 1 ? 6 + 2 * rows * (128 + 2) * 4 / 4e6 : 0);
}

Plan masked_plan(int cap, int B, int Sq, int H, int Hk, int D, int window, int sinks, bool causal) {
  const int seen = seen_most(cap, Sq, H / Hk, window, sinks, causal);
  Plan p = plan_of(seen, 0, 0, B, Sq, H, Hk, D);
  Part& own = p.own.p;
  const int64_t cus = device_cu_count() > 0 ? device_cu_count() : 256;
  if (window > 0 && own.few && own.rows <= 32 && own.budget > 0 &&
      whole_streams((int64_t)B * Hk, (seen + kFewTile - 1) / kFewTile, D, cus)) {
    own.budget = 0;
    own.items = B;
    p.own.blocks = (int64_t)B * Hk;
    p.own.floats = 0;
    p.wide = p.own.blocks <= cus;
  }
  if (!own.few && D == 128 && (B == 1 || own.budget > 0 || seen < cap)) {
    Planned wide = plan_part(B, own.rows, 1, seen, Hk, D, cus, cus, false, false, 2 * kManyRows);
    wide.p.one_round = false;
    const int64_t tiles = (seen + kManyTile - 1) / kManyTile;
    if (many_time(wide, B, tiles, true, cus) < many_time(p.own, B, tiles, false, cus)) {
      p.own = wide;
      p.wide = true;
    }
  }
  return p;
}

template <int D, int MASK>
int launch(const MaskedAttnArgs& a, hipStream_t st, const char** launched) {
  Plan pl = masked_plan(a.c.cap, a.B, a.Sq, a.H, a.c.Hk, D, a.window, a.sinks, a.causal != 0);
  Part& own = pl.own.p;
  own.s = Streams{a.c, a.kv_len, a.slots, a.B};
  own.ws = a.ws;
  const dim3 grid((unsigned)pl.own.blocks), threads(kThreads);
  if (own.few && pl.wide) {
    hipLaunchKernelGGL((few_masked_kernel<D, 8, MASK>), grid, dim3(512), 0, st, a, own);
    *launched = MASK == kTree ? (D == 128 ? "few_masked_kernel<128, 8, tree>" : "few_masked_kernel<64, 8, tree>")
                              : (D == 128 ? "few_masked_kernel<128, 8, window>" : "few_masked_kernel<64, 8, window>");
  } else if (own.few) {
    hipLaunchKernelGGL((few_masked_kernel<D, 4, MASK>), grid, threads, 0, st, a, own);
    *launched = MASK == kTree ? (D == 128 ? "few_masked_kernel<128, 4, tree>" : "few_masked_kernel<64, 4, tree>")
                              : (D == 128 ? "few_masked_kernel<128, 4, window>" : "few_masked_kernel<64, 4, window>");
  } else if (D == 128 && pl.wide) {
    hipLaunchKernelGGL((many_masked_kernel<128, MASK, 8>), grid, dim3(512), 0, st, a, own);
    *launched = MASK == kTree ? "many_masked_kernel<128, 8, tree>" : "many_masked_kernel<128, 8, window>";
  } else {
    hipLaunchKernelGGL((many_masked_kernel<D, MASK, 4>), grid, threads, 0, st, a, own);
    *launched = MASK == kTree ? (D == 128 ? "many_masked_kernel<128, tree>" : "many_masked_kernel<64, tree>")
                              : (D == 128 ? "many_masked_kernel<128, window>" : "many_masked_kernel<64, window>");
  }
  int err = (int)hipGetLastError();
  if (err == 0 && own.budget > 0) {
    const int split = merge_split(pl.own.usual_parts, D);
    const int64_t per_wg = kThreads / (D / 4) / split;
    // (a tree's ranges are those of all its keys)
    constexpr int kRanges = MASK == kWindow ? kWindow : kPlain;
    hipLaunchKernelGGL((merge_kernel<D, kRanges>),
                       dim3((unsigned)(((int64_t)a.c.Hk * own.rows + per_wg - 1) / per_wg), a.B), threads, 0, st, a,
                       own, Part{}, split);
    err = (int)hipGetLastError();
  }
  return err;
}

}  // namespace

int64_t masked_attn_workspace(int32_t cap, int32_t B, int32_t Sq, int32_t H, int32_t Hk, int32_t D, int32_t window,
                              int32_t sinks, bool causal) {
  const Plan p = masked_plan(cap, B, Sq, H, Hk, D, window, sinks, causal);
  return p.own.floats * (int64_t)sizeof(float);
}

int launch_masked_attn(const MaskedAttnArgs& a, void* stream, const char** launched) {
  const hipStream_t st = (hipStream_t)stream;
  if (a.parents != nullptr)
    return a.c.D == 128 ? launch<128, kTree>(a, st, launched) : launch<64, kTree>(a, st, launched);
  return a.c.D == 128 ? launch<128, kWindow>(a, st, launched) : launch<64, kWindow>(a, st, launched);
}

}  // namespace vx
