// Attention over the 8-bit key/value cache for gfx950, bf16 queries and output,
// D = 128 or 64.
//
// The query rows that share a cached head's keys -- the G heads of a group times
// the queries of an item, for a prefix times the items that share it -- are a
// stream's rows. Its keys are cut into ranges, one workgroup each per tile of rows:
//
//   few_part   32 rows: four (or eight) waves, each on every fourth 32-key tile of
//              the range (single tokens, short prompts, small prefixes)
//   many_part  128 rows: four waves of 32 rows each on the same 64-key tiles
//              (prompts in chunks, cross-attention, a long prefix under a batch)
//   merge      joins the parts of a stream, and a prefix's with the items' own
//
// All compute S^T = K Q^T and O^T = V^T P^T with v_mfma_f32_32x32x16_bf16, so that a
// lane holds one query row: its maximum, sum and rescaling are the lane's own,
// and the two halves of a wave exchange them by one v_permlane32_swap. e4m3
// values are exact in bf16, and so are they times a power of two, so the only
// roundings are the weights' and the output's to bf16; scores, sums, outputs and
// partial results are fp32. (The weights are rounded because the MFMA takes bf16: fp32
// ones would be two products, high and low part, for a relative error against 64 bits
// of 1.6e-3, the output's rounding alone, in place of 1.6e-3 to 1.8e-3. The sum that
// divides is that of the rounded weights, so values that agree come out as they are.)
//
// few_part reads K and V as they lie, by DMA to LDS rings of the waves' own (no
// barrier in the loop), and converts them behind the LDS reads: K with its scale in
// the same instruction, V unscaled, its scales multiplied into the weights, since
// the transposed read gives a lane eight keys of one dim. It is bound by memory for
// single tokens: 64 sequences of 227 to 8192 keys, 8 kv heads, 562 MB in 105 us (5.4
// TB/s); two of 131000 and 105009 keys 488 MB in 90 us (5.4 TB/s).
// many_part converts each 64-key tile once for its four waves, on the way to LDS,
// and runs the matrix cores of a tile beside the next one's softmax and conversions:
// 1000 and 943 queries of 32 heads on 5003 and 4324 keys 138 us (0.96 PFLOP/s; 150 to
// 175 us in the first calls after an idle time). The matrix cores are busy 44 % of that
// and the VALU 45 %: a tile's products and its softmax and conversions hardly overlap.
#include "vx_fp8_cache.hpp"
#include "vx_kernels.h"

#include <algorithm>
#include <type_traits>

namespace vx {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * 64;
constexpr float kNone = -__FLT_MAX__;  // "no key seen yet": a reference point that no score lies below
constexpr float kSlack = 8.0f;         // weights up to 2^kSlack before the reference point moves
// A weight is 2^(score * c - m) in one fused operation, m such a product, rounded. Past
// this magnitude of m that rounding (up to 2^-24 of it) is more than a factor of two of
// the weight, and far past it weights are all infinite or nothing. A workgroup that
// ends a part with such an m does it once more with the products rounded on both sides.
constexpr float kFar = 16777216.0f;

typedef VX_LDS unsigned char lds_u8;
// (a pointer made from an integer is a flat one unless its type says more, and a
// flat load holds up the LDS counter that every barrier waits for)
#define VX_GLOBAL __attribute__((address_space(1)))
typedef VX_GLOBAL const uint8_t global_u8;

template <int N>
__device__ __forceinline__ void wait_copies() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void wait_lds_reads() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

__device__ __forceinline__ bool is_far(float m) { return fabsf(m) > kFar && m > kNone; }

// x == 0 by its bits, hidden from the compiler (which may take floats to be no NaN).
__device__ __forceinline__ bool is_zero(float x) {
  uint32_t u = __float_as_uint(x);
  asm("" : "+v"(u));
  return (u & 0x7fffffffu) == 0;
}

// ---- streams: the own keys of each batch item, or the prefix of each group
struct Streams {
  KvCache c;
  const int32_t* len;
  const int32_t* slots;
  int32_t n;  // streams
};

__device__ __forceinline__ int clamp_len(const int32_t* len, int i, int most) {
  return len != nullptr ? min(max(len[i], 0), most) : most;
}

// Slot of a stream, -1 if the cache does not have it.
__device__ __forceinline__ int slot_of(const Streams& s, int i) {
  const int slot = s.slots != nullptr ? s.slots[i] : i;
  return (uint32_t)slot < (uint32_t)s.c.slots ? slot : -1;
}

// Keys of a stream.
__device__ __forceinline__ int keys_of(const Streams& s, int i) {
  return slot_of(s, i) < 0 ? 0 : clamp_len(s.len, i, s.c.cap);
}

// The streams' key tiles (TILE keys each) stand one after another in one line,
// which is cut into `budget` equal ranges (none shorter than min_chunk), one
// workgroup each: however the lengths differ, all workgroups have the same work.
// A range's piece of a stream is a part; range w's part of stream s has the number
// w + s, which no other has. Every wave works its range out for itself from the
// lengths, 64 streams per step. budget 0: range w is stream w, whole.
template <int TILE>
__device__ __forceinline__ int tiles_in(int keys) {
  return (keys + TILE - 1) / TILE;
}

__device__ __forceinline__ int lane_keys(const Streams& s, int i) { return i < s.n ? keys_of(s, i) : 0; }

__device__ __forceinline__ int wave_sum(int x) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) x += __shfl_xor(x, off, 64);
  return x;
}

// Tiles of a range. (All streams' tiles together are below 2^31: checked by the C ABI.)
__device__ __forceinline__ int range_tiles(int total, int budget, int min_chunk) {
  return max((int)(((uint32_t)total + budget - 1) / (uint32_t)budget), min_chunk);
}

// Where range w begins: its first stream, that one's keys, the tile in it, and the range's tiles (0: none).
struct Range {
  int stream, len, tile, tiles;
};
template <int TILE>
__device__ __forceinline__ Range range_of(const Streams& s, int budget, int min_chunk, int w) {
  const int lane = threadIdx.x & 63;
  const int first = lane_keys(s, lane);  // (64 streams are the usual case: read once)
  int total = wave_sum(tiles_in<TILE>(first));
  for (int i0 = 64; i0 < s.n; i0 += 64) total += wave_sum(tiles_in<TILE>(lane_keys(s, i0 + lane)));
  const int each = range_tiles(total, budget, min_chunk);
  const int64_t lo = (int64_t)w * each;
  Range r{0, 0, 0, 0};
  if (lo < total) {
    r.tiles = min(each, total - (int)lo);
    int base = 0;
    for (int i0 = 0;; i0 += 64) {  // (ends: lo is below the total)
      const int keys = i0 == 0 ? first : lane_keys(s, i0 + lane), t = tiles_in<TILE>(keys);
      int upto = t;  // inclusive scan over the lanes
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const int o = __shfl_up(upto, off, 64);
        if (lane >= off) upto += o;
      }
      const uint64_t past = __builtin_amdgcn_ballot_w64(base + upto > (int)lo);
      if (past != 0 || i0 + 64 >= s.n) {
        const int l = past != 0 ? __builtin_ctzll(past) : 63;
        r.stream = min(i0 + l, s.n - 1);
        r.len = __shfl(keys, l, 64);
        r.tile = (int)lo - base - __shfl(upto - t, l, 64);
        break;
      }
      base += __shfl(upto, 63, 64);
    }
  }
  return Range{__builtin_amdgcn_readfirstlane(r.stream), __builtin_amdgcn_readfirstlane(r.len),
               __builtin_amdgcn_readfirstlane(r.tile), __builtin_amdgcn_readfirstlane(r.tiles)};
}

__device__ __forceinline__ Range whole_stream(const Streams& s, int i) {
  return Range{i, __builtin_amdgcn_readfirstlane(keys_of(s, i)), 0, 1};
}

// The next stream that has keys, and its keys. (There is one while a range has
// tiles left; false, past the last, only if the lengths changed under the launch.)
__device__ __forceinline__ bool next_stream(const Streams& s, int& stream, int& len) {
  for (++stream; stream < s.n; ++stream) {
    len = __builtin_amdgcn_readfirstlane(keys_of(s, stream));
    if (len > 0) return true;
  }
  return false;
}

// The parts of stream `want`.
struct Parts {
  int first, count;
};
template <int TILE>
__device__ __forceinline__ Parts parts_of(const Streams& s, int budget, int min_chunk, int want) {
  if (budget == 0) return Parts{want, 1};
  const int lane = threadIdx.x & 63;
  int total = 0, before = 0, mine = 0;
  for (int i0 = 0; i0 < s.n; i0 += 64) {
    const int t = tiles_in<TILE>(lane_keys(s, i0 + lane));
    total += wave_sum(t);
    if (i0 <= want) before += wave_sum(i0 + lane < want ? t : 0);
    if (want >= i0 && want < i0 + 64) mine = __shfl(t, want - i0, 64);
  }
  if (mine == 0) return Parts{0, 0};
  const uint32_t each = range_tiles(total, budget, min_chunk);
  const int w0 = (uint32_t)before / each, w1 = (uint32_t)(before + mine - 1) / each;
  return Parts{w0 + want, w1 - w0 + 1};
}

// ---- the rows of a stream
struct RowMap {
  const CachedAttnArgs& a;
  int stream, kvh, G, per;  // per: batch items of a stream
  __device__ __forceinline__ void place(int r, int& b, int& i, int& h) const {
    const int q = r / G;
    h = kvh * G + (r - q * G);
    const int item = per == 1 ? 0 : q / a.Sq;
    i = q - item * a.Sq;
    b = stream * per + item;
  }
};

// Keys that query i of item b sees of its own `len` (0 for a padding row).
__device__ __forceinline__ int own_bound(const CachedAttnArgs& a, int b, int i, int len) {
  const int m = clamp_len(a.q_len, b, a.Sq);
  if (i >= m) return 0;
  return a.causal ? min(max(len - m + i + 1, 0), len) : len;
}

// One launch's work on one kind of streams.
struct Part {
  Streams s;
  int32_t rows, per;          // rows of a stream per kv head; batch items that share it
  int32_t budget, min_chunk;  // ranges of its tiles, per kv head and row tile (0: one per stream)
  int32_t items;              // ranges that are launched
  int32_t prefix;             // 1: every row sees every key
  int32_t one_round;          // 1: all workgroups find a place at once (many_part)
  int32_t direct;             // 1: a stream of one part writes its output itself
  int32_t few;                // few_part, else many_part
  float* ws;                  // partial results
};

// Partial results in the workspace, one block per (part, kv head): rows x D
// unnormalised fp32 outputs, then (reference point, sum) per row.
__device__ __forceinline__ int64_t part_floats(int64_t rows, int D) { return (rows * (D + 2) + 3) & ~(int64_t)3; }

template <int D>
struct Fp8Tile {
  static constexpr int kChunks = D / 16;  // 16-byte chunks of a row
  // XOR swizzle of a row's chunks in LDS (64 banks of 4 bytes): 16 keys' reads of one chunk
  // (ds_read_b128) and 8 keys' reads of two neighbouring ones (ds_read_b64_tr_b8)
  // each touch 16 different 16-byte bank groups.
  static __device__ __forceinline__ int swizzle(int key) {
    if (D == 128) return half_swizzle(key);
    return (((key >> 2) & 1) << 1) | ((key >> 3) & 1);
  }
};

// ------------------------------------------------------------------ few rows
constexpr int kFewTile = 32;  // keys per tile of few_kernel

template <int D, int W>
struct FewCfg {
  static constexpr int kTileBytes = kFewTile * D;        // of K, and of V
  static constexpr int kCopies = kTileBytes / 1024;      // DMA copies of each
  static constexpr int kPerTile = 2 * kCopies + 1;       // ... of a tile, with its scales
  static constexpr int kBuf = 2 * kTileBytes + 128;      // K, V, 32 + 32 scale bytes
  static constexpr int kRing = 2;
  static constexpr int kOutRow = D + 4;                  // fp32 values between rows of the exchange
  static constexpr int kExchange = 32 * kOutRow * 4;
  static constexpr int kTiles = (kRing * kBuf > kExchange ? kRing * kBuf : kExchange) * W;
  static constexpr int kFlags = kTiles + W * 32 * 8;  // then (reference point, sum) of the waves' rows
  static constexpr int kSmem = kFlags + W * 4;        // ... whether any of them is far, per wave
};

// Keys of one kv head as few_part reads them.
struct FewKeys {
  uint64_t k, v;          // addresses of the first rows
  const uint8_t* scales;  // this lane's 16 bytes of a tile's scales (lanes 0-1 K, 2-3 V)
  int len;                // keys
  int bound, all;         // those that this lane's row sees, those that every row does
};

// A range of tiles of streams, for 32 rows of one kv head (BOTH: stream `block`, the
// group's prefix in front of its own keys). The W waves take every W-th tile.
template <int D, int W, bool BOTH>
__device__ __forceinline__ void few_part(const CachedAttnArgs& a, const Part& pt, const Part* pre, const int block,
                                         unsigned char* smem) {
  using C = FewCfg<D, W>;
  using T = Fp8Tile<D>;
  const Streams& s = pt.s;
  float(*const ml)[32][2] = (float(*)[32][2])(smem + C::kTiles);
  VX_LDS int* const far = (VX_LDS int*)((lds_u8*)smem + C::kFlags);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hf = lane >> 5, col = lane & 31;
  // kv heads side by side, then the row tiles: with 8 heads each XCD keeps one
  // head's keys in its L2 for all of its row tiles
  const int Hk = s.c.Hk, kvh = block % Hk, n_rt = (pt.rows + 31) / 32;
  const int item = block / Hk / n_rt, row0 = (block / Hk - item * n_rt) * 32;
  const int rows = min(pt.rows - row0, 32);
  lds_u8* const ring = (lds_u8*)smem + wave * C::kRing * C::kBuf;
  const uint32_t ring_addr = (uint32_t)(uintptr_t)ring;
  const float c = a.scale * kLog2e;
  // K fragment row of this lane: MFMA row x holds key (x with bits 2 and 3
  // swapped), so that a lane's 16 scores are keys 16 j + 8 hf + 0..7, j = 0, 1:
  // the order in which the B operand of PV takes its weights
  const int kkey = (col & 0x13) | ((col & 4) << 1) | ((col & 8) >> 1);

  auto keys = [&](const Streams& from, int stream, int len) {
    const int64_t at = ((int64_t)slot_of(from, stream) * Hk + kvh) * from.c.cap;
    return FewKeys{uniform_u64((uint64_t)(uintptr_t)(from.c.k + at * D)),
                   uniform_u64((uint64_t)(uintptr_t)(from.c.v + at * D)),
                   (lane & 2 ? from.c.vs : from.c.ks) + at + 16 * (lane & 1), len, len, len};
  };
  // ---- staging: copy p of a tile fills 1024 / D rows; lane L takes row L / (D / 16),
  // LDS chunk L % (D / 16), which holds the row's chunk with that number XOR the swizzle
  auto stage = [&](const FewKeys& x, int t, int buf) {
    const uint32_t dst = ring_addr + buf * C::kBuf;
    const int last = x.len - 1 - t * kFewTile;  // last row of the tile that holds a key
    const i32x4_rsrc rk = raw_rsrc_u64(x.k + (uint64_t)t * C::kTileBytes);
    const i32x4_rsrc rv = raw_rsrc_u64(x.v + (uint64_t)t * C::kTileBytes);
#pragma unroll
    for (int p = 0; p < C::kCopies; ++p) {
      const int r = p * (1024 / D) + lane / T::kChunks;
      // (rows past the last key repeat it: what lies there may be anything)
      const uint32_t off = (uint32_t)(min(r, last) * D + ((lane % T::kChunks) ^ T::swizzle(r)) * 16);
      lds_dma16_buf(rk, off, dst + p * 1024);
      lds_dma16_buf(rv, off, dst + C::kTileBytes + p * 1024);
    }
    if (lane < 4) lds_dma16(x.scales + (int64_t)t * kFewTile, dst + 2 * C::kTileBytes);
  };

  const Range range = pt.budget == 0 ? whole_stream(s, item) : range_of<kFewTile>(s, pt.budget, pt.min_chunk, item);
  int stream = range.stream, len = range.len, first = range.tile, left = range.tiles;
  bool rounded = false;  // the products are
  while (left > 0) {
    const int tiles = tiles_in<kFewTile>(len), take = pt.budget == 0 ? tiles : min(left, tiles - first);

    const RowMap map{a, stream, kvh, a.H / Hk, pt.per};
    int rb, ri, rh;
    map.place(row0 + min(col, rows - 1), rb, ri, rh);
    bf16x8 q[D / 16];
    {
      const bf16* p = (const bf16*)a.q + rb * a.qs[0] + ri * a.qs[1] + rh * a.qs[2] + hf * 16;
#pragma unroll
      for (int x = 0; x < D / 32; ++x) {
        q[2 * x] = *(const bf16x8*)(p + 32 * x);
        q[2 * x + 1] = *(const bf16x8*)(p + 32 * x + 8);
      }
    }
    FewKeys own = keys(s, stream, len), shared = own;
    int pre_tiles = 0;
    if (BOTH) {
      const int group = stream / pre->per;
      shared = keys(pre->s, group, __builtin_amdgcn_readfirstlane(keys_of(pre->s, group)));
      pre_tiles = (shared.len + kFewTile - 1) / kFewTile;
      if (ri >= clamp_len(a.q_len, rb, a.Sq)) shared.bound = 0;  // (a padding row)
    }
    if (!pt.prefix) own.bound = own_bound(a, rb, ri, len);
    auto least = [&](int x) {
#pragma unroll
      for (int off = 16; off >= 1; off >>= 1) x = min(x, __shfl_xor(x, off, 64));
      return __builtin_amdgcn_readfirstlane(x);
    };
    own.all = least(own.bound);
    const int any = -least(-own.bound);  // keys that some row sees
    if (BOTH) shared.all = least(shared.bound);
    if (rounded) own.all = shared.all = 0;

    f32x16 O[D / 32];
#pragma unroll
    for (int db = 0; db < D / 32; ++db) O[db] = f32x16{};
    float m = kNone, l = 0.f;
    auto step = [&](const int key0, const int bound, const int all, const int buf) {
      const lds_u8* kb = ring + buf * C::kBuf;
      const lds_u8* vb = kb + C::kTileBytes;
      const lds_u8* sc = vb + C::kTileBytes;
      const uint32_t ksb = sc[kkey], vsb = sc[32 + kkey];
      // (a value row of scale NaN reaches the queries through its key's score)
      const float kf = __uint_as_float(max(ksb, vsb) == 255u ? 0x7fc00000u : ksb << 23);
      u32x2 vsc[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) vsc[j] = *(const VX_LDS u32x2*)(sc + 32 + 16 * j + 8 * hf);
      f32x16 S = f32x16{};
#pragma unroll
      for (int x = 0; x < D / 32; ++x) {
        const u32x4 kr = *(const VX_LDS u32x4*)(kb + kkey * D + (((2 * x + hf) ^ T::swizzle(kkey)) * 16));
        S = mfma32x32x16(e4m3x8_bf16(u32x2{kr[0], kr[1]}, kf), q[2 * x], S);
        S = mfma32x32x16(e4m3x8_bf16(u32x2{kr[2], kr[3]}, kf), q[2 * x + 1], S);
      }
      const bool slow = key0 + kFewTile > all;  // some row does not see some key (or the products are rounded)
      float cc = c;
      if (slow) {
        cc = 1.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i)
          S[i] = key0 + 16 * (i >> 3) + 8 * hf + (i & 7) < bound ? S[i] * c : -__builtin_inff();
      }
      float mx = S[0];
#pragma unroll
      for (int i = 1; i < 16; ++i) mx = fmaxf(mx, S[i]);
      mx = halves_max(mx) * cc;
      if (__builtin_amdgcn_ballot_w64(mx > m + kSlack) != 0) {
        const float mn = fmaxf(m, mx), alpha = fast_exp2(m - mn);
        m = mn;
        l *= alpha;
#pragma unroll
        for (int db = 0; db < D / 32; ++db) O[db] *= alpha;
      }
      // The weights times their value rows' scales, rounded to bf16 (a power of two changes
      // no rounding), and the sum of the rounded weights, so that those that multiply V
      // sum to one (as in many_part).
      bf16x8 P[2];
      const float mneg = -m;
      const bf16x2 one2 = {(bf16)1.0f, (bf16)1.0f};
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          float p[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            p[i] = fast_exp2(__builtin_fmaf(S[8 * j + e + i], cc, mneg));
            float w = p[i] * __uint_as_float(((vsc[j][e >> 2] >> (8 * ((e & 3) + i))) & 0xffu) << 23);
            if (slow && !(key0 + 16 * j + 8 * hf + e + i < bound)) w = 0.f;  // (its scale may be anything)
            P[j][e + i] = (bf16)w;
          }
          l = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{(bf16)p[0], (bf16)p[1]}, one2, l, false);
        }
      // V^T fragment (db, j): lane group g = lane / 16 takes dims db 32 + (g % 2) 16
      // + 0..15 of keys 16 j + 8 (g / 2) + 0..7
      const int vr = (lane & 15) >> 1, vkey0 = 8 * hf + vr;
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int db = 0; db < D / 32; ++db) {
          const int key = 16 * j + vkey0;
          typedef int i32x2 __attribute__((ext_vector_type(2)));
          const i32x2 vr8 = __builtin_amdgcn_ds_read_tr8_b64_v2i32((VX_LDS i32x2*)(
              vb + key * D + (((2 * db + ((lane >> 4) & 1)) ^ T::swizzle(key)) * 16) + (lane & 1) * 8));
          O[db] = mfma32x32x16(e4m3x8_bf16(u32x2{(uint32_t)vr8[0], (uint32_t)vr8[1]}, 1.0f), P[j], O[db]);
        }
    };

    // tile t of the part: the prefix's first, then the stream's own from `first` on
    const int here = pre_tiles + max(min(take, tiles_in<kFewTile>(any) - first), 0);
    auto stage_at = [&](int t, int buf) {
      if (BOTH && t < pre_tiles)
        stage(shared, t, buf);
      else
        stage(own, first + t - pre_tiles, buf);
    };
    const int n = here > wave ? (here - wave + W - 1) / W : 0;  // this wave's tiles
    if (n > 0) stage_at(wave, 0);
    if (n > 1) stage_at(wave + W, 1);
    for (int it = 0; it < n; ++it) {
      if (it + 1 < n)
        wait_copies<C::kPerTile>();
      else
        wait_copies<0>();
      const int t = wave + it * W;
      const bool of_prefix = BOTH && t < pre_tiles;
      step((of_prefix ? t : first + t - pre_tiles) * kFewTile, of_prefix ? shared.bound : own.bound,
           of_prefix ? shared.all : own.all, it & 1);
      if (it + 2 < n) {
        wait_lds_reads();
        stage_at(t + 2 * W, it & 1);
      }
    }

    // ---- the waves' results: rows x D through LDS, then D / 4 lanes per row
    __syncthreads();
    VX_LDS float* const xo = (VX_LDS float*)((lds_u8*)smem + wave * C::kExchange);
    const float lsum = halves_sum(l);
    if (col < rows) {
#pragma unroll
      for (int db = 0; db < D / 32; ++db)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *(VX_LDS f32x4*)(xo + col * C::kOutRow + db * 32 + 8 * g + 4 * hf) =
              f32x4{O[db][4 * g], O[db][4 * g + 1], O[db][4 * g + 2], O[db][4 * g + 3]};
      if (hf == 0) {
        ml[wave][col][0] = m;
        ml[wave][col][1] = lsum;
      }
    }
    const bool some_far = __builtin_amdgcn_ballot_w64(is_far(m)) != 0;
    if (lane == 0) far[wave] = some_far;
    __syncthreads();
    int any_far = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) any_far |= far[w];
    if (!rounded && __builtin_amdgcn_readfirstlane(any_far) != 0) {
      rounded = true;
      __syncthreads();  // (the rings take the part again)
      continue;
    }
    rounded = false;
    const bool final_rows = pt.direct && take == tiles;
    float* const part =
        final_rows ? nullptr
                   : pt.ws + ((int64_t)(pt.budget == 0 ? item : item + stream) * Hk + kvh) * part_floats(pt.rows, D);
    for (int x = threadIdx.x; x < rows * (D / 4); x += W * 64) {
      const int r = x / (D / 4), d = (x % (D / 4)) * 4;
      float M = ml[0][r][0];
#pragma unroll
      for (int w = 1; w < W; ++w) M = fmaxf(M, ml[w][r][0]);
      f32x4 o = {0.f, 0.f, 0.f, 0.f};
      float L = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float al = fast_exp2(ml[w][r][0] - M);
        L += ml[w][r][1] * al;
        o += *(const VX_LDS f32x4*)((lds_u8*)smem + w * C::kExchange + (r * C::kOutRow + d) * 4) * al;
      }
      if (final_rows) {
        int b, i, h;
        map.place(row0 + r, b, i, h);
        const float inv = is_zero(L) ? 0.f : 1.0f / L;
        bf16x4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = (bf16)(o[e] * inv);
        *(bf16x4*)((bf16*)a.o + b * a.os[0] + i * a.os[1] + h * a.os[2] + d) = y;
      } else {
        *(f32x4*)(part + (int64_t)(row0 + r) * D + d) = o;
        if (d == 0) {
          part[(int64_t)pt.rows * D + 2 * (row0 + r)] = M;
          part[(int64_t)pt.rows * D + 2 * (row0 + r) + 1] = L;
        }
      }
    }
    left -= pt.budget == 0 ? left : take;
    if (left > 0) {
      if (!next_stream(s, stream, len)) return;
      first = 0;
      __syncthreads();  // (the rings take the next part)
    }
  }
}

// ------------------------------------------------------------------ many rows
constexpr int kManyTile = 64;  // keys per tile of many_part

// A workgroup of kWaves waves of 32 rows. LDS: two K tiles, two V tiles of bf16; a
// tile is D / 64 half planes of 64 keys x 128 bytes, a row's 16-byte chunks XOR
// half_swizzle (as in flash_fwd.hip).
template <int D>
struct ManyCfg {
  static constexpr int kRows = 32 * kWaves;
  static constexpr int kHalf = kManyTile * 128;         // 64 keys x 64 dims
  static constexpr int kTileBytes = kManyTile * D * 2;  // of K, and of V
  static constexpr int kVBuf = 0, kKBuf = 2 * kTileBytes;
  static constexpr int kLoads = kManyTile * (D / 16) / kThreads;  // 16-byte chunks of K, and of V, per thread
  static constexpr int kSmem = 4 * kTileBytes;
  static constexpr int kDB = D / 32, kDS = D / 16;
  static constexpr int kPV = 4 * kDB, kQK = 2 * kDS, kSlots = kPV + kQK;
  static constexpr int kAhead = 2;  // fragments read ahead of their MFMA
};

// Tiles first .. first + take - 1 of a stream (`whole`: all it has) for rows rt
// kRows + 0 .. kRows - 1 of kv head kvh; part_no: the number of its partial result.
// False, with nothing written, if a reference point is far and the products are not
// `rounded`.
template <int D>
__device__ __forceinline__ bool many_one(const CachedAttnArgs& a, const Part& pt, const int kvh, const int rt,
                                         const int stream, const int len, const int first, const int take,
                                         const bool whole, const int part_no, const bool rounded,
                                         unsigned char* smem) {
  using C = ManyCfg<D>;
  const Streams& s = pt.s;
  const int rows = pt.rows, Hk = s.c.Hk;
  constexpr int kDB = C::kDB, kDS = C::kDS, kPV = C::kPV, kSlots = C::kSlots, kAhead = C::kAhead;
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));  // (what follows from it is formed here, not kept over the caller's loop)
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hf = lane >> 5, col = lane & 31;
  const RowMap map{a, stream, kvh, a.H / Hk, pt.per};
  bf16x8 q[kDS];
  int bound;  // keys that this lane's row sees
  {
    int rb, ri, rh;
    map.place(min(rt * C::kRows + wave * 32 + col, rows - 1), rb, ri, rh);
    bound = pt.prefix ? len : own_bound(a, rb, ri, len);
    const bf16* p = (const bf16*)a.q + rb * a.qs[0] + ri * a.qs[1] + rh * a.qs[2] + hf * 8;
#pragma unroll
    for (int ds = 0; ds < kDS; ++ds) q[ds] = *(const bf16x8*)(p + ds * 16);
  }
  int all = bound;  // keys that every row of the wave sees
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) all = min(all, __shfl_xor(all, off, 64));
  all = rounded ? 0 : __builtin_amdgcn_readfirstlane(all);
  // keys that any row of the workgroup sees
  int end = len;
  if (!pt.prefix) {
    const int m = clamp_len(a.q_len, stream, a.Sq);
    const int i0 = rt * C::kRows / map.G, i1 = min(rt * C::kRows + C::kRows - 1, rows - 1) / map.G;
    end = i0 < m ? own_bound(a, stream, min(i1, m - 1), len) : 0;
    end = __builtin_amdgcn_readfirstlane(end);
  }
  const int tiles = (end + kManyTile - 1) / kManyTile;
  const int t0 = first, n = min(take, tiles - first);
  f32x16 O[kDB];
#pragma unroll
  for (int db = 0; db < kDB; ++db) O[db] = f32x16{};
  float m_run = kNone, l_run = 0.f;
  const float c = a.scale * kLog2e;

  // ---- staging: a thread takes 16-byte chunks (16 values of one key) of K and
  // of V to registers, an iteration ahead, and converts them with the key's scale
  // on the way to LDS: once per workgroup, not once per wave. 8 lanes take four
  // chunks of keys k and k + 8, whose even (then odd) 16-byte halves the swizzle
  // sends to eight different bank groups of a cycle's 128 bytes.
  const int64_t row0 = ((int64_t)slot_of(s, stream) * Hk + kvh) * s.c.cap;
  // (uniform bases and 32-bit offsets per lane)
  const uint64_t kg = uniform_u64((uint64_t)(uintptr_t)(s.c.k + row0 * D));
  const uint64_t vg = uniform_u64((uint64_t)(uintptr_t)(s.c.v + row0 * D));
  const uint64_t ksg = uniform_u64((uint64_t)(uintptr_t)(s.c.ks + row0));
  const uint64_t vsg = uniform_u64((uint64_t)(uintptr_t)(s.c.vs + row0));
  constexpr int kPlanes = D / 64;
  // thread bits: chunk (2), key bits 3, 0, 1 and 2, plane, the key's other bits
  const int plane = kPlanes == 2 ? (tid >> 6) & 1 : 0;
  const int skey = ((tid >> 3) & 1) | (((tid >> 4) & 3) << 1) | (((tid >> 2) & 1) << 3) |
                   ((tid >> (kPlanes == 2 ? 7 : 6)) << 4);
  const int ssrc = plane * 64 + (tid & 3) * 16;                          // byte of the row
  const int sdst = plane * C::kHalf + skey * 128;
  const int sat = ((2 * (tid & 3)) ^ half_swizzle(skey)) * 16;           // its first half (the second: ^ 16)
  constexpr int kKeysPerPass = kManyTile / C::kLoads;
  struct Raw {
    u32x4 x[C::kLoads];
    uint32_t ks[C::kLoads], vs[C::kLoads];
  };
  // (through a buffer resource that ends with the last key: what lies behind
  // reads as zeros)
  const uint32_t sofs = skey * D + ssrc;
  auto load = [&](uint64_t base, int u, Raw& w) {
    const int tile = t0 + u, keys = min(end - tile * kManyTile, kManyTile);
    auto rsrc = [&](uint64_t p, int bytes) {
      return __builtin_amdgcn_make_buffer_rsrc((void*)(uintptr_t)p, 0, bytes, 0x00020000);
    };
    const auto rows_r = rsrc(base + (uint64_t)tile * (kManyTile * D), keys * D);
    const auto ks_r = rsrc(ksg + (uint64_t)tile * kManyTile, keys);
    const auto vs_r = rsrc(vsg + (uint64_t)tile * kManyTile, keys);
#pragma unroll
    for (int p = 0; p < C::kLoads; ++p) {
      w.x[p] = __builtin_amdgcn_raw_buffer_load_b128(rows_r, sofs, p * kKeysPerPass * D, 0);
      w.ks[p] = __builtin_amdgcn_raw_buffer_load_b8(ks_r, skey, p * kKeysPerPass, 0);
      w.vs[p] = __builtin_amdgcn_raw_buffer_load_b8(vs_r, skey, p * kKeysPerPass, 0);
    }
  };
  // piece j of 2 kLoads: half of a chunk to the tile at `buf`
  auto store = [&](const Raw& w, bool is_k, int buf, int j) {
    const int p = j / 2, half = j % 2;
    // (a row whose key or value has scale NaN: a NaN key; its value bytes are zeros)
    const float f = is_k ? __uint_as_float(max(w.ks[p], w.vs[p]) == 255u ? 0x7fc00000u : w.ks[p] << 23)
                         : __uint_as_float(min(w.vs[p], 254u) << 23);
    lds_u8* const row = (lds_u8*)smem + buf + p * kKeysPerPass * 128 + sdst;
    *(VX_LDS bf16x8*)(row + (half ? sat ^ 16 : sat)) =
        e4m3x8_bf16(u32x2{w.x[p][2 * half], w.x[p][2 * half + 1]}, f);
  };
  auto store_all = [&](const Raw& w, bool is_k, int buf) {
#pragma unroll
    for (int j = 0; j < 2 * C::kLoads; ++j) store(w, is_k, buf, j);
  };
  static_assert(kKeysPerPass % 16 == 0, "a pass's keys keep their swizzle");

  // ---- per-lane LDS offsets of the fragments
  const int ksw = half_swizzle(col);
  int koff[4];
#pragma unroll
  for (int d4 = 0; d4 < 4; ++d4) koff[d4] = col * 128 + (((2 * d4 + hf) ^ ksw) * 16);
  const int vr = (lane & 15) >> 2, vc = lane & 3, dh = (lane >> 4) & 1;
  int voff[2];
#pragma unroll
  for (int db1 = 0; db1 < 2; ++db1) {
    const int key = hf * 4 + vr;
    voff[db1] = key * 128 + (((4 * db1 + 2 * dh + (vc >> 1)) ^ half_swizzle(key)) * 16) + (vc & 1) * 8;
  }
  auto frag_k = [&](const lds_u8* kb, int ds, int k2) -> bf16x8 {
    return *(const VX_LDS bf16x8*)(kb + koff[ds & 3] + k2 * 32 * 128 + (ds >> 2) * C::kHalf);
  };
  auto frag_v = [&](const lds_u8* vb, int k2, int j, int db) -> bf16x8 {
    const lds_u8* p = vb + (k2 * 32 + 16 * j) * 128 + (db >> 1) * C::kHalf;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((VX_LDS s16x4*)(p + voff[db & 1]));
    const s16x4 hi4 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((VX_LDS s16x4*)(p + 8 * 128 + (voff[db & 1] ^ 16)));
    return concat(__builtin_bit_cast(bf16x4, lo), __builtin_bit_cast(bf16x4, hi4));
  };

  if (n > 0) {
    // Tile u's keys in K buffer u % 2, its values in V buffer u % 2. Iteration u
    // issues the MFMAs of PV(u - 1) and of QK^T(u + 1) in one block and the
    // softmax of tile u as a VALU block, writes K(u + 2) and V(u) (loaded in the
    // last iteration) to the buffers that iteration u - 1 read, and loads the
    // next two tiles. "V(-1)" is zeros, its weights are zeros.
    Raw wk, wv;
    Raw w0;
    load(kg, 0, w0);
    load(kg, min(1, n - 1), wk);
    const int kZero = kThreads * 16;
#pragma unroll
    for (int p = 0; p < C::kTileBytes / (kThreads * 16); ++p)
      *(VX_LDS u32x4*)((lds_u8*)smem + C::kVBuf + C::kTileBytes + p * kZero + tid * 16) = u32x4{0, 0, 0, 0};
    store_all(w0, true, C::kKBuf);
    store_all(wk, true, C::kKBuf + C::kTileBytes);
    load(kg, min(2, n - 1), wk);  // (in the loop's order)
    load(vg, 0, wv);
    __syncthreads();
    f32x16 S[2] = {f32x16{}, f32x16{}};
#pragma unroll
    for (int ds = 0; ds < kDS; ++ds)
#pragma unroll
      for (int k2 = 0; k2 < 2; ++k2) S[k2] = mfma32x32x16(frag_k((lds_u8*)smem + C::kKBuf, ds, k2), q[ds], S[k2]);
    bf16x8 Pp[2][2];
#pragma unroll
    for (int k2 = 0; k2 < 2; ++k2)
#pragma unroll
      for (int j = 0; j < 2; ++j) Pp[k2][j] = bf16x8{};

    auto iteration = [&](auto odd_tag, const int u, f32x16 (&S)[2], f32x16 (&Sn)[2], const bf16x8 (&Pp)[2][2],
                         bf16x8 (&P)[2][2]) __attribute__((always_inline)) {
      constexpr int kOdd = decltype(odd_tag)::value;  // u % 2
      // scores of a tile with a key that some row does not see: to log2 units
      // here, the unseen ones to -inf
      const int key0 = (t0 + u) * kManyTile;
      float cc = c;
      if (key0 + kManyTile > all) {
        cc = 1.0f;
#pragma unroll
        for (int k2 = 0; k2 < 2; ++k2)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            S[k2][i] = key0 + k2 * 32 + (i >> 2) * 8 + hf * 4 + (i & 3) < bound ? S[k2][i] * c : -__builtin_inff();
      }
      // The reference point of the weights moves up when a tile's maximum is
      // 2^kSlack above it. (O takes alpha after PV(u - 1), whose weights are against
      // the old point.)
      float mx = fmaxf(S[0][0], S[1][0]);
#pragma unroll
      for (int i = 1; i < 16; ++i) mx = fmaxf(fmaxf(mx, S[0][i]), S[1][i]);
      mx = halves_max(mx) * cc;
      float alpha = 1.0f;
      const bool moved = __builtin_amdgcn_ballot_w64(mx > m_run + kSlack) != 0;
      if (moved) {
        const float mn = fmaxf(m_run, mx);
        alpha = fast_exp2(m_run - mn);
        m_run = mn;
        l_run *= alpha;
      }
      __syncthreads();
      const lds_u8* kb = (const lds_u8*)smem + C::kKBuf + (1 - kOdd) * C::kTileBytes;
      const lds_u8* vb = (const lds_u8*)smem + C::kVBuf + (1 - kOdd) * C::kTileBytes;
      auto frag = [&](int x) -> bf16x8 {
        if (x < kPV) return frag_v(vb, x / (2 * kDB), (x / kDB) & 1, x % kDB);
        return frag_k(kb, (x - kPV) >> 1, (x - kPV) & 1);
      };
      // One block of kSlots MFMAs, each with the fragment kAhead MFMAs on, and
      // behind it what does not depend on it, in the cycles that the matrix core
      // takes: behind PV's the tile's weights (two exponentials and four other
      // instructions fill an MFMA's 32 cycles), behind QK^T's the conversion of the
      // next tiles, then their successors' loads. l is the sum of the rounded
      // weights, so that the ones that multiply V sum to one.
      const bf16x2 one2 = {(bf16)1.0f, (bf16)1.0f};
      const float mneg = -m_run;
      bf16x2 pk[16];
      float l2[2] = {0.f, 0.f};
      auto weights = [&](int i) {
        const float p0 = fast_exp2(__builtin_fmaf(S[i >> 3][2 * (i & 7)], cc, mneg));
        const float p1 = fast_exp2(__builtin_fmaf(S[i >> 3][2 * (i & 7) + 1], cc, mneg));
        pk[i] = bf16x2{(bf16)p0, (bf16)p1};
        l2[i & 1] = __builtin_amdgcn_fdot2_f32_bf16(pk[i], one2, l2[i & 1], false);
        asm volatile("" ::"v"(pk[i]));  // (here, not where the next iteration uses it)
      };
      // (at a higher priority than the other workgroup's waves while those are
      // between their blocks: chunk of 1000 queries on 5003 keys 145 -> 136 us)
      __builtin_amdgcn_s_setprio(1);
      bf16x8 fr[kSlots];
#pragma unroll
      for (int x = 0; x < kAhead; ++x) fr[x] = frag(x);
#pragma unroll
      for (int x = 0; x < kSlots; ++x) {
        if (x + kAhead < kSlots) fr[x + kAhead] = frag(x + kAhead);
        if (x < kPV) {
          O[x % kDB] = mfma32x32x16(fr[x], Pp[x / (2 * kDB)][(x / kDB) & 1], O[x % kDB]);
#pragma unroll
          for (int i = 0; i < 16 / kPV; ++i) weights(x * (16 / kPV) + i);
        } else {
          const int y = x - kPV;
          if (y < 2) Sn[y] = f32x16{};
          Sn[y & 1] = mfma32x32x16(fr[x], q[y >> 1], Sn[y & 1]);
          constexpr int kPieces = 4 * C::kLoads, kEvery = C::kQK / kPieces;
          if (y % kEvery == 0) {
            const int j = y / kEvery;
            if (j < kPieces / 2)
              store(wk, true, C::kKBuf + kOdd * C::kTileBytes, j);
            else
              store(wv, false, C::kVBuf + kOdd * C::kTileBytes, j - kPieces / 2);
            if (j == kPieces / 2 - 1) load(kg, min(u + 3, n - 1), wk);
            if (j == kPieces - 1) load(vg, min(u + 1, n - 1), wv);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      __builtin_amdgcn_s_setprio(0);
      l_run += l2[0] + l2[1];
      if (moved) {
#pragma unroll
        for (int db = 0; db < kDB; ++db) O[db] *= alpha;
      }
#pragma unroll
      for (int k2 = 0; k2 < 2; ++k2)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int x = k2 * 8 + j * 4;
          P[k2][j] = __builtin_shufflevector(__builtin_shufflevector(pk[x], pk[x + 1], 0, 1, 2, 3),
                                             __builtin_shufflevector(pk[x + 2], pk[x + 3], 0, 1, 2, 3), 0, 1, 2, 3, 4,
                                             5, 6, 7);
        }
    };
    f32x16 S2[2];
    bf16x8 P2[2][2];
    using Even = std::integral_constant<int, 0>;
    using Odd = std::integral_constant<int, 1>;
    auto last_pv = [&](auto odd_tag, const bf16x8 (&P)[2][2]) __attribute__((always_inline)) {
      __syncthreads();
      const lds_u8* vb = (const lds_u8*)smem + C::kVBuf + decltype(odd_tag)::value * C::kTileBytes;
#pragma unroll
      for (int x = 0; x < kPV; ++x)
        O[x % kDB] =
            mfma32x32x16(frag_v(vb, x / (2 * kDB), (x / kDB) & 1, x % kDB), P[x / (2 * kDB)][(x / kDB) & 1], O[x % kDB]);
    };
    int u = 0;
    for (; u + 1 < n; u += 2) {
      iteration(Even{}, u, S, S2, Pp, P2);
      iteration(Odd{}, u + 1, S2, S, P2, Pp);
    }
    if (u < n) {
      iteration(Even{}, u, S, S2, Pp, P2);
      last_pv(Even{}, P2);
    } else {
      last_pv(Odd{}, Pp);
    }
    if (!rounded) {
      // (one answer for the workgroup, whose waves share the tiles)
      VX_LDS int* const far = (VX_LDS int*)(lds_u8*)smem;
      __syncthreads();
      far[wave] = __builtin_amdgcn_ballot_w64(is_far(m_run)) != 0;
      __syncthreads();
      int any_far = 0;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) any_far |= far[w];
      if (__builtin_amdgcn_readfirstlane(any_far) != 0) return false;
    }
  }

  const float L = halves_sum(l_run);
  const int r = rt * C::kRows + wave * 32 + col;
  if (pt.direct && whole) {
    int rb, ri, rh;
    map.place(min(r, rows - 1), rb, ri, rh);
    const float inv = is_zero(L) ? 0.f : 1.0f / L;
    u32x4 out[kDB][2];
    pack_out_rows<kDB>(O, inv, out);
    if (r < rows) {
      bf16* const o = (bf16*)a.o + rb * a.os[0] + ri * a.os[1] + rh * a.os[2];
#pragma unroll
      for (int db = 0; db < kDB; ++db)
#pragma unroll
        for (int pr = 0; pr < 2; ++pr) *(u32x4*)(o + db * 32 + 8 * (2 * pr + hf)) = out[db][pr];
    }
  } else if (r < rows) {
    float* const part =
        pt.ws + ((int64_t)part_no * Hk + kvh) * part_floats(rows, D);
#pragma unroll
    for (int db = 0; db < kDB; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *(f32x4*)(part + (int64_t)r * D + db * 32 + 8 * g + 4 * hf) =
            f32x4{O[db][4 * g], O[db][4 * g + 1], O[db][4 * g + 2], O[db][4 * g + 3]};
    if (hf == 0) {
      part[(int64_t)rows * D + 2 * r] = m_run;
      part[(int64_t)rows * D + 2 * r + 1] = L;
    }
  }
  return true;
}

// A range of tiles of streams of more rows, for one tile of rows of one kv head.
template <int D>
__device__ __forceinline__ void many_part(const CachedAttnArgs& a, const Part& pt, const int block,
                                          unsigned char* smem) {
  const int Hk = pt.s.c.Hk;
  const int n_rt = (pt.rows + ManyCfg<D>::kRows - 1) / ManyCfg<D>::kRows;
  // Order: a prompt's last row tiles, which see the most keys, first; kv heads
  // side by side, so that with 8 of them each XCD keeps one head's keys in its L2.
  // Where all workgroups find a place at once (two per CU), the second half runs
  // the other way, so that a long one shares its CU with a short one.
  const int kvh = __builtin_amdgcn_readfirstlane(block % Hk);
  int place = block / Hk;
  if (pt.one_round) {
    const int all_places = pt.items * n_rt, half = all_places / 2;
    if (place >= half) place = half + all_places - 1 - place;
  }
  const int rt = __builtin_amdgcn_readfirstlane(n_rt - 1 - place / pt.items);
  const int item = __builtin_amdgcn_readfirstlane(place % pt.items);
  const Range range =
      pt.budget == 0 ? whole_stream(pt.s, item) : range_of<kManyTile>(pt.s, pt.budget, pt.min_chunk, item);
  int stream = range.stream, len = range.len, first = range.tile, left = range.tiles;
  bool rounded = false;
  while (left > 0) {
    const int tiles = tiles_in<kManyTile>(len), take = pt.budget == 0 ? tiles : min(left, tiles - first);
    if (!many_one<D>(a, pt, kvh, rt, stream, len, first, take, take == tiles, pt.budget == 0 ? item : item + stream,
                     rounded, smem)) {
      rounded = true;
      __syncthreads();  // (the tiles' buffers take the part again)
      continue;
    }
    rounded = false;
    left -= pt.budget == 0 ? left : take;
    if (left > 0) {
      if (!next_stream(pt.s, stream, len)) return;
      first = 0;
      __syncthreads();  // (the tiles' buffers take the next part)
    }
  }
}

// BOTH: prefixes and items of few positions in one pass, the prefix read (from
// the L2) by each item rather than merged. W: eight waves where the grid leaves a
// CU to each workgroup.
template <int D, int W, bool BOTH>
__global__ __launch_bounds__(W * 64, 2) void few_kernel(const CachedAttnArgs a, const Part own, const Part pre) {
  __shared__ __attribute__((aligned(256))) unsigned char smem[FewCfg<D, W>::kSmem];
  few_part<D, W, BOTH>(a, own, &pre, blockIdx.x, smem);
}

template <int D>
__global__ __launch_bounds__(kThreads, 2) void many_kernel(const CachedAttnArgs a, const Part own) {
  __shared__ __attribute__((aligned(256))) unsigned char smem[ManyCfg<D>::kSmem];
  many_part<D>(a, own, blockIdx.x, smem);
}

// A prefix's chunks (the first pre_blocks workgroups) and the items' own, side by
// side: the prefix alone would leave most of the chip idle, and so would they.
template <int D, bool PRE_FEW, bool OWN_FEW>
__global__ __launch_bounds__(kThreads, 2) void prefix_kernel(const CachedAttnArgs a, const Part pre, const Part own,
                                                           const int pre_blocks) {
  constexpr int kFew = FewCfg<D, kWaves>::kSmem, kMany = ManyCfg<D>::kSmem;
  constexpr int kPre = PRE_FEW ? kFew : kMany, kOwn = OWN_FEW ? kFew : kMany;
  __shared__ __attribute__((aligned(256))) unsigned char smem[kPre > kOwn ? kPre : kOwn];
  const int block = blockIdx.x;
  if (block < pre_blocks) {
    if constexpr (PRE_FEW)
      few_part<D, kWaves, false>(a, pre, nullptr, block, smem);
    else
      many_part<D>(a, pre, block, smem);
  } else {
    if constexpr (OWN_FEW)
      few_part<D, kWaves, false>(a, own, nullptr, block - pre_blocks, smem);
    else
      many_part<D>(a, own, block - pre_blocks, smem);
  }
}

// ------------------------------------------------------------------ merge
// Output rows of item blockIdx.y from the parts of the item's own chunks and of
// its group's prefix chunks. D / 4 lanes take a row; `split` such groups share
// the parts of a row, and join in LDS, in a fixed order.
template <int D>
__global__ __launch_bounds__(kThreads) void merge_kernel(const CachedAttnArgs a, const Part own, const Part pre,
                                                       const int split) {
  constexpr int kLanes = D / 4, kGroups = kThreads / kLanes;
  __shared__ f32x4 xo[kGroups][kLanes];
  __shared__ float xml[kGroups][2];
  const int b = blockIdx.y, Hk = a.c.Hk, G = a.H / Hk;
  const Parts oc = own.few ? parts_of<kFewTile>(own.s, own.budget, own.min_chunk, b)
                           : parts_of<kManyTile>(own.s, own.budget, own.min_chunk, b);
  const bool with_prefix = pre.s.n > 0;
  if (!with_prefix && oc.count == 1) return;  // (written by the part itself)
  Parts pc{0, 0};
  if (with_prefix)
    pc = pre.few ? parts_of<kFewTile>(pre.s, pre.budget, pre.min_chunk, b / pre.per)
                 : parts_of<kManyTile>(pre.s, pre.budget, pre.min_chunk, b / pre.per);
  const int group = threadIdx.x / kLanes, d = (threadIdx.x % kLanes) * 4;
  const int part0 = group % split;
  const int64_t x = (int64_t)blockIdx.x * (kGroups / split) + group / split;
  const bool real = x < (int64_t)Hk * own.rows;
  const int kvh = real ? (int)(x / own.rows) : 0, r = real ? (int)(x - (int64_t)kvh * own.rows) : 0;
  float M = kNone, L = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  const int total = real ? pc.count + oc.count : 0;
  const int64_t pre_block = part_floats(pre.rows, D), own_block = part_floats(own.rows, D);
  const int pre_row = with_prefix ? (b % pre.per) * own.rows + r : 0;
#pragma unroll 4
  for (int n = part0; n < total; n += split) {
    const bool p = n < pc.count;
    const int64_t block = p ? pre_block : own_block, rows = p ? pre.rows : own.rows;
    const int64_t at = (int64_t)(p ? pc.first + n : oc.first + n - pc.count) * Hk + kvh;
    const float* part = (p ? pre.ws : own.ws) + at * block;
    const int row = p ? pre_row : r;
    const f32x4 po = *(const f32x4*)(part + (int64_t)row * D + d);
    const float pm = part[rows * D + 2 * row], pl = part[rows * D + 2 * row + 1];
    const float mn = fmaxf(M, pm), a0 = fast_exp2(M - mn), a1 = fast_exp2(pm - mn);
    o = o * a0 + po * a1;
    L = L * a0 + pl * a1;
    M = mn;
  }
  if (split > 1) {
    xo[group][threadIdx.x % kLanes] = o;
    if (d == 0) {
      xml[group][0] = M;
      xml[group][1] = L;
    }
    __syncthreads();
    if (part0 != 0) return;
    for (int g = 1; g < split; ++g) {
      const float pm = xml[group + g][0], pl = xml[group + g][1];
      const float mn = fmaxf(M, pm), a0 = fast_exp2(M - mn), a1 = fast_exp2(pm - mn);
      o = o * a0 + xo[group + g][threadIdx.x % kLanes] * a1;
      L = L * a0 + pl * a1;
      M = mn;
    }
  }
  if (!real) return;
  const int i = r / G, h = kvh * G + r % G;
  const bool none = is_zero(L) || i >= clamp_len(a.q_len, b, a.Sq);
  const float inv = 1.0f / L;
  bf16x4 y;
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = (bf16)(none ? 0.f : o[e] * inv);
  *(bf16x4*)((bf16*)a.o + b * a.os[0] + i * a.os[1] + h * a.os[2] + d) = y;
}

// ------------------------------------------------------------------ launch plan
constexpr int kManyRows = 32 * kWaves;
// Caches of up to this many 32-key tiles are one item per stream of few rows: at
// 1024 positions (eight tiles a wave) the launch that would merge costs more than
// the parts save (12 heads, 700 keys: 11.5 us a call, with parts 15.5).
constexpr int kFewWhole = 32;

// Fills a part's plan; returns its workgroups.
struct Planned {
  Part p{};
  int64_t blocks = 0;
  int64_t floats = 0;  // of partial results
  int usual_parts = 1;  // of a stream
};

// Ranges that a stream is cut into, `groups` workgroups without a cut: the number
// for which a model of the time is least. A workgroup has `steps` steps that take
// t1 us each where its CU holds no other, t2 where it holds two; the merging launch
// takes 6 us, and the partial results (rows x D of fp32 per workgroup) are written and
// read at 4 TB/s. (12 heads, 2048 queries: 512 keys in two ranges 37 us, in one 15; a
// prefix of 4001 and 3520 keys under 1024 rows and 8 heads in 2, 4, 6 and 8 ranges
// 86, 60, 66 and 69 us; 8192 keys under 128 rows and 8 heads in 8, 16 and 24 23, 29
// and 32 us with few_kernel.)
int64_t best_ranges(int64_t groups, int64_t steps, double t1, double t2, int64_t rows, int D, int64_t slots,
                    int64_t cus) {
  int64_t best = 1;
  double least = 0;
  for (int64_t k = 1; k * 2 <= steps && (k == 1 || groups * k <= slots); k += 1 + k / 8) {
    const double crowded = std::min(1.0, std::max(0.0, (double)(groups * k - cus) / (double)cus));
    const double t = (double)((steps + k - 1) / k) * (t1 + (t2 - t1) * crowded) * D / 128 +
                     (k > 1 ? 6 + 2.0 * (double)(groups * k) * (double)rows * (D + 2) * 4 / 4e6 : 0);
    if (k == 1 || t < least) best = k, least = t;
  }
  return best;
}

// Whether few_kernel takes rows so many. In the time that a CU takes for a tile of
// 64 keys and 128 rows with many_kernel (1.05 us with two workgroups, head dim
// 128), it takes ten 32 x 32 tiles with few_kernel (1.65 us for eight waves'): 2.5
// row tiles. So up to 64 rows and a little past each 128 few_kernel wins whatever
// the length; at 128 rows while its shorter start and fewer partial results (about
// 5 us) outweigh that (32 sharers' 128 rows on 8192 keys of 8 heads 22.7 us, with
// many_kernel 25.7; 1024 rows on 4001 keys 67 and 60; 4000 rows on 5003 210 and 139).
bool runs_few(int64_t heads, int64_t rows, int64_t cap, int D, int64_t cus) {
  if (rows <= 32) return true;
  const double x = (double)(heads * ((cap + kManyTile - 1) / kManyTile)) / (double)cus * D / 128;
  return 0.4125 * (double)((rows + 31) / 32) * x < 1.05 * (double)((rows + kManyRows - 1) / kManyRows) * x + 5;
}

Planned plan_part(int streams, int64_t rows, int per, int cap, int Hk, int D, int64_t slots, int64_t cus, bool prefix,
                  bool with_prefix) {
  Planned h;
  Part& p = h.p;
  p.rows = (int)rows;
  p.per = per;
  p.few = runs_few(streams * (int64_t)Hk, rows, cap, D, cus);
  p.prefix = prefix;
  p.direct = !with_prefix;
  const int64_t row_tiles = p.few ? (rows + 31) / 32 : (rows + kManyRows - 1) / kManyRows;
  const int64_t tile = p.few ? kFewTile : kManyTile;
  const int64_t tiles = (cap + tile - 1) / tile, groups = streams * row_tiles * Hk;
  p.min_chunk = p.few ? 4 : 2;
  if (p.few && row_tiles == 1) {
    // (partial results of few rows: as many ranges as find a place)
    if (tiles > kFewWhole)
      p.budget = (int)std::min<int64_t>(std::max<int64_t>(slots / Hk, 1),
                                        streams * ((tiles + p.min_chunk - 1) / p.min_chunk));
  } else {
    const int64_t k = p.few ? best_ranges(groups, (tiles + kWaves - 1) / kWaves, 0.9, 1.65, 32, D, slots, cus)
                            : best_ranges(groups, tiles, 1.3, 2.1, kManyRows, D, slots, cus);
    if (k > 1) p.budget = (int)(k * streams);
  }
  p.items = p.budget != 0 ? p.budget : streams;
  h.usual_parts = p.budget / streams + 1;
  h.blocks = p.items * row_tiles * Hk;
  p.one_round = h.blocks <= slots;
  // (part numbers go up to budget + streams - 2)
  const int64_t parts = p.budget != 0 ? p.budget + (int64_t)streams - 1 : streams;
  if (with_prefix || p.budget > 0) h.floats = parts * Hk * ((rows * (D + 2) + 3) & ~(int64_t)3);
  return h;
}

struct Plan {
  Planned own, pre;
  bool both = false;  // few_kernel<D, W, true>
  bool wide = false;  // few_kernel's W: 8, else 4
};

Plan plan_of(int cap, int n_prefix, int p_cap, int B, int Sq, int H, int Hk, int D) {
  const int64_t cus = device_cu_count() > 0 ? device_cu_count() : 256;
  const int64_t slots = 2 * cus;  // workgroups that the device holds at once
  const int64_t rows = (int64_t)Sq * (H / Hk);
  Plan p;
  p.own = plan_part(B, rows, 1, cap, Hk, D, slots, cus, false, n_prefix > 0);
  // Eight waves where each workgroup has a CU to itself and its waves several tiles
  // (8 / 4 waves: 12 heads, 700 keys 10.2 / 10.6 us; 16 items of 8 queries and 64
  // heads on 4096 keys 38 / 44; 8 of 40 queries on 1500 keys of 8 heads 17.3 / 18.7)
  const int64_t few_tiles = ((int64_t)cap + (n_prefix > 0 ? p_cap : 0)) / kFewTile;
  p.wide = p.own.p.few && p.own.blocks <= cus && p.own.p.budget == 0 && few_tiles > kWaves;
  if (n_prefix == 0) return p;
  const int per = B / n_prefix;
  // (each item then reads its group's whole prefix: streams that are not cut)
  if (rows <= 32 && few_tiles <= kFewWhole && (int64_t)B * Hk <= slots) {
    p.both = true;
    p.own = plan_part(B, rows, 1, cap, Hk, D, slots, cus, false, false);
    p.pre.p.per = per;
    return p;
  }
  // The prefix takes what the items' own workgroups leave, where they are whole
  // streams on at most half of the chip: all start at once. Otherwise each takes
  // its share of the positions (by the capacities; three times as heavy where 128
  // rows read them).
  const int64_t pre_rows = rows * per;
  const auto weight = [&](int64_t streams, int64_t r, int64_t c) {
    return streams * c * (r <= 32 ? 1 : 3 * ((r + kManyRows - 1) / kManyRows));
  };
  const int64_t w_pre = weight(n_prefix, pre_rows, p_cap), w_own = weight(B, rows, cap);
  int64_t pre_slots = std::max<int64_t>(slots * w_pre / (w_pre + w_own), 1);
  if (p.own.p.budget > 0)
    p.own = plan_part(B, rows, 1, cap, Hk, D, std::max<int64_t>(slots - pre_slots, 1), cus, false, true);
  else if (p.own.blocks <= slots / 2)
    pre_slots = slots - p.own.blocks;
  p.pre = plan_part(n_prefix, pre_rows, per, p_cap, Hk, D, pre_slots, cus, true, true);
  return p;
}

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
    constexpr int kGroups = kThreads / (D / 4);
    int split = 1;  // about four parts in turn per group of lanes
    while (split < kGroups && 4 * split < pl.own.usual_parts + (n_prefix > 0 ? pl.pre.usual_parts : 0)) split *= 2;
    const int64_t per_wg = kGroups / split;
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
