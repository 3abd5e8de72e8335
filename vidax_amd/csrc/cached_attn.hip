// Attention over the 8-bit key/value cache for gfx950, bf16 queries and output,
// D = 128 or 64.
//
// The query rows that share a cached head's keys -- the G heads of a group times
// the queries of an item, for a prefix times the items that share it -- form a
// stream's rows; its keys are cut into chunks, one workgroup each:
//
//   few_kernel   streams of at most 32 rows (single tokens): four waves, each on
//                every fourth 32-key tile of the chunk with all the rows
//   many_kernel  more rows (prompts in chunks, cross-attention, a prefix under a
//                batch): four waves of 32 rows each on the same 64-key tiles
//   merge_kernel joins the chunks of a stream, and a prefix's with the items'
//
// All compute S^T = K Q^T and O^T = V^T P^T with v_mfma_f32_32x32x16_bf16, so that a
// lane holds one query row: its maximum, sum and rescaling are the lane's own,
// and the two halves of a wave exchange them by one v_permlane32_swap. e4m3
// values are exact in bf16, and so are they times a power of two, so the only
// roundings are the weights' and the output's to bf16.
//
// Chunks. All streams' key tiles are cut evenly: chunk = total tiles / budget,
// with the lengths read on the device by every workgroup (one load and a scan
// over the lanes), so that no launch depends on lengths that the host does not
// know, and one long sequence in a batch of short ones is spread over the chip
// like the others.
#include "vx_fp8_cache.hpp"
#include "vx_kernels.h"

#include <algorithm>

namespace vx {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * 64;
constexpr float kNegBig = -1.0e30f;  // finite "no key seen yet" reference point
constexpr float kSlack = 8.0f;       // weights up to 2^kSlack before the reference point moves

typedef VX_LDS unsigned char lds_u8;

template <int N>
__device__ __forceinline__ void wait_copies() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void wait_lds_reads() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

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

// How the streams' key tiles (TILE keys each) are cut: every stream into
// items of `chunk` tiles (at least one), numbered one after another.
struct Cut {
  int chunk;
  int first, count;  // items of the stream that was asked for
};

// The items of stream `want`. Every wave works this out for itself, 64 streams
// per step. budget 0: one item per stream.
template <int TILE>
__device__ __forceinline__ Cut cut_of(const Streams& s, int budget, int min_chunk, int want) {
  if (budget == 0) return Cut{0x7fffffff, want, 1};
  const int lane = threadIdx.x & 63;
  int64_t total = 0;
  int mine = 0;
  for (int i0 = 0; i0 < s.n; i0 += 64) {
    const int t = i0 + lane < s.n ? (keys_of(s, i0 + lane) + TILE - 1) / TILE : 0;
    if (s.n <= 64) mine = t;
    int64_t x = t;
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) x += __shfl_xor(x, off, 64);
    total += x;
  }
  Cut c{(int)max((total + budget - 1) / budget, (int64_t)min_chunk), 0, 0};
  for (int i0 = 0; i0 <= want; i0 += 64) {
    const int i = i0 + lane;
    if (s.n > 64) mine = i < s.n ? (keys_of(s, i) + TILE - 1) / TILE : 0;
    const int items = i < s.n ? max((mine + c.chunk - 1) / c.chunk, 1) : 0;
    int before = i < want ? items : 0;
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) before += __shfl_xor(before, off, 64);
    c.first += before;
    if (want - i0 < 64) c.count = __shfl(items, want - i0, 64);
  }
  return c;
}

// The stream of item `item` and its cut (stream -1: there is no such item).
template <int TILE>
__device__ __forceinline__ int stream_of(const Streams& s, int budget, int min_chunk, int item, Cut& c) {
  if (budget == 0) {
    c = Cut{0x7fffffff, item, 1};
    return item < s.n ? item : -1;
  }
  const int lane = threadIdx.x & 63;
  int64_t total = 0;
  int mine = 0;
  for (int i0 = 0; i0 < s.n; i0 += 64) {
    mine = i0 + lane < s.n ? (keys_of(s, i0 + lane) + TILE - 1) / TILE : 0;
    int64_t x = mine;
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) x += __shfl_xor(x, off, 64);
    total += x;
  }
  c.chunk = (int)max((total + budget - 1) / budget, (int64_t)min_chunk);
  int base = 0;
  for (int i0 = 0; i0 < s.n; i0 += 64) {
    const int i = i0 + lane;
    if (s.n > 64) mine = i < s.n ? (keys_of(s, i) + TILE - 1) / TILE : 0;
    const int items = i < s.n ? max((mine + c.chunk - 1) / c.chunk, 1) : 0;
    int upto = items;  // inclusive scan over the lanes
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int o = __shfl_up(upto, off, 64);
      if (lane >= off) upto += o;
    }
    const uint64_t past = __builtin_amdgcn_ballot_w64(base + upto > item);
    if (past != 0) {
      const int l = __builtin_ctzll(past);
      c.count = __shfl(items, l, 64);
      c.first = base + __shfl(upto, l, 64) - c.count;
      return i0 + l;
    }
    base += __shfl(upto, 63, 64);
  }
  return -1;
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

// Partial results in the workspace, one block per (item, kv head): rows x D
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

template <int D>
struct FewCfg {
  static constexpr int kTileBytes = kFewTile * D;        // of K, and of V
  static constexpr int kCopies = kTileBytes / 1024;      // DMA copies of each
  static constexpr int kPerTile = 2 * kCopies + 1;       // ... of a tile, with its scales
  static constexpr int kBuf = 2 * kTileBytes + 128;      // K, V, 32 + 32 scale bytes
  static constexpr int kRing = 2;
  static constexpr int kOutRow = D + 4;                  // fp32 values between rows of the exchange
  static constexpr int kExchange = 32 * kOutRow * 4;
  static constexpr int kSmem = (kRing * kBuf > kExchange ? kRing * kBuf : kExchange) * kWaves;
};

// One wave's softmax state and the step over 32 keys.
template <int D>
struct FewState {
  bf16x8 q[D / 16];
  f32x16 O[D / 32];
  float m, l;
};

template <int D>
__global__ __launch_bounds__(kThreads, 2) void few_kernel(const CachedAttnArgs a, const Streams s, const int rows,
                                                        const int per, const int prefix, const int budget,
                                                        const int min_chunk, const int direct, float* ws) {
  using C = FewCfg<D>;
  using T = Fp8Tile<D>;
  __shared__ __attribute__((aligned(256))) unsigned char smem[C::kSmem];
  __shared__ float ml[kWaves][32][2];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hf = lane >> 5, col = lane & 31;
  const int kvh = blockIdx.y, Hk = s.c.Hk;
  Cut cut;
  const int stream = __builtin_amdgcn_readfirstlane(stream_of<kFewTile>(s, budget, min_chunk, blockIdx.x, cut));
  if (stream < 0) return;  // (the whole workgroup)
  const int len = __builtin_amdgcn_readfirstlane(keys_of(s, stream));
  const int tiles = (len + kFewTile - 1) / kFewTile;
  const int chunk_no = blockIdx.x - __builtin_amdgcn_readfirstlane(cut.first);
  const int chunk = __builtin_amdgcn_readfirstlane(cut.chunk);
  const int t0 = min((int64_t)chunk_no * chunk, (int64_t)tiles);
  const int t1 = min((int64_t)t0 + chunk, (int64_t)tiles);

  const RowMap map{a, stream, kvh, a.H / Hk, per};
  int rb, ri, rh;
  map.place(min(col, rows - 1), rb, ri, rh);
  FewState<D> st;
  {
    const bf16* q = (const bf16*)a.q + rb * a.qs[0] + ri * a.qs[1] + rh * a.qs[2] + hf * 16;
#pragma unroll
    for (int x = 0; x < D / 32; ++x) {
      st.q[2 * x] = *(const bf16x8*)(q + 32 * x);
      st.q[2 * x + 1] = *(const bf16x8*)(q + 32 * x + 8);
    }
  }
  // keys this lane's row sees, and those that every row sees
  const int bound = prefix ? len : own_bound(a, rb, ri, len);
  int all = bound;
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) all = min(all, __shfl_xor(all, off, 64));
  all = __builtin_amdgcn_readfirstlane(all);
#pragma unroll
  for (int db = 0; db < D / 32; ++db) st.O[db] = f32x16{};
  st.m = kNegBig;
  st.l = 0.f;

  // ---- staging: copy p of a tile fills 1024 / D rows; lane L takes row L / (D / 16),
  // LDS chunk L % (D / 16), which holds the row's chunk with that number XOR the swizzle
  const int64_t row0 = ((int64_t)slot_of(s, stream) * Hk + kvh) * s.c.cap;
  const uint64_t k_addr = uniform_u64((uint64_t)(uintptr_t)(s.c.k + row0 * D));
  const uint64_t v_addr = uniform_u64((uint64_t)(uintptr_t)(s.c.v + row0 * D));
  lds_u8* const ring = (lds_u8*)smem + wave * C::kRing * C::kBuf;
  const uint32_t ring_addr = (uint32_t)(uintptr_t)ring;
  const uint8_t* scale_src = (lane & 2 ? s.c.vs : s.c.ks) + row0 + 16 * (lane & 1);
  auto stage = [&](int t, int buf) {
    const uint32_t dst = ring_addr + buf * C::kBuf;
    const int last = len - 1 - t * kFewTile;  // last row of the tile that holds a key
    const i32x4_rsrc rk = raw_rsrc_u64(k_addr + (uint64_t)t * C::kTileBytes);
    const i32x4_rsrc rv = raw_rsrc_u64(v_addr + (uint64_t)t * C::kTileBytes);
#pragma unroll
    for (int p = 0; p < C::kCopies; ++p) {
      const int r = p * (1024 / D) + lane / T::kChunks;
      // (rows past the last key repeat it: what lies there may be anything)
      const uint32_t off = (uint32_t)(min(r, last) * D + ((lane % T::kChunks) ^ T::swizzle(r)) * 16);
      lds_dma16_buf(rk, off, dst + p * 1024);
      lds_dma16_buf(rv, off, dst + C::kTileBytes + p * 1024);
    }
    if (lane < 4) lds_dma16(scale_src + (int64_t)t * kFewTile, dst + 2 * C::kTileBytes);
  };

  const float c = a.scale * kLog2e;
  // K fragment row of this lane: MFMA row x holds key (x with bits 2 and 3
  // swapped), so that a lane's 16 scores are keys 16 j + 8 hf + 0..7, j = 0, 1:
  // the order in which the B operand of PV takes its weights
  const int kkey = (col & 0x13) | ((col & 4) << 1) | ((col & 8) >> 1);
  auto step = [&](int t, int buf) {
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
      S = mfma32x32x16(e4m3x8_bf16(u32x2{kr[0], kr[1]}, kf), st.q[2 * x], S);
      S = mfma32x32x16(e4m3x8_bf16(u32x2{kr[2], kr[3]}, kf), st.q[2 * x + 1], S);
    }
    const int key0 = t * kFewTile;
    const bool slow = key0 + kFewTile > all;  // some row does not see some key
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
    if (__builtin_amdgcn_ballot_w64(mx > st.m + kSlack) != 0) {
      const float mn = fmaxf(st.m, mx), alpha = fast_exp2(st.m - mn);
      st.m = mn;
      st.l *= alpha;
#pragma unroll
      for (int db = 0; db < D / 32; ++db) st.O[db] *= alpha;
    }
    bf16x8 P[2];
    const float mneg = -st.m;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float p = fast_exp2(__builtin_fmaf(S[8 * j + e], cc, mneg));
        st.l += p;
        float w = p * __uint_as_float(((vsc[j][e >> 2] >> (8 * (e & 3))) & 0xffu) << 23);
        if (slow && !(key0 + 16 * j + 8 * hf + e < bound)) w = 0.f;  // (its scale may be anything)
        P[j][e] = (bf16)w;
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
        st.O[db] = mfma32x32x16(e4m3x8_bf16(u32x2{(uint32_t)vr8[0], (uint32_t)vr8[1]}, 1.0f), P[j], st.O[db]);
      }
  };

  const int n = t1 - t0 > wave ? (t1 - t0 - wave + kWaves - 1) / kWaves : 0;  // this wave's tiles
  if (n > 0) stage(t0 + wave, 0);
  if (n > 1) stage(t0 + wave + kWaves, 1);
  for (int it = 0; it < n; ++it) {
    if (it + 1 < n)
      wait_copies<C::kPerTile>();
    else
      wait_copies<0>();
    step(t0 + wave + it * kWaves, it & 1);
    if (it + 2 < n) {
      wait_lds_reads();
      stage(t0 + wave + (it + 2) * kWaves, it & 1);
    }
  }

  // ---- the four waves' results: rows x D through LDS, then D / 4 lanes per row
  __syncthreads();
  VX_LDS float* const xo = (VX_LDS float*)((lds_u8*)smem + wave * C::kExchange);
  const float lsum = halves_sum(st.l);
  if (col < rows) {
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *(VX_LDS f32x4*)(xo + col * C::kOutRow + db * 32 + 8 * g + 4 * hf) =
            f32x4{st.O[db][4 * g], st.O[db][4 * g + 1], st.O[db][4 * g + 2], st.O[db][4 * g + 3]};
    if (hf == 0) {
      ml[wave][col][0] = st.m;
      ml[wave][col][1] = lsum;
    }
  }
  __syncthreads();
  const bool final_rows = direct && cut.count == 1;
  float* const part = final_rows ? nullptr : ws + ((int64_t)blockIdx.x * Hk + kvh) * part_floats(rows, D);
  for (int x = threadIdx.x; x < rows * (D / 4); x += kThreads) {
    const int r = x / (D / 4), d = (x % (D / 4)) * 4;
    float M = ml[0][r][0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) M = fmaxf(M, ml[w][r][0]);
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    float L = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float al = fast_exp2(ml[w][r][0] - M);
      L += ml[w][r][1] * al;
      o += *(const VX_LDS f32x4*)((lds_u8*)smem + w * C::kExchange + (r * C::kOutRow + d) * 4) * al;
    }
    if (final_rows) {
      int b, i, h;
      map.place(r, b, i, h);
      const float inv = is_zero(L) ? 0.f : 1.0f / L;
      bf16x4 y;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = (bf16)(o[e] * inv);
      *(bf16x4*)((bf16*)a.o + b * a.os[0] + i * a.os[1] + h * a.os[2] + d) = y;
    } else {
      *(f32x4*)(part + r * D + d) = o;
      if (d == 0) {
        part[(int64_t)rows * D + 2 * r] = M;
        part[(int64_t)rows * D + 2 * r + 1] = L;
      }
    }
  }
}

// ------------------------------------------------------------------ many rows
constexpr int kManyTile = 64;             // keys per tile of many_kernel
constexpr int kManyRows = 32 * kWaves;    // rows per workgroup

template <int D>
struct ManyCfg {
  static constexpr int kHalf = kManyTile * 128;          // 64 keys x 64 dims of bf16
  static constexpr int kTileBytes = kManyTile * D * 2;   // of K, and of V
  static constexpr int kBuf = 2 * kTileBytes;
  static constexpr int kLoads = kManyTile * (D / 16) / kThreads;  // 16-byte chunks of K, and of V, per thread
  static constexpr int kSmem = 2 * kBuf;
};

template <int D>
__global__ __launch_bounds__(kThreads, 2) void many_kernel(const CachedAttnArgs a, const Streams s, const int rows,
                                                         const int per, const int prefix, const int budget,
                                                         const int min_chunk, const int direct, float* ws) {
  using C = ManyCfg<D>;
  __shared__ __attribute__((aligned(256))) unsigned char smem[C::kSmem];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hf = lane >> 5, col = lane & 31;
  const int kvh = blockIdx.y, Hk = s.c.Hk;
  const int n_rt = (rows + kManyRows - 1) / kManyRows;
  const int item = blockIdx.x / n_rt;
  // (a prompt's last row tiles see the most keys: they start first)
  const int rt = n_rt - 1 - (int)(blockIdx.x - item * n_rt);
  Cut cut;
  const int stream = __builtin_amdgcn_readfirstlane(stream_of<kManyTile>(s, budget, min_chunk, item, cut));
  if (stream < 0) return;
  const int len = __builtin_amdgcn_readfirstlane(keys_of(s, stream));
  const RowMap map{a, stream, kvh, a.H / Hk, per};
  const int r = rt * kManyRows + wave * 32 + col;
  int rb, ri, rh;
  map.place(min(r, rows - 1), rb, ri, rh);
  bf16x8 q[D / 16];
  {
    const bf16* p = (const bf16*)a.q + rb * a.qs[0] + ri * a.qs[1] + rh * a.qs[2] + hf * 8;
#pragma unroll
    for (int ds = 0; ds < D / 16; ++ds) q[ds] = *(const bf16x8*)(p + ds * 16);
  }
  const int bound = prefix ? len : own_bound(a, rb, ri, len);
  int all = bound, any = bound;  // keys that every row of the wave sees, and that any does
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) {
    all = min(all, __shfl_xor(all, off, 64));
    any = max(any, __shfl_xor(any, off, 64));
  }
  all = __builtin_amdgcn_readfirstlane(all);
  any = __builtin_amdgcn_readfirstlane(any);
  // keys that any row of the workgroup sees
  int end = len;
  if (!prefix) {
    const int m = clamp_len(a.q_len, stream, a.Sq);
    const int i0 = rt * kManyRows / map.G, i1 = min(rt * kManyRows + kManyRows - 1, rows - 1) / map.G;
    end = i0 < m ? own_bound(a, stream, min(i1, m - 1), len) : 0;
    end = __builtin_amdgcn_readfirstlane(end);
  }
  const int tiles = (end + kManyTile - 1) / kManyTile;
  const int chunk = __builtin_amdgcn_readfirstlane(cut.chunk);
  const int chunk_no = item - __builtin_amdgcn_readfirstlane(cut.first);
  const int t0 = min((int64_t)chunk_no * chunk, (int64_t)tiles);
  const int t1 = min((int64_t)t0 + chunk, (int64_t)tiles);

  f32x16 O[D / 32];
#pragma unroll
  for (int db = 0; db < D / 32; ++db) O[db] = f32x16{};
  float m_run = kNegBig, l_run = 0.f;
  const float c = a.scale * kLog2e;

  // ---- staging: a thread takes 16-byte chunks (16 values of one key) of K and
  // of V to registers, and converts them with the key's scale on the way to LDS:
  // once per workgroup, not once per wave.
  const int64_t row0 = ((int64_t)slot_of(s, stream) * Hk + kvh) * s.c.cap;
  const uint8_t* const kg = s.c.k + row0 * D;
  const uint8_t* const vg = s.c.v + row0 * D;
  constexpr int kPerRow = D / 16, kRowsPerPass = kThreads / kPerRow;
  const int srow = threadIdx.x / kPerRow, sch = threadIdx.x % kPerRow;
  u32x4 rk[C::kLoads], rv[C::kLoads];
  uint32_t sk[C::kLoads], sv[C::kLoads];
  auto load = [&](int t) {
#pragma unroll
    for (int p = 0; p < C::kLoads; ++p) {
      const int64_t key = min(t * (int64_t)kManyTile + p * kRowsPerPass + srow, (int64_t)end - 1);
      rk[p] = *(const u32x4*)(kg + key * D + sch * 16);
      rv[p] = *(const u32x4*)(vg + key * D + sch * 16);
      sk[p] = s.c.ks[row0 + key];
      sv[p] = s.c.vs[row0 + key];
    }
  };
  // Tile layout in LDS: K, then V; D / 64 half planes of 64 keys x 128 bytes, a
  // row's 16-byte chunks XOR half_swizzle. Lanes with chunks of the second
  // plane write their two halves in the other order: no two of a cycle's 16 lanes
  // meet in a bank.
  auto store = [&](int buf) {
    lds_u8* const kb = (lds_u8*)smem + buf * C::kBuf;
#pragma unroll
    for (int p = 0; p < C::kLoads; ++p) {
      const int key = p * kRowsPerPass + srow;
      const float kf = __uint_as_float(max(sk[p], sv[p]) == 255u ? 0x7fc00000u : sk[p] << 23);
      const float vf = __uint_as_float(min(sv[p], 254u) << 23);  // (such a row's bytes are zeros)
      lds_u8* const row = kb + (sch >> 2) * C::kHalf + key * 128;
      const int flip = (sch >> 2) & 1;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int h = x ^ flip;
        const u32x2 k2 = h ? u32x2{rk[p][2], rk[p][3]} : u32x2{rk[p][0], rk[p][1]};
        const u32x2 v2 = h ? u32x2{rv[p][2], rv[p][3]} : u32x2{rv[p][0], rv[p][1]};
        const int at = ((2 * (sch & 3) + h) ^ half_swizzle(key)) * 16;
        *(VX_LDS bf16x8*)(row + at) = e4m3x8_bf16(k2, kf);
        *(VX_LDS bf16x8*)(row + C::kTileBytes + at) = e4m3x8_bf16(v2, vf);
      }
    }
  };

  // ---- per-lane LDS offsets of the fragments (see flash_fwd.hip: the same
  // tile layout)
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

  auto step = [&](int t, int buf) {
    const lds_u8* kb = (const lds_u8*)smem + buf * C::kBuf;
    const lds_u8* vb = kb + C::kTileBytes;
    f32x16 S[2] = {f32x16{}, f32x16{}};
#pragma unroll
    for (int ds = 0; ds < D / 16; ++ds)
#pragma unroll
      for (int k2 = 0; k2 < 2; ++k2) {
        const bf16x8 kf = *(const VX_LDS bf16x8*)(kb + koff[ds & 3] + k2 * 32 * 128 + (ds >> 2) * C::kHalf);
        S[k2] = mfma32x32x16(kf, q[ds], S[k2]);
      }
    // a lane's score i of block k2: key k2 32 + (i / 4) 8 + hf 4 + i % 4
    const int key0 = t * kManyTile;
    float cc = c;
    if (key0 + kManyTile > all) {
      cc = 1.0f;
#pragma unroll
      for (int k2 = 0; k2 < 2; ++k2)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          S[k2][i] = key0 + k2 * 32 + (i >> 2) * 8 + hf * 4 + (i & 3) < bound ? S[k2][i] * c : -__builtin_inff();
    }
    float mx = fmaxf(S[0][0], S[1][0]);
#pragma unroll
    for (int i = 1; i < 16; ++i) mx = fmaxf(fmaxf(mx, S[0][i]), S[1][i]);
    mx = halves_max(mx) * cc;
    if (__builtin_amdgcn_ballot_w64(mx > m_run + kSlack) != 0) {
      const float mn = fmaxf(m_run, mx), alpha = fast_exp2(m_run - mn);
      m_run = mn;
      l_run *= alpha;
#pragma unroll
      for (int db = 0; db < D / 32; ++db) O[db] *= alpha;
    }
    const float mneg = -m_run;
    bf16x8 P[2][2];
#pragma unroll
    for (int k2 = 0; k2 < 2; ++k2)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float p = fast_exp2(__builtin_fmaf(S[k2][8 * j + e], cc, mneg));
          l_run += p;
          P[k2][j][e] = (bf16)p;
        }
#pragma unroll
    for (int k2 = 0; k2 < 2; ++k2)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int db = 0; db < D / 32; ++db) {
          const lds_u8* p = vb + (k2 * 32 + 16 * j) * 128 + (db >> 1) * C::kHalf;
          const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((VX_LDS s16x4*)(p + voff[db & 1]));
          const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((VX_LDS s16x4*)(p + 8 * 128 + (voff[db & 1] ^ 16)));
          const bf16x8 vf = concat(__builtin_bit_cast(bf16x4, lo), __builtin_bit_cast(bf16x4, hi));
          O[db] = mfma32x32x16(vf, P[k2][j], O[db]);
        }
  };

  if (t0 < t1) {
    load(t0);
    store(0);
    __syncthreads();
    for (int t = t0; t < t1; ++t) {
      const int buf = (t - t0) & 1;
      if (t + 1 < t1) load(t + 1);
      if (t * kManyTile < any) step(t, buf);
      if (t + 1 < t1) store(buf ^ 1);
      __syncthreads();
    }
  }

  const float L = halves_sum(l_run);
  if (direct && cut.count == 1) {
    const float inv = is_zero(L) ? 0.f : 1.0f / L;
    u32x4 chunk[D / 32][2];
    pack_out_rows<D / 32>(O, inv, chunk);
    if (r < rows) {
      bf16* const o = (bf16*)a.o + rb * a.os[0] + ri * a.os[1] + rh * a.os[2];
#pragma unroll
      for (int db = 0; db < D / 32; ++db)
#pragma unroll
        for (int pr = 0; pr < 2; ++pr) *(u32x4*)(o + db * 32 + 8 * (2 * pr + hf)) = chunk[db][pr];
    }
  } else if (r < rows) {
    float* const part = ws + ((int64_t)item * Hk + kvh) * part_floats(rows, D);
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *(f32x4*)(part + (int64_t)r * D + db * 32 + 8 * g + 4 * hf) =
            f32x4{O[db][4 * g], O[db][4 * g + 1], O[db][4 * g + 2], O[db][4 * g + 3]};
    if (hf == 0) {
      part[(int64_t)rows * D + 2 * r] = m_run;
      part[(int64_t)rows * D + 2 * r + 1] = L;
    }
  }
}

// ------------------------------------------------------------------ merge
// Output rows of item blockIdx.y: D / 4 lanes per row over the parts of the
// item's own chunks and of its group's prefix chunks, in order.
struct Parts {
  Streams s;
  int32_t budget, min_chunk, few;
  int32_t rows;  // per stream and kv head
  float* ws;
};

template <int D>
__global__ __launch_bounds__(kThreads) void merge_kernel(const CachedAttnArgs a, const Parts own, const Parts pre) {
  const int b = blockIdx.y, Hk = a.c.Hk, G = a.H / Hk;
  const Cut oc = own.few ? cut_of<kFewTile>(own.s, own.budget, own.min_chunk, b)
                         : cut_of<kManyTile>(own.s, own.budget, own.min_chunk, b);
  const bool with_prefix = pre.s.n > 0;
  if (!with_prefix && oc.count == 1) return;  // (written by its only chunk)
  Cut pc{0, 0, 0};
  const int per = with_prefix ? a.B / pre.s.n : 1;
  if (with_prefix)
    pc = pre.few ? cut_of<kFewTile>(pre.s, pre.budget, pre.min_chunk, b / per)
                 : cut_of<kManyTile>(pre.s, pre.budget, pre.min_chunk, b / per);
  const int64_t x = (int64_t)blockIdx.x * (kThreads / (D / 4)) + threadIdx.x / (D / 4);
  if (x >= (int64_t)Hk * own.rows) return;
  const int d = (threadIdx.x % (D / 4)) * 4;
  const int kvh = (int)(x / own.rows), r = (int)(x - (int64_t)kvh * own.rows);
  const int i = r / G, h = kvh * G + r % G;
  float M = kNegBig, L = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  auto add = [&](const Parts& p, const Cut& cut, int row) {
    const int64_t block = part_floats(p.rows, D);
    const float* base = p.ws + ((int64_t)cut.first * Hk + kvh) * block;
#pragma unroll 4
    for (int n = 0; n < cut.count; ++n) {
      const float* part = base + (int64_t)n * Hk * block;
      const f32x4 po = *(const f32x4*)(part + (int64_t)row * D + d);
      const float pm = part[(int64_t)p.rows * D + 2 * row], pl = part[(int64_t)p.rows * D + 2 * row + 1];
      const float mn = fmaxf(M, pm), a0 = fast_exp2(M - mn), a1 = fast_exp2(pm - mn);
      o = o * a0 + po * a1;
      L = L * a0 + pl * a1;
      M = mn;
    }
  };
  if (with_prefix) add(pre, pc, (b % per) * own.rows + r);
  add(own, oc, r);
  const bool none = is_zero(L) || i >= clamp_len(a.q_len, b, a.Sq);
  const float inv = 1.0f / L;
  bf16x4 y;
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = (bf16)(none ? 0.f : o[e] * inv);
  *(bf16x4*)((bf16*)a.o + b * a.os[0] + i * a.os[1] + h * a.os[2] + d) = y;
}

// ------------------------------------------------------------------ launch plan
struct Half {
  int streams = 0, rows = 0, per = 1;
  bool few = false;
  int budget = 0, min_chunk = 1;
  int64_t items = 0;  // workgroups per kv head and row tile
  int64_t floats = 0;  // of partial results
};

Half plan_half(int streams, int64_t rows, int per, int cap, int Hk, int D, int cus, bool parts) {
  Half h;
  h.streams = streams;
  h.rows = (int)rows;
  h.per = per;
  h.few = rows <= 32;
  const int64_t slots = 2 * (int64_t)cus;
  const int64_t row_tiles = h.few ? 1 : (rows + kManyRows - 1) / kManyRows;
  const int64_t groups = streams * row_tiles * Hk;
  const int64_t tiles = (cap + (h.few ? kFewTile : kManyTile) - 1) / (h.few ? kFewTile : kManyTile);
  h.min_chunk = 4;
  if (tiles > h.min_chunk && (h.few || groups < slots))
    h.budget = (int)std::min<int64_t>((slots * (h.few ? 2 : 1) + Hk * row_tiles - 1) / (Hk * row_tiles),
                                      streams * ((tiles + h.min_chunk - 1) / h.min_chunk));
  h.items = h.budget + (int64_t)streams;
  if (h.budget == 0) h.items = streams;
  if (parts || h.budget > 0) h.floats = h.items * Hk * ((rows * (D + 2) + 3) & ~(int64_t)3);
  return h;
}

struct Plan {
  Half own, pre;
};

Plan plan_of(int cap, int n_prefix, int p_cap, int B, int Sq, int H, int Hk, int D) {
  const int cus = device_cu_count() > 0 ? device_cu_count() : 256;
  const int64_t rows = (int64_t)Sq * (H / Hk);
  Plan p;
  p.own = plan_half(B, rows, 1, cap, Hk, D, cus, n_prefix > 0);
  if (n_prefix > 0) p.pre = plan_half(n_prefix, rows * (B / n_prefix), B / n_prefix, p_cap, Hk, D, cus, true);
  return p;
}

template <int D>
int launch_half(const CachedAttnArgs& a, const Streams& s, const Half& h, bool prefix, float* ws, hipStream_t st) {
  const int direct = !prefix && a.prefix.k == nullptr;
  if (h.few) {
    hipLaunchKernelGGL(few_kernel<D>, dim3((unsigned)h.items, s.c.Hk), dim3(kThreads), 0, st, a, s, h.rows, h.per,
                       (int)prefix, h.budget, h.min_chunk, direct, ws);
  } else {
    const int64_t n = h.items * ((h.rows + (int64_t)kManyRows - 1) / kManyRows);
    hipLaunchKernelGGL(many_kernel<D>, dim3((unsigned)n, s.c.Hk), dim3(kThreads), 0, st, a, s, h.rows, h.per,
                       (int)prefix, h.budget, h.min_chunk, direct, ws);
  }
  return (int)hipGetLastError();
}

template <int D>
int launch(const CachedAttnArgs& a, hipStream_t st, const char** launched) {
  const int n_prefix = a.prefix.k != nullptr ? a.prefix.slots : 0;
  const Plan p = plan_of(a.c.cap, n_prefix, a.prefix.cap, a.B, a.Sq, a.H, a.c.Hk, D);
  const Streams own{a.c, a.kv_len, a.slots, a.B};
  const Streams pre{a.prefix, a.prefix_len, nullptr, n_prefix};
  float* const ws_pre = a.ws + p.own.floats;
  int err = 0;
  if (n_prefix > 0 && (err = launch_half<D>(a, pre, p.pre, true, ws_pre, st)) != 0) return err;
  if ((err = launch_half<D>(a, own, p.own, false, a.ws, st)) != 0) return err;
  if (n_prefix > 0 || p.own.budget > 0) {
    const Parts po{own, p.own.budget, p.own.min_chunk, p.own.few, p.own.rows, a.ws};
    const Parts pp{pre, p.pre.budget, p.pre.min_chunk, p.pre.few, p.pre.rows, ws_pre};
    const int64_t per_wg = kThreads / (D / 4);
    hipLaunchKernelGGL(merge_kernel<D>, dim3((unsigned)(((int64_t)a.c.Hk * p.own.rows + per_wg - 1) / per_wg), a.B),
                       dim3(kThreads), 0, st, a, po, pp);
    err = (int)hipGetLastError();
  }
  *launched = p.own.few ? (D == 128 ? "few_kernel<128>" : "few_kernel<64>")
                        : (D == 128 ? "many_kernel<128>" : "many_kernel<64>");
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
