/*
 * vx_decode.h -- C ABI of the steps of a rollout or a decoding loop over the 8-bit
 * key/value cache of vx_cache.h (MI355X, gfx950): rotary positions on several axes,
 * alone and on the way into the cache, attention with a sliding window behind first
 * tokens that stay visible, attention of a tree of drafted tokens. Same library,
 * conventions and error codes as vx_attn.h; the cache's arrays, lengths and slots
 * are those of vx_cache.h, device arrays that may change while a captured graph is
 * replayed, and the kernels hold to the bounds whatever they contain.
 */
#ifndef VX_DECODE_H_
#define VX_DECODE_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Version of this header's entries (major * 10000 + minor * 100 + patch): 1.0.0. */
int32_t vx_decode_abi_version(void);

/*
 * Rotary positions: pair j of a head's channels (j < head_dim / 2) of token t of
 * batch item b turns by positions[b, t, axis[j]] * turns[j],
 *   (u, w) -> (u cos - w sin, u sin + w cos),
 * or, with inverse, by as much the other way, which is also the gradient: of the
 * turn's input, from that of its output.
 *   x          bf16 (batch, seq, num_heads, head_dim), 16-byte aligned; strides
 *              {batch, seq, head} in elements, multiples of 8 (NULL: contiguous)
 *   out        bf16, the same shape, contiguous, 16-byte aligned; x itself, if that is
 *              contiguous (refused if not), or no part of it
 *   positions  int32 at strides {batch, token, axis} in elements (>= 0; 0: shared;
 *              NULL: contiguous (batch, seq, num_axes))
 *   num_axes   1 to 4
 *   turns      uint64[head_dim / 2], turns per position in units of 2^-64 turns
 *              (whole turns left out); 0: the pair stays as it is
 *   axis       int32[head_dim / 2]; a pair whose axis is not 0 .. num_axes - 1
 *              does not turn
 *   halves     1: pair j is channels (j, j + head_dim / 2); 0: (2 j, 2 j + 1)
 * head_dim is 64 or 128. The angle is formed modulo a turn in integers, so it is
 * as exact for far positions as for near ones: off by less than 2^-32 turns and
 * position * 2^-65. A sine or cosine is off by at most 2^-21 in all; the turn is in
 * fp32, rounded once.
 */
int32_t vx_axis_rope_fwd(const void* x, void* out, const int64_t* x_strides, const int32_t* positions,
                         const int64_t* position_strides, int32_t num_axes, const uint64_t* turns,
                         const int32_t* axis, int32_t halves, int32_t inverse, int32_t batch, int32_t seq,
                         int32_t num_heads, int32_t head_dim, void* stream);

/* Host-only argument check for vx_axis_rope_fwd (no GPU needed; whether out is x is not looked at). */
int32_t vx_axis_rope_check(const void* x, const void* out, const int64_t* x_strides, const int32_t* positions,
                           const int64_t* position_strides, int32_t num_axes, const uint64_t* turns,
                           const int32_t* axis, int32_t halves, int32_t inverse, int32_t batch, int32_t seq,
                           int32_t num_heads, int32_t head_dim);

/*
 * vx_kv_write_fwd of keys turned as by vx_axis_rope_fwd (in fp32, rounded once, to
 * the cache's e4m3) and of values as they are. positions are those of the tokens
 * that k holds, whatever position of the cache they go to. A turned row with a NaN
 * or an infinity is stored as NaN.
 */
int32_t vx_kv_write_rope_fwd(const void* k, const void* v, const int64_t* k_strides, const int64_t* v_strides,
                             void* cache_k, void* cache_v, uint8_t* k_scale, uint8_t* v_scale, int32_t num_slots,
                             int32_t capacity, const int32_t* start, const int32_t* num, const int32_t* slots,
                             const int32_t* positions, const int64_t* position_strides, int32_t num_axes,
                             const uint64_t* turns, const int32_t* axis, int32_t halves, int32_t batch, int32_t seq,
                             int32_t num_kv_heads, int32_t head_dim, void* stream);

/* Host-only argument check for vx_kv_write_rope_fwd (no GPU needed). */
int32_t vx_kv_write_rope_check(const void* k, const void* v, const int64_t* k_strides, const int64_t* v_strides,
                               const void* cache_k, const void* cache_v, const uint8_t* k_scale,
                               const uint8_t* v_scale, int32_t num_slots, int32_t capacity, const int32_t* start,
                               const int32_t* num, const int32_t* slots, const int32_t* positions,
                               const int64_t* position_strides, int32_t num_axes, const uint64_t* turns,
                               const int32_t* axis, int32_t halves, int32_t batch, int32_t seq, int32_t num_kv_heads,
                               int32_t head_dim);

/*
 * vx_cached_attn_fwd (no prefix) whose queries see, of the positions j that they
 * would see there, those of a sliding window and the first `sinks`:
 *   j < e and (j >= e - window or j < sinks),
 * e one past query i's position kv_len[b] - q_len[b] + i with causal, else kv_len[b].
 *   window  >= 1, the query's own position (not causal: the last one) among it
 *   sinks   >= 0
 * The other arguments, the numerics, and rows without a visible key, as there.
 * What the cache holds at positions that no query of a call sees may be anything:
 * never written, codes and scales of NaN. (Tiles of it are not read; what shares a
 * tile of 64 positions with seen ones has no effect.)
 */
int32_t vx_window_attn_fwd(const void* q, void* out, const int64_t* q_strides, const int64_t* out_strides,
                           const void* cache_k, const void* cache_v, const uint8_t* k_scale, const uint8_t* v_scale,
                           int32_t num_slots, int32_t capacity, const int32_t* kv_len, const int32_t* q_len,
                           const int32_t* slots, int32_t batch, int32_t seq_q, int32_t num_heads,
                           int32_t num_kv_heads, int32_t head_dim, int32_t window, int32_t sinks, int32_t causal,
                           float scale, void* workspace, int64_t workspace_bytes, void* stream);

/* Host-only argument check for vx_window_attn_fwd (no GPU needed; the workspace is not looked at). */
int32_t vx_window_attn_check(const void* q, const void* out, const int64_t* q_strides, const int64_t* out_strides,
                             const void* cache_k, const void* cache_v, const uint8_t* k_scale,
                             const uint8_t* v_scale, int32_t num_slots, int32_t capacity, const int32_t* kv_len,
                             const int32_t* q_len, const int32_t* slots, int32_t batch, int32_t seq_q,
                             int32_t num_heads, int32_t num_kv_heads, int32_t head_dim, int32_t window,
                             int32_t sinks, int32_t causal, float scale);

/* Workspace bytes vx_window_attn_fwd needs for these sizes on the current device (0: none; -1 on failure). */
int64_t vx_window_attn_workspace_size(int32_t capacity, int32_t batch, int32_t seq_q, int32_t num_heads,
                                      int32_t num_kv_heads, int32_t head_dim, int32_t window, int32_t sinks,
                                      int32_t causal);

/*
 * vx_cached_attn_fwd (no prefix) of drafted tokens: the last q_len[b] of the
 * kv_len[b] cached tokens of item b are drafted, its queries theirs in the same
 * order. Query i sees every token in front of the drafted ones, of those its
 * ancestors, and itself.
 *   parents  int32: item b's drafted token i has the parent parents[b *
 *            parents_stride + i], an earlier drafted token; any value that is not
 *            0 .. i - 1 stands for none (a token that follows the last one in
 *            front). parents_stride >= 0; 0: all items have the same tree
 *   seq_q    at most 512
 * A chain (parents i - 1) is what vx_cached_attn_fwd computes with causal.
 */
int32_t vx_tree_attn_fwd(const void* q, void* out, const int64_t* q_strides, const int64_t* out_strides,
                         const void* cache_k, const void* cache_v, const uint8_t* k_scale, const uint8_t* v_scale,
                         int32_t num_slots, int32_t capacity, const int32_t* kv_len, const int32_t* q_len,
                         const int32_t* slots, const int32_t* parents, int64_t parents_stride, int32_t batch,
                         int32_t seq_q, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim, float scale,
                         void* workspace, int64_t workspace_bytes, void* stream);

/* Host-only argument check for vx_tree_attn_fwd (no GPU needed; the workspace is not looked at). */
int32_t vx_tree_attn_check(const void* q, const void* out, const int64_t* q_strides, const int64_t* out_strides,
                           const void* cache_k, const void* cache_v, const uint8_t* k_scale, const uint8_t* v_scale,
                           int32_t num_slots, int32_t capacity, const int32_t* kv_len, const int32_t* q_len,
                           const int32_t* slots, const int32_t* parents, int64_t parents_stride, int32_t batch,
                           int32_t seq_q, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim, float scale);

/* Workspace bytes vx_tree_attn_fwd needs for these sizes on the current device (0: none; -1 on failure). */
int64_t vx_tree_attn_workspace_size(int32_t capacity, int32_t batch, int32_t seq_q, int32_t num_heads,
                                    int32_t num_kv_heads, int32_t head_dim);

#ifdef __cplusplus
}
#endif

#endif /* VX_DECODE_H_ */
