/*
 * vx_cache.h -- C ABI of the 8-bit key/value cache and the attention over it
 * (MI355X, gfx950). Same library, conventions and error codes as vx_attn.h.
 *
 * A cache holds the keys and values of num_slots sequences of up to capacity
 * tokens, contiguous and 16-byte aligned:
 *   k, v              e4m3 bytes [num_slots][num_kv_heads][capacity][head_dim]
 *   k_scale, v_scale  e8m0 bytes [num_slots][num_kv_heads][capacity]
 * A row of head_dim values with scale byte s stands for value * 2^(s - 127); s
 * is the smallest byte >= 1 for which the row's largest magnitude is at most
 * 448 * 2^(s - 127), so a stored value is off by at most 2^-4 of itself, or
 * 2^-10 of the scale where it is below 2^-6 of it. A row that holds a NaN or an
 * infinity has zeros and scale byte 255, and reads as NaN; no other byte stands for
 * one. (Rows from elsewhere: no value byte within a length may be e4m3's NaN, 0x7f
 * or 0xff, and the value bytes of a row of scale 255 are zeros.)
 * capacity is a multiple of 64, head_dim 64 or 128.
 *
 * Lengths, positions and slots are device arrays, so that a captured graph can
 * be replayed while they change; the kernels hold to the cache's bounds
 * whatever they contain (see each entry point).
 */
#ifndef VX_CACHE_H_
#define VX_CACHE_H_

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Version of this header's entries (major * 10000 + minor * 100 + patch): 1.0.0. A library
 * without them does not export this one; vx_abi_version() is that of vx_attn.h alone. */
int32_t vx_cache_abi_version(void);

/*
 * Quantises new tokens' keys and values into the cache: token t of batch item
 * b goes to position start[b] + t of slot slots[b].
 *   k, v     bf16 (batch, seq, num_kv_heads, head_dim), 16-byte aligned;
 *            strides {batch, seq, head} in elements, multiples of 8 (NULL:
 *            contiguous); the head dim is contiguous
 *   start    int32[batch] or NULL (0)
 *   num      int32[batch] or NULL (seq): tokens t >= num[b] are padding and
 *            not written
 *   slots    int32[batch] or NULL (slot b; batch <= num_slots)
 * Tokens whose slot or position lies outside the cache are dropped. Where two
 * batch items name the same slot and position, the later one's token is kept.
 */
int32_t vx_kv_write_fwd(const void* k, const void* v, const int64_t* k_strides, const int64_t* v_strides,
                        void* cache_k, void* cache_v, uint8_t* k_scale, uint8_t* v_scale, int32_t num_slots,
                        int32_t capacity, const int32_t* start, const int32_t* num, const int32_t* slots,
                        int32_t batch, int32_t seq, int32_t num_kv_heads, int32_t head_dim, void* stream);

/* Host-only argument check for vx_kv_write_fwd (no GPU needed). */
int32_t vx_kv_write_check(const void* k, const void* v, const int64_t* k_strides, const int64_t* v_strides,
                          const void* cache_k, const void* cache_v, const uint8_t* k_scale, const uint8_t* v_scale,
                          int32_t num_slots, int32_t capacity, const int32_t* start, const int32_t* num,
                          const int32_t* slots, int32_t batch, int32_t seq, int32_t num_kv_heads, int32_t head_dim);

/*
 * Reads seq positions from start[b] of slot slots[b] on back as bf16: k_out
 * and v_out, contiguous (batch, seq, num_kv_heads, head_dim), 16-byte aligned.
 * start and slots as in vx_kv_write_fwd. Positions outside the cache give
 * zeros. The bf16 values are the stored ones rounded to bf16, which holds all of
 * magnitudes 2^-126 to below 2^128 exactly (a bf16 value above 1.9375 * 2^127 is
 * stored as 2^128, and reads as infinite).
 */
int32_t vx_kv_read_fwd(const void* cache_k, const void* cache_v, const uint8_t* k_scale, const uint8_t* v_scale,
                       int32_t num_slots, int32_t capacity, const int32_t* start, const int32_t* slots,
                       int32_t batch, int32_t seq, int32_t num_kv_heads, int32_t head_dim, void* k_out, void* v_out,
                       void* stream);

/* Host-only argument check for vx_kv_read_fwd (no GPU needed). */
int32_t vx_kv_read_check(const void* cache_k, const void* cache_v, const uint8_t* k_scale, const uint8_t* v_scale,
                         int32_t num_slots, int32_t capacity, const int32_t* start, const int32_t* slots,
                         int32_t batch, int32_t seq, int32_t num_kv_heads, int32_t head_dim, const void* k_out,
                         const void* v_out);

/*
 * Attention of bf16 queries over cached keys and values:
 *   out[b, i, h, :] = sum_j softmax_j(scale * q[b, i, h, :] . K[j, h / G, :]) V[j, h / G, :],
 *   G = num_heads / num_kv_heads
 * with fp32 softmax statistics and accumulation, over the positions j of
 *   - the first prefix_len[g] positions of prefix slot g, g = b / (batch / num_prefixes)
 *     (if a prefix cache is given), all of them for every query, and
 *   - the first kv_len[b] positions of slot slots[b]; with causal, query i of
 *     the q_len[b] ones sits at position kv_len[b] - q_len[b] + i and sees no
 *     later position.
 *   q, out        bf16 (batch, seq_q, num_heads, head_dim), 16-byte aligned;
 *                 strides {batch, seq, head} in elements, multiples of 8 (NULL:
 *                 contiguous)
 *   kv_len        int32[batch] or NULL (capacity), held to [0, capacity]
 *   q_len         int32[batch] or NULL (seq_q), held to [0, seq_q]; output rows
 *                 i >= q_len[b] are zeros
 *   slots         int32[batch] or NULL (slot b; batch <= num_slots); an item
 *                 whose slot lies outside the cache has no keys of its own
 *   prefix_*      the prefix cache, of the same heads and head dim, NULL for
 *                 none; batch is a multiple of num_prefixes
 *   prefix_len    int32[num_prefixes] or NULL (prefix_capacity), held to
 *                 [0, prefix_capacity]
 *   workspace     vx_cached_attn_workspace_size() bytes of device memory,
 *                 16-byte aligned, untouched until the work on `stream` has
 *                 finished; calls that overlap need workspaces of their own.
 *                 (Some calls expand the cached keys and values to bf16 in it:
 *                 see vx_cached_attn_workspace_size.)
 * A weight is at most 2^8 before the division by the sum, and is multiplied by its
 * value row's scale in bf16's range: values from 2^-100 to 2^100 keep their precision.
 * The logits (scale * q . k, and q . k itself) may be of any size that fp32 holds,
 * times log2(e); calls that expand the cache (see the workspace) take magnitudes up
 * to 2^24.
 * A query without a visible key gives zeros. A key or value row of scale 255
 * makes NaN the outputs of exactly those queries of its head that see it.
 */
int32_t vx_cached_attn_fwd(const void* q, void* out, const int64_t* q_strides, const int64_t* out_strides,
                           const void* cache_k, const void* cache_v, const uint8_t* k_scale, const uint8_t* v_scale,
                           int32_t num_slots, int32_t capacity, const void* prefix_k, const void* prefix_v,
                           const uint8_t* prefix_k_scale, const uint8_t* prefix_v_scale, int32_t num_prefixes,
                           int32_t prefix_capacity, const int32_t* kv_len, const int32_t* q_len, const int32_t* slots,
                           const int32_t* prefix_len, int32_t batch, int32_t seq_q, int32_t num_heads,
                           int32_t num_kv_heads, int32_t head_dim, int32_t causal, float scale, void* workspace,
                           int64_t workspace_bytes, void* stream);

/* Host-only argument check for vx_cached_attn_fwd (no GPU needed; the workspace is not looked at). */
int32_t vx_cached_attn_check(const void* q, const void* out, const int64_t* q_strides, const int64_t* out_strides,
                             const void* cache_k, const void* cache_v, const uint8_t* k_scale, const uint8_t* v_scale,
                             int32_t num_slots, int32_t capacity, const void* prefix_k, const void* prefix_v,
                             const uint8_t* prefix_k_scale, const uint8_t* prefix_v_scale, int32_t num_prefixes,
                             int32_t prefix_capacity, const int32_t* kv_len, const int32_t* q_len,
                             const int32_t* slots, const int32_t* prefix_len, int32_t batch, int32_t seq_q,
                             int32_t num_heads, int32_t num_kv_heads, int32_t head_dim, int32_t causal, float scale);

/*
 * Workspace bytes vx_cached_attn_fwd needs for these sizes on the current
 * device (0: none; -1 on failure). num_prefixes is 0 without a prefix; cross is
 * 1 for a call that is not causal and has no q_len.
 *
 * Where a cross call has no prefix, as many heads as the cache, seq_q >= capacity
 * and batch * num_heads * seq_q >= 300000, the cached keys and values are expanded
 * to bf16 in the workspace: 4 * head_dim bytes per position, head and batch item of
 * the capacity (not of kv_len; what lies past kv_len is not written): at most twice
 * the bytes of q. A capacity above seq_q, or a q_len, leaves such a call with the
 * kernels that read the cache as it is and need no workspace: 3 to 48 % more time
 * (2 x 32760 queries of 40 heads on 512 and 384 keys 664 us, with q_len 804 to 842).
 */
int64_t vx_cached_attn_workspace_size(int32_t capacity, int32_t num_prefixes, int32_t prefix_capacity, int32_t batch,
                                      int32_t seq_q, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                                      int32_t cross);

#ifdef __cplusplus
}
#endif

#endif /* VX_CACHE_H_ */
