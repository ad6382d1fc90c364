/*
 * clove_fp8.h — C ABI of the 8-bit paged KV cache: a quantising append, the
 * decode over it, accumulated attention weights and eviction by weight.
 * No counterpart in the reference, whose kv_cache is f32 only
 * (src/nn.rs:534); the conventions (status codes, int32 tables and lengths,
 * asynchronous calls on `stream`, device check flags) are clove_cuda.h's.
 *
 * The cache
 *   codes   e4m3 bytes [2, num_blocks, num_kv_heads, block_size, head_dim]
 *           (K plane, V plane): a (block, KV head) tile is contiguous.
 *   scales  f32 [2, num_blocks, num_kv_heads]: an element is code * scale.
 *   mass    f32 [num_blocks, num_kv_heads, block_size], optional: the
 *           attention weight that each cached token has received from decode
 *           calls that accumulate.  Written tokens start at 0, prompts too:
 *           before the first such decode an eviction finds nothing but ties
 *           and keeps the lowest indices (and the `recent` last ones).
 *
 * Scale rule.  The scale of a (block, KV head) of a plane is 2^e with the
 * smallest e >= -126 for which 448 * 2^e covers the largest finite magnitude
 * of the rows written.  While a block fills, its scale only grows, and the
 * codes already there are rounded to the larger scale (exact unless a code
 * falls below e4m3's normal range).  A write to row 0 of a block starts the
 * block anew: the old scale no longer counts, and the other rows not written
 * by the same call hold nothing.  So blocks are filled from row 0 on, as the
 * block manager's tables do.  Infinities are stored as +-448 * scale, NaN as
 * NaN; neither counts towards a scale.  Scales written by other means (a
 * loaded cache) may be any positive number up to 2^127.  A decode's outputs
 * are as exact as float32 weights make them while the V scales of a sequence
 * and KV head are within 2^100 of one another; a block whose scale is further
 * below the largest one keeps as many bits less.
 *
 * Shapes: head_dim 64, 128 or 256; block_size a power of two in [8, 256];
 * num_q_heads / num_kv_heads in 1..8.  q, k, v and the new token may be f32,
 * f16 or bf16 (CLOVE_DTYPE_*, one type per call), 16-byte aligned.
 *
 * Bad block ids, context lengths and slots are clamped or skipped, never
 * followed, and raise CLOVE_FLAG_* in the pool's status word
 * (clove_fp8_pool_status).  No call allocates device memory or synchronises,
 * except where it says so; every call may be captured in a CUDA graph.
 * Calls on different streams may run at the same time when none writes a block
 * that another reads or writes, and they use different workspaces.  A token
 * written to a block may rewrite the block's other rows (to a grown scale), so
 * unlike in the 16-bit pools even a reader of earlier rows alone must not run
 * beside it.
 */
#ifndef CLOVE_FP8_H
#define CLOVE_FP8_H

#include "clove_cuda.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct clove_fp8_pool* clove_fp8_pool_t;

typedef struct clove_fp8_pool_info {
    int device;
    int num_blocks;
    int block_size;
    int num_kv_heads;
    int head_dim;
    int owns_memory;     /* 1: created by clove_fp8_pool_create, 0: wrapped */
    void* codes;         /* device pointers */
    float* scales;
    float* mass;         /* null: the pool keeps no attention weights */
    size_t codes_bytes;
} clove_fp8_pool_info_t;

/* How the decode forms a score from scale * <q, K_t>.  In this order:
 *   softcap > 0     z = softcap * tanh(z / softcap); 0, or 2^-126 at least
 *   alibi_slopes    z += alibi_slopes[hq] * (t - (L - 1)): f32 [num_q_heads]
 *                   device array or null; t the token's index in the cache,
 *                   L the tokens cached (the new one included)
 *   window > 0      only the last `window` tokens are attended to
 * accumulate != 0: the call adds each token's attention weight, summed over
 * the query heads of its KV head, to the pool's mass (a token the call
 * appends starts at its own weight).  Sequences of one call may share blocks
 * (forks): their weights add up, in an order that may change the last bit.
 * A call that gives up on a wait (CLOVE_FLAG_TIMEOUT) adds no weights. */
typedef struct clove_fp8_scores {
    float softcap;
    const float* alibi_slopes;
    int window;
    int accumulate;
} clove_fp8_scores_t;

/* Allocate a cache (codes, scales and, with with_mass, mass; all zero), or
 * wrap caller-owned device arrays (codes 128-byte aligned, scales and mass
 * 16-byte aligned; mass may be null) without taking ownership.  Both allocate
 * the pool's status word and its append index (4 bytes per token slot). */
int clove_fp8_pool_create(int device, int num_blocks, int block_size, int num_kv_heads, int head_dim,
                          int with_mass, clove_fp8_pool_t* out);
int clove_fp8_pool_wrap(int device, void* codes, float* scales, float* mass, int num_blocks, int block_size,
                        int num_kv_heads, int head_dim, clove_fp8_pool_t* out);
int clove_fp8_pool_destroy(clove_fp8_pool_t pool);
int clove_fp8_pool_info(clove_fp8_pool_t pool, clove_fp8_pool_info_t* info);

/* Synchronise `stream`, read and clear the check flags that this pool's
 * calls raised since the last call; CLOVE_ERR_DEVICE_CHECK if any was set. */
int clove_fp8_pool_status(clove_fp8_pool_t pool, void* stream, int* flags);

/* Quantising append: token i goes to slot slot_mapping[i] (block slot /
 * block_size, row slot % block_size); negative slots are skipped.  k, v
 * [num_tokens, num_kv_heads, head_dim].  Of two tokens with the same slot the
 * later one counts.  The result does not depend on the tokens' order
 * otherwise.  The mass of a written row becomes 0. */
size_t clove_fp8_append_workspace_size(clove_fp8_pool_t pool, int num_tokens);
int clove_fp8_append(clove_fp8_pool_t pool, int dtype, const void* k, const void* v, const int32_t* slot_mapping,
                     int num_tokens, void* workspace, size_t workspace_bytes, void* stream);

/* The cached tokens as the values they stand for: k_out, v_out f32 [batch,
 * max_ctx, num_kv_heads, head_dim], rows t >= context_lens[b] zero. */
int clove_fp8_gather(clove_fp8_pool_t pool, const int32_t* block_tables, int bt_stride, const int32_t* context_lens,
                     int batch, int max_ctx, float* k_out, float* v_out, void* stream);

/* Decode: out [batch, num_q_heads, head_dim] f32 = softmax(z) . V over the
 * cached tokens of each sequence, z as above.  With k_new and v_new [batch,
 * num_kv_heads, head_dim] (both or neither) the new token is appended first:
 * context_lens then holds the lengths before it, and max_ctx bounds the
 * lengths after it.  No sequence may append to a block that another sequence of
 * the call holds (the block manager's copy-on-write keeps forks apart).  A
 * sequence without tokens gets a zero row.  scores may be null: no cap, bias
 * or window.  The workspace needs no initialisation. */
size_t clove_fp8_decode_workspace_size(clove_fp8_pool_t pool, int batch, int num_q_heads, int max_ctx,
                                       int accumulate);
int clove_fp8_decode(clove_fp8_pool_t pool, int dtype, const void* q, const void* k_new, const void* v_new,
                     int num_q_heads, const int32_t* block_tables, int bt_stride, const int32_t* context_lens,
                     int batch, float scale, int max_ctx, const clove_fp8_scores_t* scores, float* out,
                     void* workspace, size_t workspace_bytes, void* stream);

/* Eviction: every sequence is brought down to n = min(context_lens[b],
 * budget) tokens.  Each KV head keeps its own: the last `recent` tokens
 * (0 <= recent <= budget) and, of the others, those of largest mass (ties to
 * the lower index).  The kept tokens move, in order, with their mass to rows
 * 0 .. n-1 of the blocks new_tables[b] (int32 [batch, new_stride], new_stride
 * * block_size >= min(budget, max_ctx)), a new block's scale being the largest of
 * its rows' old scales.  The new blocks must be distinct and not among the blocks
 * the call reads.
 * kept int32 [batch, num_kv_heads, budget]: the kept tokens' old indices,
 * ascending, -1 behind the n-th; new_lens int32 [batch]: n.  Rows behind a
 * sequence's last token stay as they were.  Needs a pool with mass; budget and
 * max_ctx are 2^31 - 2^16 - 1 at most. */
size_t clove_fp8_evict_workspace_size(clove_fp8_pool_t pool, int batch, int max_ctx, int budget);
int clove_fp8_evict(clove_fp8_pool_t pool, const int32_t* block_tables, int bt_stride, const int32_t* context_lens,
                    int batch, int max_ctx, const int32_t* new_tables, int new_stride, int budget, int recent,
                    int32_t* kept, int32_t* new_lens, void* workspace, size_t workspace_bytes, void* stream);

/* Copy blocks src[i] -> dst[i] (codes, scales and mass; device int32 arrays
 * of n entries): the copies of the block manager's copy-on-write.  They run at
 * the same time: a block that is written is no other copy's source or
 * destination. */
int clove_fp8_copy_blocks(clove_fp8_pool_t pool, const int32_t* src, const int32_t* dst, int n, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* CLOVE_FP8_H */
