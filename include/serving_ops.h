/*
 * serving_ops.h - C ABI of libserving_ops.so: what a generating step needs around its W4A16 products on
 * AMD MI355X (gfx950): keys and values appended to a paged cache that holds them in 4 bits, with the rotation
 * of queries and keys on the way; attention over that cache; log probabilities of given tokens.
 *
 * As in w4a16.h: plain pointers and sizes, every pointer a DEVICE pointer; no entry point allocates, frees or
 * synchronises, each enqueues its kernels on `stream` (a hipStream_t, NULL = the default stream) and returns,
 * so all of them may be called under HIP graph capture; the current HIP device must be the one that owns the
 * buffers.  Return value: 0 on success, a negative SERVING_E_* code otherwise; nothing is enqueued when a code
 * is returned for an argument error.  Strides are in elements.  `bf16`: 0 = fp16, 1 = bf16 activations.
 *
 * The cache is one buffer [num_blocks][kv_heads][block_size * (head_size + 8)] of bytes, zeroed or not.  What a
 * block (P = block_size tokens, a multiple of 16, at most 4096) holds of one head (D = head_size elements, 64 or 128) is
 *   keys        [P][D / 2]               element d of a token in bits 4 (d % 2) .. + 3 of byte d / 2
 *   values      [P / 16][D / 8][16][4]   the same bytes in pieces of 4 (8 elements), 16 tokens of a piece together
 *   parameters  [2][P][2] fp16           of the keys, then of the values: scale and least of each token
 * and an element stands for  least + code * scale.  A head x[D] of a token is stored as
 *   least = fp16(min x),  scale = fp16((max x - least) * fp32(1 / 15)),
 *   code = clamp(rint((x - least) / scale), 0, 15)
 * in fp32 arithmetic on the values before they are rounded to 16 bits (code = 0 where scale is 0).  A head that
 * holds a NaN or an infinity, or whose parameters fp16 cannot hold, is stored as NaN (both parameters).  The
 * parameters' type does not follow the activations': one cache serves fp16 and bf16 callers.
 */
#ifndef SERVING_OPS_H_
#define SERVING_OPS_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define SERVING_ABI_VERSION 1

enum {
  SERVING_OK = 0,
  SERVING_E_NULL = -1,      /* a required pointer is NULL                                              */
  SERVING_E_SHAPE = -2,     /* a size is out of its range, or sizes do not fit each other              */
  SERVING_E_HEAD = -3,      /* head_size is neither 64 nor 128                                         */
  SERVING_E_BLOCK = -4,     /* block_size is not a multiple of 16 from 16 to 4096                       */
  SERVING_E_ROTARY = -5,    /* the rotated part is not a multiple of 16 elements, or larger than a head */
  SERVING_E_ALIGN = -6,     /* a pointer is not 16-byte aligned, or a stride not a multiple of 8       */
  SERVING_E_LAUNCH = -7,    /* the HIP runtime refused the launch; see serving_last_hip_error()        */
  SERVING_E_TOO_LARGE = -8, /* more work than one launch can index                                     */
  SERVING_E_WORKSPACE = -9  /* the workspace is smaller than serving_*_workspace_bytes() says          */
};

/* Human-readable text for a return code (host pointer, static storage). */
const char* serving_strerror(int code);

/* hipError_t of the last failed launch on this host thread (0 if none). */
int serving_last_hip_error(void);

/* Returns SERVING_ABI_VERSION of the loaded library. */
int serving_abi_version(void);

/* Bytes of a cache (0 for sizes that a cache cannot have). */
size_t serving_kv4_cache_bytes(long long num_blocks, int block_size, int kv_heads, int head_size);

/*
 * One pass over a step's queries, keys and values:
 *   out[t]  = query[t] with the first `rotary` elements of each head rotated by position t's angles
 *   the cache's slot of token t  =  key[t], rotated the same way, and value[t], in 4 bits
 * query [tokens, heads, D], key and value [tokens, kv_heads, D] with strides (token, head); out [tokens, heads, D]
 * contiguous.  cos_sin: fp32 rows of `rotary` values (row stride cs_stride), the cosines of rotary / 2 angles and
 * then their sines, one row for each of `positions` positions.  Pairs are (i, i + rotary / 2), or neighbours
 * (2 i, 2 i + 1) where `interleaved`.  a' = a cos - b sin, b' = b cos + a sin in fp32, each product rounded, rounded
 * once more to the activations' type for the queries.  pos and slots: int64 [tokens]; slot = block * block_size +
 * place in the block.  A slot outside the cache (a padded row's -1) stores nothing; a position outside the table
 * gives NaN queries and stores NaN.  Slots that are stored to have to differ from each other.  rotary may be 0.
 */
int serving_rope_append_kv4(const void* query, long long q_token, long long q_head, const void* key,
                            long long k_token, long long k_head, const void* value, long long v_token,
                            long long v_head, const float* cos_sin, long long cs_stride, const int64_t* pos,
                            const int64_t* slots, void* out, void* cache, int tokens, int heads, int kv_heads,
                            int head_size, int rotary, int interleaved, long long positions, long long num_blocks,
                            int block_size, int bf16, void* stream);

/*
 * key[i], value[i] [rows, kv_heads, D] = what slot slots[i] of the cache stands for, rounded once to fp16 / bf16;
 * zeros for a slot outside the cache.
 */
int serving_read_kv4(const void* cache, const int64_t* slots, void* key, void* value, long long rows, int kv_heads,
                     int head_size, long long num_blocks, int block_size, int bf16, void* stream);

/*
 * out[t] [tokens, heads, D] = softmax(scale * query[t] . keys) values over the cache.
 * Sequence b (of seqs) has seq_lens[b] tokens in the cache, in the blocks tables[b * table_stride + i], i = 0, 1, ..
 * (at most table_width of them), and the query rows query_start[b] .. query_start[b + 1] - 1 (ascending), which are its LAST
 * tokens: row i of n sees keys 0 .. seq_lens[b] - n + i, with window > 0 only the last `window` of these.
 * query_start NULL: one row for each sequence (tokens = seqs).  heads is a multiple of kv_heads; query head h reads
 * kv head h / (heads / kv_heads).  A row that sees no key gives zeros; rows of no sequence are left as they were; rows
 * past the first max_query_len of a sequence are NaN; keys in a block outside the cache are NaN.  max_query_len and
 * max_seq_len size the launch only: a sequence longer than max_seq_len is still read whole, and a max_query_len above
 * `tokens` counts as `tokens`.
 * Arithmetic: products of fp16 numbers summed in fp32; a weight, p times the scale of its token's values, is rounded to
 * fp16 once, against the largest of the row's, whose rounding a result of fp16 has times the value itself and one of
 * bf16 times up to 15 codes; results are rounded once.  A row's result does not depend on keys that it does not see, nor,
 * but for roundings of fp32, on how large other rows are.  Scores have to be finite in fp32, and below 2^115 what the
 * scale, a query's largest element and a key's multiply to; rows with scores beyond 2^25 make their column tile take the
 * slower steps of masks (1.7 times as long for a prompt).
 * workspace: serving_attend_kv4_workspace_bytes() of the same arguments (0: none needed), used by one launch at a
 * time, nothing is kept in it.
 */
size_t serving_attend_kv4_workspace_bytes(int tokens, int seqs, int heads, int kv_heads, int head_size,
                                          int max_query_len, int max_seq_len, int window);
int serving_attend_kv4(const void* query, long long q_token, long long q_head, const void* cache,
                       const int32_t* tables, long long table_stride, int table_width, const int32_t* seq_lens,
                       const int32_t* query_start, void* out, int tokens, int seqs, int heads, int kv_heads,
                       int head_size, long long num_blocks, int block_size, float scale, int window,
                       int max_query_len, int max_seq_len, int bf16, void* workspace, size_t workspace_bytes,
                       void* stream);

/*
 * Of each row of logits [rows, vocab] (vocab up to 2096640; type: 0 = fp16, 1 = bf16, 2 = fp32; row stride in elements):
 *   logprob[r]  = x[token_ids[r]] - log sum exp x          (NaN for a token outside the vocabulary)
 *   entropy[r]  = - sum p log p,  p = softmax x            (a logit of -inf adds nothing)
 *   top_ids[r], top_logprobs[r] [rows, top]: the `top` (0 .. 64) most likely tokens, the most likely first, among
 *                 equals the lowest index first (both zeros are equal, a NaN ranks above all numbers).
 * A row that is -inf throughout, or holds a NaN or +inf, has NaN for all its probabilities, as the formulas give.
 * Arithmetic: exponentials and their sums in fp32, the logarithm and what follows in 64 bits, results rounded once.
 * logprob, entropy, top_logprobs fp32; token_ids and top_ids int64.
 */
size_t serving_token_logprobs_workspace_bytes(int rows, int vocab, int top, int type);
int serving_token_logprobs(const void* logits, long long row_stride, const int64_t* token_ids, float* logprob,
                           float* entropy, int64_t* top_ids, float* top_logprobs, int rows, int vocab, int top,
                           int type, void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* SERVING_OPS_H_ */
