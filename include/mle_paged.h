/*
 * mle_paged.h -- C ABI of the paged KV cache on MI355X (gfx950): page planning for a
 * batch of requests, rotary embedding with the cache write, and the attention of the
 * new tokens over the cache.  Library: llmengine_amd/libmle_q8_0.so, with the
 * conventions of mle_q8_0.h: device pointers, work enqueued on `stream`, 0 or an
 * ErrorCode value returned, mle_last_error() for the message, the per-(device, stream)
 * workspace, fp32 activations 16-byte aligned.
 *
 * A decoder layer of a serving step:
 *
 *   mle_paged_plan        once per step: pages for the requests' new tokens
 *   mle_q8_0_linear_multi q, k, v of the new tokens
 *   mle_paged_kv_write    q and k rotated, k and v put into the cache
 *   mle_paged_attention   the new tokens' attention over the cache
 *   mle_q8_0_linear       the output projection
 *
 * One token per request is decoding, several are a prompt or a chunk of one; a batch
 * may mix them.
 */
#ifndef MLE_PAGED_H
#define MLE_PAGED_H

#include "mle_q8_0.h"

#ifdef __cplusplus
extern "C" {
#endif

/* What a cache holds.  f16 and bf16: the value rounded once.  int8: q = rint(x / s)
 * with one fp32 scale s = amax * (1/127) per token and KV head (over its head_dim
 * values, for K after the rotation); the value is q * s.  A row that holds a NaN or an
 * infinity gets such a scale, so it reads back as NaN, not as finite numbers.  A V row
 * whose s is at or below 2^-64 is stored as zeros with s = 0; the attention reads V scales
 * above 2^-64 and 0.  Rows of zeros have their weights beside V scales up to 2^40. */
#define MLE_KV_F16 0
#define MLE_KV_BF16 1
#define MLE_KV_INT8 2

/*
 * One layer's cache: `num_pages` pages of `page_size` tokens for `kv_heads` heads.
 * K and V hold num_pages * kv_heads * page_size * head_dim elements each, 16-byte
 * aligned.  Page p, KV head g, token t of the page (tile t / 16, row r = t % 16) and
 * dimension d are at element
 *   ((p * kv_heads + g) * page_size + t - r) * head_dim +
 *     K: (d / 8) * 128 + r * 8 + d % 8
 *     V: (r / 4 % 2) * head_dim * 8 + d * 8 + (r / 8) * 4 + r % 4
 * that is, in the order in which the matrix cores take K as rows of keys and V as rows
 * of dimensions: a wave's load is one run of memory and no kernel transposes anything.
 * k_scale, v_scale (int8 only, else NULL): [num_pages][kv_heads][page_size] fp32.
 * head_dim is 64, 96, 128 or 256, page_size a multiple of 16 up to 1024.
 */
typedef struct mle_paged_cache {
  void* k;
  void* v;
  float* k_scale;
  float* v_scale;
  int32_t type;
  int32_t num_pages;
  int32_t page_size;
  int32_t kv_heads;
  int32_t head_dim;
} mle_paged_cache;

/*
 * Page plan of one step, on the device: block tables, slot map, row offsets.
 *
 * Request b has cached_lens[b] tokens in the cache and brings new_lens[b] (0: none;
 * negative: the request is finished and gives its pages back).  block_table
 * [sequences][max_pages] names its pages, in order; free_pages [num_pages] is a stack
 * of which the first *free_count entries are free.
 *   1. The first ceil(cached / page_size) pages of each finished request go on top of
 *      the stack, requests in order.
 *   2. The pages that a request needs past the ones it has are popped from the top,
 *      requests in order, and written to its row of block_table.  A request whose pages
 *      are not there (the pages asked for up to and including it are more than the
 *      stack holds), that would outgrow max_pages or 2^31 - 1 tokens or whose rows pass
 *      `tokens` (a request without new tokens has none) is refused and its table row left
 *      as it is; requests that need no page are never short of one.
 *   3. kv_lens[b] = cached + new (refused or finished: 0).  cu_tokens[sequences + 1] =
 *      the first row of each request among the step's rows: prefix sums of the
 *      requested new tokens, refused requests included, at most `tokens`.
 *      granted[b] = 0 for a refused request, else 1.  free_count_out = pages left (may
 *      be free_count itself).  For row r < tokens: positions[r] = its position in its
 *      sequence, slots[r] = page * page_size + offset; 0 and -1 where the request was
 *      refused and for rows that no request has.
 * A page number outside [0, num_pages) in table or stack gives slot -1.  Deterministic;
 * with free_count_out apart from free_count a repeated call gives the same again.  But
 * for those two no output may overlap another array.  A plan of more than 1024 rows takes
 * a counter of the per-stream workspace (before a graph is captured: 256 bytes and 32
 * counters, or what mle_paged_attention_workspace_size says for as many rows).
 * Errors: NULL pointers, sequences or sizes <= 0, tokens < 0 -> InvalidArgument;
 * sequences * max_pages or num_pages * page_size above 2^31 - 1, num_pages, max_pages or
 * tokens of 2^30 or more -> Unsupported.  tokens == 0: positions and slots may be NULL.
 */
int mle_paged_plan(const int32_t* cached_lens, const int32_t* new_lens, int sequences,
                   int32_t* block_table, int max_pages, int page_size, int num_pages,
                   int32_t* free_pages, const int32_t* free_count, int32_t* free_count_out,
                   int tokens, int32_t* kv_lens, int32_t* cu_tokens, int32_t* positions,
                   int32_t* slots, int32_t* granted, hipStream_t stream);

/*
 * Table of rotations: table[p][i] = (cos a, sin a) with a = p * theta^(-2i / rope_dim) /
 * freq_factors[i] (NULL: 1) for p < positions, i < rope_dim / 2; angles and functions in
 * 64 bits, rounded once.  freq_factors are a GGUF file's rope_freqs.  table is
 * 16-byte aligned, [positions][rope_dim / 2][2] fp32.
 * Errors: NULL table, positions or rope_dim <= 0, odd rope_dim, theta not positive and
 * finite -> InvalidArgument; positions * rope_dim / 2 above 2^32 - 256 -> Unsupported.
 */
int mle_rope_table(float* table, int positions, int rope_dim, double theta,
                   const float* freq_factors, hipStream_t stream);

/* Which elements turn together: 2i and 2i + 1, or i and i + rope_dim / 2. */
#define MLE_ROPE_PAIRS 0
#define MLE_ROPE_HALVES 1

/*
 * Rotary embedding of q and k, and the write of k and v into the cache.  Row r < tokens
 * of q [heads][head_dim], k and v [kv_heads][head_dim] starts at r * its stride (floats;
 * a multiple of 4, at least the row's size), so q, k and v may lie in one buffer of a
 * fused Linear.  With (c, s) = rope[positions[r]][i], elements (a, b) of a pair become
 * (a c - b s, a s + b c): exact products, their sum in 64 bits, then rounded to fp32;
 * elements from rope_dim on stay.  rope NULL: no rotation, positions may be NULL.  Rotated
 * q goes to q_out (may be q with the same stride); k and v, in the cache's type, to
 * slots[r].  A slot outside the cache (-1) writes none; two rows of one slot race.  A position
 * outside [0, rope_positions) has no rotation: its q_out row is zero and nothing of it
 * is cached.
 * Errors: NULL pointers, tokens < 0, sizes <= 0, misalignment -> InvalidArgument;
 * strides too small or not a multiple of 4, rope_dim not a multiple of 8 or above
 * head_dim, unknown type or mode -> InvalidArgument; a head_dim or page_size the cache
 * does not take, tokens * (heads + 2 kv_heads) above 2^30, or as many threads as a launch
 * does not hold (8, 16 or 32 lanes for each k and v row and each two rows of q at head_dim
 * 64, up to 128, 256: above 2^32 - 256) -> Unsupported.  tokens == 0 is a no-op.
 */
int mle_paged_kv_write(const mle_paged_cache* cache, const float* q, int q_stride,
                       float* q_out, int q_out_stride, int heads, const float* k, int k_stride,
                       const float* v, int v_stride, const float* rope, int rope_positions,
                       int rope_dim, int rope_mode, const int32_t* positions,
                       const int32_t* slots, int tokens, hipStream_t stream);

/*
 * Attention of the new tokens over the cache.  Rows cu_tokens[b] .. cu_tokens[b+1] of q
 * [tokens][heads][head_dim] are the last new_b of the kv_lens[b] tokens of sequence b, so
 * row i stands at position p = kv_lens[b] - new_b + i and sees the keys j <= p, with
 * window > 0 only those with j > p - window.  Query head h reads KV head
 * h / (heads / kv_heads).
 *   out[row][h] = sum_j softmax_j(scale * q . k_j) v_j
 * in fp32 accuracy: q and the probabilities go to the matrix cores as sums of 16-bit
 * parts (two of f16, 22 bits, three of bf16 over a bf16 cache), the cache's values are
 * taken as they are, sums are fp32: a logit of 2^127 or more makes its row NaN, and sums
 * of more than 256 values within 2^8 of the largest bf16 may overflow.
 * A row that sees no key is zero.  A key in a page outside [0, num_pages) counts as hidden;
 * hidden keys and values may hold anything, NaN included.  A NaN or an infinity that a row
 * sees reaches that row alone, where a logit of minus infinity is a weight of 0.  Rows
 * outside every sequence are not written.  Long sequences with few rows are split over the
 * keys and joined in a fixed order: deterministic run to run.
 * Row strides in floats, multiples of 4; out must not overlap q unless it is q with the
 * same stride.  `sequences` may include some without new rows.
 * Errors: NULL pointers, sizes <= 0, tokens < 0, heads not a multiple of kv_heads, a
 * window < 0, a scale that is not finite, bad strides or alignment -> InvalidArgument;
 * a head_dim or page_size the cache does not take, heads / kv_heads above 64, more than
 * 31 bits of max_pages * page_size or tokens * heads / kv_heads -> Unsupported.
 * tokens == 0 is a no-op.
 *
 * mle_paged_attention_workspace_size: what any call of 1 .. tokens rows in 1 ..
 * sequences sequences takes of the per-stream workspace (mle_workspace_reserve; to be
 * reserved before a graph is captured): 9 MB for up to 16 rows of a KV head, 69 MB above
 * (head_dim 128), whatever the lengths.
 */
int mle_paged_attention(const mle_paged_cache* cache, const float* q, int q_stride, float* out,
                        int out_stride, int heads, float scale, int window,
                        const int32_t* block_table, int max_pages, const int32_t* kv_lens,
                        const int32_t* cu_tokens, int sequences, int tokens,
                        hipStream_t stream);
int mle_paged_attention_workspace_size(const mle_paged_cache* cache, int heads, int sequences,
                                       int tokens, size_t* bytes, size_t* counters);

#ifdef __cplusplus
}  /* extern "C" */
#endif

#endif /* MLE_PAGED_H */
