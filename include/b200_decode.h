/*
 * b200_decode.h - C ABI of the operators around the delta in a decode step: the base projection with 4-bit weights
 * that the delta is added to, the append of rotated keys and values (and their deltas) to a paged cache, and
 * the attention that reads the cache.
 *
 * Conventions as in b200_lora.h: device pointers on the current device, work enqueued on `stream`, nothing is
 * allocated or synchronised, nothing throws, each call returns a b200_lora_status.  Strides are in elements; the
 * last dimension of every tensor is contiguous.  16-bit operands of one call share one type (B200_LORA_F16 or
 * B200_LORA_BF16).
 *
 * `status` (may be NULL) is a device word into which a kernel ORs B200_DECODE_* bits when it meets indices or lengths
 * it cannot use; the caller clears and reads it.  Nothing is read or written out of bounds either way.
 */
#ifndef B200_DECODE_H
#define B200_DECODE_H

#include "b200_lora.h"

#ifdef __cplusplus
extern "C" {
#endif

enum {
    B200_DECODE_BAD_SLOT = 1,      /* append: a slot behind the cache; the row was left out */
    B200_DECODE_BAD_POSITION = 2,  /* append: a position outside the tables; the row was left out */
    B200_DECODE_BAD_PAGE = 4,      /* attention: a page outside the cache; its keys were not attended to */
    B200_DECODE_BAD_LENGTH = 8,    /* attention: a negative length, or one longer than the row of the page table; it
                                      was taken as zero, or as the row's */
    B200_DECODE_BAD_GROUPS = 16,   /* attention: group starts that descend or lie outside the batch; no prefix was used */
    B200_DECODE_TIMEOUT = 32       /* attention, 4-bit products: a bounded wait inside a kernel expired; the outputs
                                      concerned are NaN */
};
enum { B200_DECODE_MAX_REQUESTS = 4096, B200_DECODE_MAX_GROUPS = 2048 };

/* One layer's paged cache: k and v are [n_pages, page_size, n_kv_heads, head_dim] with these strides (the same for
 * both; a head-major page is a matter of strides).  The reference's table of token slots
 * (lightllm/common/mem_manager.py:28-38) is a cache of page_size 1. */
typedef struct b200_kv_cache {
    void *k, *v;
    int64_t page_stride, token_stride, head_stride;
    int32_t n_pages, page_size, n_kv_heads, head_dim;
} b200_kv_cache;

/* ---- append ------------------------------------------------------------------------------------------
 * For every token row t with slot[t] >= 0:
 *     q_out[t, h] = rot(q[t, h] + dq[t, h])        k[slot] = rot(k[t, h] + dk[t, h])        v[slot] = v[t, h] + dv[t, h]
 * where slot = page * page_size + place in the page and rot turns the first `rotary_dim` elements of a head by
 * the angle whose cosine and sine are row positions[t] of the tables: pairs (i, i + rotary_dim / 2), or (2 i, 2 i + 1)
 * when `interleaved`.  Sums and products are fp32 and rounded once.  dq, dk, dv (NULL: none) are the LoRA deltas that
 * the layer code otherwise adds first (lightllm/models/llama/layer_infer/transformer_layer_infer.py:160-170).
 * Rows with a negative slot are padding: nothing of theirs is written, q_out included.  q_out may be q.  The slots
 * of a call differ; of rows that share one, any row's values may stay, element by element. */
typedef struct b200_append {
    void* q_out;
    const void *q, *k, *v;          /* [n_tokens, heads, head_dim] */
    const void *dq, *dk, *dv;
    int64_t q_out_row, q_out_head, q_row, q_head, k_row, k_head, v_row, v_head;
    int64_t dq_row, dq_head, dk_row, dk_head, dv_row, dv_head;
    const void *positions, *slots;  /* [n_tokens] int32, or int64 */
    const void *cos, *sin;          /* [n_positions, rotary_dim / 2], row stride table_row */
    int64_t table_row;
    int32_t positions_are_i64, slots_are_i64, tables_are_f32 /* else of the 16-bit type */;
    int32_t n_positions, rotary_dim, n_tokens, n_heads, interleaved;
    int32_t* status;
} b200_append;
int b200_kv_append(const b200_append* a, const b200_kv_cache* cache, int32_t dtype, void* stream);

/* ---- attention ---------------------------------------------------------------------------------------
 * One query token per request.  Request b attends to the keys of its group's prefix, then to its own:
 *     out[b, h] = sum_j softmax_j(scale * q[b, h] . k_j) v_j
 * own keys: the first lens[b] of the pages table[b]; prefix: group g holds requests [starts[g], starts[g + 1]) and its
 * keys are the first prefix_lens[g] of the pages prefix_table[g].  Requests in no group have no prefix.  A request
 * without any key gets zeros (lse: -inf).  Query head h reads cache head h / (n_heads / n_kv_heads).  lse (may be
 * NULL) receives the natural logarithm of the sum of exponentials, [n_requests, n_heads] contiguous.
 * Keys and values behind the lengths may hold anything.  page_size is a power of two up to 256; head_dim 64 or 128.
 * The workspace needs no preparation; calls that may overlap each need their own. */
typedef struct b200_attention {
    void* out;
    const void* q;                  /* [n_requests, n_heads, head_dim] */
    float* lse;
    int64_t q_row, q_head, out_row, out_head;
    const int32_t *table, *lens;    /* [n_requests, max_pages] with row stride table_row, [n_requests] */
    const int32_t *prefix_table, *prefix_lens, *group_starts;   /* [n_groups, max_prefix_pages], [n_groups], [n_groups + 1] */
    int64_t table_row, prefix_table_row;
    int32_t max_pages, max_prefix_pages, n_requests, n_groups, n_heads;
    float scale;
    int32_t* status;
} b200_attention;
size_t b200_prefix_attention_workspace_bytes(int32_t n_requests, int32_t n_groups, int32_t n_heads, int32_t n_kv_heads,
                                             int32_t head_dim);
int b200_prefix_attention(const b200_attention* a, const b200_kv_cache* cache, int32_t dtype, void* workspace,
                          size_t workspace_bytes, void* stream);

/* ---- products with 4-bit weights -----------------------------------------------------------------------
 *     y[t, n] = sum_g scales[n, g] * sum_{k in g} (code[n, k] - zero[n, g]) * x[t, k]  (+ add[t, n])
 * codes [n_out, n_in / 2] bytes: column 2 i in the low four bits of byte i, column 2 i + 1 in the high ones.
 * scales [n_out, n_in / group] of x's type; zeros (NULL: 8 everywhere) [n_out, n_in / group] bytes, of which the low
 * four bits count; both contiguous.  group is 32, 64 or 128 and divides n_in.  x [n_tokens, n_in] and y
 * [n_tokens, n_out] with row strides (x's rows do not overlap); y and add are of x's type or both fp32; add (NULL: none) may be y.  Made for the
 * few tokens of a decode step; at most 65535 * 32 of them, and at most 2^31 - 256 inputs and outputs. */
typedef struct b200_int4 {
    void* y;
    const void *x, *codes, *scales, *zeros, *add;
    int64_t x_row, y_row, add_row;
    int32_t n_tokens, n_in, n_out, group;
    int32_t* status;
} b200_int4;
int b200_int4_linear(const b200_int4* a, int32_t dtype, int32_t y_dtype, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* B200_DECODE_H */
