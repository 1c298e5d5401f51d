/*
 * pmkl_cache.h - C ABI of the MI355X (gfx950) key / value cache: block tables
 * and slot maps, appends, and attention over the cache.
 *
 * No counterpart in the reference, whose attention takes whole [B, H, S, D]
 * tensors: these are the operators of a serving step, whose queries are the
 * newest tokens of many requests of different lengths and whose keys and
 * values are kept from step to step.
 *
 * The cache.  Tokens live in pages of `page_size` tokens (a power of two, 16 to
 * 256).  Keys and values are held in 8 bits, as OCP e4m3 codes (largest value
 * 448, no infinity), with one float32 scale for each page and head:
 *   key   token t, column d of page p, head h:  k_scale[p][h] * k[p][h][t][d]
 *   value token t, column d of page p, head h:  v_scale[p][h] * v[p][h][d][t]
 * Values lie with a column's tokens side by side: the product P V sums over
 * tokens, so that is the order in which the matrix unit takes them.
 * Request b's tokens w * page_size .. (w + 1) * page_size - 1 are in page
 * block_table[b][w].
 *
 * Contract, as pmkl_attn.h: device pointers only, the caller allocates
 * everything, a call allocates nothing, launches kernels alone (it can be
 * captured into a HIP graph) and is asynchronous on the given stream;
 * re-entrant; errors leave text in pmkl_last_error().  What lives on the device
 * (lengths, tables, slots) is not read by the host: the kernels check it, and
 * each declaration says what a value out of range does.
 */
#ifndef PMKL_CACHE_H_
#define PMKL_CACHE_H_

#include <stdint.h>

#include "pmkl_attn.h" /* pmkl_dtype, pmkl_status, pmkl_last_error */

#ifdef __cplusplus
extern "C" {
#endif

#define PMKL_CACHE_MIN_PAGE_SIZE 16
#define PMKL_CACHE_MAX_PAGE_SIZE 256

/* A cache.  Strides are in elements (bytes for the codes); a stride group that
 * is all zero means contiguous.  The codes' last dimension is contiguous, their
 * strides are multiples of 16 and their bases 16-byte aligned; pages lie less than
 * 2 GiB apart. */
typedef struct pmkl_kv_cache {
    void *k;                    /* [pages, kv_heads, page_size, head_dim] e4m3          */
    void *v;                    /* [pages, kv_heads, head_dim, page_size] e4m3          */
    float *k_scale;             /* [pages, kv_heads]                                     */
    float *v_scale;             /* [pages, kv_heads]                                     */
    int64_t pages;
    int64_t kv_heads;
    int64_t page_size;
    int64_t head_dim;           /* 32, 64 or 128                                         */
    int64_t k_strides[3];       /* page, head, token                                     */
    int64_t v_strides[3];       /* page, head, column                                    */
    int64_t k_scale_strides[2]; /* page, head                                            */
    int64_t v_scale_strides[2];
} pmkl_kv_cache;

/* Arguments of pmkl_cache_slots. */
typedef struct pmkl_cache_slots_args {
    const int32_t *cached_lens; /* [batch] tokens in the cache before the step           */
    const int32_t *new_lens;    /* [batch] tokens that the step adds, 0 for none         */
    int32_t *block_table;       /* [batch, table_width], rows table_stride apart; the
                                   entries of the step's new pages are written           */
    const int32_t *free_pages;  /* [free_count] pages to take, from free_pages[free_head] */
    const int32_t *free_head;   /* [1]                                                   */
    int32_t *seq_lens;          /* [batch] out: cached + new                             */
    int32_t *query_start;       /* [batch + 1] out: first token of each request, and the
                                   number of tokens                                      */
    int64_t *slots;             /* [tokens] out: page * page_size + offset in the page   */
    int32_t *free_head_out;     /* [1] out: free_head + pages taken                      */
    int64_t batch;
    int64_t table_width;
    int64_t table_stride;       /* 0: table_width                                        */
    int64_t free_count;
    int64_t page_size;
    int64_t tokens;             /* rows of slots: the sum of new_lens, or more           */
} pmkl_cache_slots_args;

/* Tables of a step.  Request b holds c = cached_lens[b] tokens and gets n =
 * new_lens[b] (negative lengths count as 0).  Its pages ceil(c / page_size) to
 * ceil((c + n) / page_size) - 1 are new: they are taken from the free list, in
 * the order of the requests, and entered into its table row.  Token t of it has
 * position c + t; its slot is that position's place in the cache.
 * -1 is written for the entry of a page that the list no longer has (free_head_out
 * counts it all the same, so that free_head_out > free_count shows it), and as the
 * slot of a token without a page, of one past the table's width and of rows past
 * the last token; pages past the table's width are not taken.  Tokens past
 * `tokens` get no slot.  Sums pass 32 bits without harm to other requests, but
 * query_start, seq_lens and free_head_out then hold 2^31 - 1.
 * Nothing is taken back: the caller puts the pages of a finished request behind
 * the list's end.  The outputs must not overlap the inputs (PMKL_EINVAL). */
int pmkl_cache_slots(const pmkl_cache_slots_args *args, void *stream);

/* Arguments of pmkl_cache_append. */
typedef struct pmkl_cache_append_args {
    const void *k;              /* [tokens, kv_heads, head_dim] of dtype                 */
    const void *v;
    const int64_t *slots;       /* [tokens] page * page_size + offset                    */
    pmkl_kv_cache cache;
    int32_t dtype;              /* pmkl_dtype of k and v                                 */
    int64_t tokens;
    int64_t k_strides[2];       /* token, head (elements, multiples of 16 bytes); all
                                   zero: contiguous                                      */
    int64_t v_strides[2];
} pmkl_cache_append_args;

/* Writes new tokens into the cache.  Tokens that follow each other in the call and
 * in a page (slots s, s + 1, ...) make a run; a run's first offset in its page is o.
 * For each head, with a the largest magnitude of the run's finite values:
 *   need    = 2^e, the least e >= -126 with a <= 448 * 2^e
 *   scale'  = need                where o = 0, or the page's scale is not finite and > 0
 *             max(scale, need)    else
 *   code    = e4m3(x / scale')    of the run's values (the quotient in fp32), to nearest
 *                                 even; NaN where x is not finite
 *   code    = e4m3(code * (scale / scale'))   of the page's tokens before o, where the
 *                                 scale grew
 * A power of two costs no precision (e4m3 is a floating type) and makes growing exact
 * down to the type's subnormals.  Everything behind the run is left as it was.
 * A slot outside 0 .. pages * page_size - 1 is skipped.  A page may take one run a
 * call: where two runs name the same page, its codes and scales of this call are
 * unspecified (other pages are not touched).  k and v must not overlap the cache. */
int pmkl_cache_append(const pmkl_cache_append_args *args, void *stream);

/* Arguments of pmkl_cache_attn_fwd. */
typedef struct pmkl_cache_attn_args {
    const void *q;              /* [tokens, heads, head_dim] of dtype                    */
    void *o;                    /* [tokens, heads, head_dim] of dtype                    */
    float *m;                   /* [tokens, heads] row max of the scaled, masked logits  */
    float *l;                   /* [tokens, heads] sum_j exp(s_j - m)                    */
    pmkl_kv_cache cache;
    const int32_t *block_table; /* [batch, table_width], rows table_stride apart         */
    const int32_t *seq_lens;    /* [batch] tokens in the cache, new ones included        */
    const int32_t *query_start; /* [batch + 1] first row of q of each request            */
    void *workspace;            /* 16-byte aligned, pmkl_cache_attn_workspace_size() bytes */
    uint64_t workspace_bytes;
    int32_t dtype;              /* pmkl_dtype of q and o                                 */
    int32_t is_causal;          /* nonzero: a token sees itself and what lies before it  */
    float scale;                /* 0 -> 1.0f / sqrtf((float)head_dim)                    */
    int64_t tokens;             /* rows of q, o, m and l                                 */
    int64_t heads;              /* a multiple of cache.kv_heads: query head h reads key
                                   head h / (heads / kv_heads)                           */
    int64_t batch;
    int64_t table_width;
    int64_t table_stride;       /* 0: table_width                                        */
    int64_t q_strides[2];       /* token, head (elements, multiples of 16 bytes); all
                                   zero: contiguous                                      */
    int64_t o_strides[2];
} pmkl_cache_attn_args;

/* Attention of the requests' newest tokens over their cached ones.  Request b has
 * rows query_start[b] .. query_start[b + 1] - 1; row t of its n stands at position
 * p = seq_lens[b] - n + t.  Over the tokens j < seq_lens[b], causal also j <= p, in
 * fp32:
 *   s_j = scale * <q, key_j>,  m = max_j s_j,  l = sum_j exp(s_j - m),
 *   o   = sum_j exp(s_j - m) / l * value_j
 * The scales must be finite and not negative, and the v_scale of the pages that a row
 * sees within 2^80 of each other (further down, values lose precision against the
 * largest).  Tokens are hidden that lie past the
 * table's width or in a page whose table entry is outside 0 .. pages - 1 (whatever
 * the cache holds there); a row that sees none has o = 0, m = -inf, l = 0.  NaN in a
 * hidden token reaches nothing.  Rows of no request are not written.  query_start must
 * not decrease and is clamped to 0 .. tokens; where it decreases, what the call's rows
 * hold is unspecified, and some may not be written (nothing else is touched).
 * o, m, l and the workspace must overlap nothing that the call reads.
 * The same call gives the same bits every time. */
int pmkl_cache_attn_fwd(const pmkl_cache_attn_args *args, void *stream);

/* Bytes of workspace that pmkl_cache_attn_fwd needs for these arguments (the pointers
 * are not looked at), 0 where it needs none or would refuse them. */
uint64_t pmkl_cache_attn_workspace_size(const pmkl_cache_attn_args *args);

/* The kernels that pmkl_cache_attn_fwd would launch for these arguments, as
 * pmkl_attn_fwd_kernel_name. */
const char *pmkl_cache_attn_kernel_name(const pmkl_cache_attn_args *args);

#ifdef __cplusplus
} /* extern "C" */
#endif

#endif /* PMKL_CACHE_H_ */
