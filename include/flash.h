/*
 * Fused causal multi-head attention, forward and backward -- C-ABI drop-in for
 * bare-metal-bard's src/flash.h -- and, in its last part, attention over a
 * paged key-value cache for generation.
 *
 * Buffer shapes (src/flash.h:29-35), all fp32, caller-owned device memory:
 *   qkv  (B, T, 3C)   fused QKV projection output, [q|k|v] along 3C,
 *                     head h at column offset h*hs, hs = C / NH
 *   out  (B, T, C)
 *   lse  (B, NH, T)   natural-log log-sum-exp of each row's scaled scores
 *   dqkv (B, T, 3C)   written, not accumulated
 *   dsum (B, NH, T)   backward scratch: rowsum(dout * out)
 * scale = 1/sqrt(hs). The T x T score matrix is never materialised. Launches
 * go to the null stream. Supported head sizes: 32, 64, 128.
 *
 * Memory: the default backward config stores the causal 32x32 tiles of dS
 * (fp32, 4 KiB each, B*NH*n(n+1)/2 of them with n = ceil(T/32)) in a
 * workspace that each call leases from a library-owned pool of the device
 * and returns once it has queued its work; the pool keeps its buffers for
 * reuse until the process ends and holds as many as were ever leased at once
 * (one per concurrently calling host thread), however many threads come and
 * go. All of it runs on the null stream, where launches from every host
 * thread run in submission order, so the next call to lease a buffer runs
 * after the last one that used it. If it cannot be allocated the backward
 * falls back to a config that recomputes S and dP instead and allocates
 * nothing; flash_attention_backward_cfg can select such a config directly.
 * The same configs run as persistent
 * workgroups on a per-shape work plan that the first backward call of a
 * shape computes on the host and uploads (a few KB per pass, kept per device
 * until the process ends): that first call therefore makes two small
 * allocations and two synchronous copies. Likewise the default forward
 * config, when its whole grid fits on the device at once, places its work
 * by a per-shape order that its first call of a shape uploads (4 bytes per
 * workgroup: one small allocation and one synchronous copy).
 */
#ifndef BMB_FLASH_H
#define BMB_FLASH_H

#include <stddef.h>
#ifndef __cplusplus
#include <stdbool.h>
#endif

struct ihipStream_t; /* hipStream_t is a pointer to it */

/* Element types of the paged cache's buffers and of logits_process (nn.h). */
#ifndef BMB_F32
#define BMB_F32 0
#define BMB_F16 1
#define BMB_BF16 2
#endif

#ifdef __cplusplus
extern "C" {
#endif
/* Only the declarations below are exported from libbmb.so (built with -fvisibility=hidden). */
#pragma GCC visibility push(default)

/* src/flash.h:36-37. Runs the default config, then any legal config; if none
 * fits the head size, prints a message and calls exit(1) like the reference
 * (src/flash.cu:419-432). */
void flash_attention_forward(float *out, float *lse, const float *qkv, int B,
                             int T, int C, int NH);

/* src/flash.h:39-41. Same fallback rule (src/flash.cu:988-1003). */
void flash_attention_backward(float *dqkv, float *dsum, const float *dout,
                              const float *qkv, const float *out,
                              const float *lse, int B, int T, int C, int NH);

/* Tuning harness, src/flash.h:48-53: configs are enumerated and named; the
 * _cfg entry returns false (launching nothing) for an unknown id, a head size
 * the config cannot serve, or a shape it cannot run. */
int flash_num_configs(void);
const char *flash_config_name(int cfg);
int flash_default_config(void);
bool flash_attention_forward_cfg(int cfg, float *out, float *lse,
                                 const float *qkv, int B, int T, int C, int NH);

/* src/flash.h:56-62 */
int flash_num_bwd_configs(void);
const char *flash_bwd_config_name(int cfg);
int flash_default_bwd_config(void);
bool flash_attention_backward_cfg(int cfg, float *dqkv, float *dsum,
                                  const float *dout, const float *qkv,
                                  const float *out, const float *lse, int B,
                                  int T, int C, int NH);

/* ---- Generation: a paged key-value cache. No counterpart in the reference,
 * which runs the whole forward again for every sampled token.
 *
 * The cache is a pool of pages, each page_size tokens of one request; a
 * request's block table lists its pages in order. A generation step is
 *   paged_plan       once: pages, slots and positions of the step's tokens;
 *   paged_append     per layer: their keys and values into the cache;
 *   paged_attention  per layer: attention of one new token a request.
 * (Prompts that start a request attend by flash_attention_forward; append puts
 * their keys and values, which lie in the fused QKV rows, into the cache.)
 *
 * Everything is queued on `stream` of the current device, where all buffers
 * live; results overlap neither inputs nor each other unless said so. Each
 * call returns 0 once its work is queued (a launch that fails shows in
 * bmb_last_error()), or -1 with a message on stderr, and nothing launched, for
 * arguments it refuses. The structs are host memory, read during the call.
 * What lies in device memory cannot be refused: lengths are read as if clipped
 * to their range, and page ids, slots and rows outside theirs are skipped. All
 * results depend on the inputs alone (no floating-point atomics; a request's
 * last bits on how its batch is split), but for a slot that is given twice.
 * Nothing is allocated and nothing outside the given buffers is used, so every
 * call can be captured into a graph (for paged_attention that holds with a
 * workspace of the caller's, below). */

/* Keys and values of one layer. Element (page, token, head, d) of either half
 * is at page*page_stride + token*token_stride + head*head_stride + d, in
 * elements; buffers and strides are multiples of 16 bytes. head_size: 32, 64
 * or 128. pages * page_size < 2^31, token_stride < 2^26. (Pages of a multiple
 * of 16 tokens are read fastest; paged_attention refuses others where the last
 * token of the last page starts 64 GiB - 16 bytes or more behind the first.) */
typedef struct PagedCache {
    void *k, *v;
    int type; /* BMB_F32, BMB_F16 or BMB_BF16 */
    int pages, page_size, kv_heads, head_size;
    long long page_stride, token_stride, head_stride;
} PagedCache;

/* One step of up to 8192 requests. Request r holds lens[r] tokens in the first
 * ceil(lens[r] / page_size) pages of its row of block_table (max_pages
 * columns); new_tokens[r] is 0 (idle), -1 (ended: its pages return to the
 * pool) or the number of tokens it brings (1, or a prompt's). Free pages are
 * the `count` entries of the ring free_pages (`pages` entries) from `head` on;
 * state is {head, count}. Ended requests' pages join the ring's end, in
 * request order, and serve from the next step on.
 *
 * A request is granted all its tokens or none: none if it would pass
 * max_pages; none if it needs new pages and the needs of all requests up to
 * it (those that would pass max_pages aside) exceed count; none if the tokens
 * of all requests up to it that have pages exceed max_tokens. */
typedef struct PagedPlan {
    int requests, max_pages, pages, page_size, max_tokens;
    const int *new_tokens; /* (requests) */
    const int *lens;       /* (requests): tokens held before the step */
    int *lens_out;         /* (requests): after it; may be lens, overlap no other way */
    const int *state;      /* (2) */
    int *state_out;        /* (2); may be state, overlap no other way */
    int *free_pages;       /* (pages): entries behind the last free one are written */
    int *block_table;      /* (requests, max_pages): columns of new pages are written */
    int *slots;            /* (max_tokens): page * page_size + place in it; -1 behind the last */
    int *positions;        /* (max_tokens): place in the request; 0 behind the last */
    int *rows;             /* (requests): its last token's row; -1 without tokens */
    int *offsets;          /* (requests + 1): its first token's row; [requests] is their number */
} PagedPlan;
int paged_plan(const PagedPlan *plan, struct ihipStream_t *stream);

/* cache[slots[t]] = k, v rows of token t for t < tokens, rounded to the
 * cache's type. A row is kv_heads * head_size elements of `type` (BMB_F32, or
 * the cache's own), row_stride elements after the one before (3C in fused QKV
 * rows); rows are multiples of 4 bytes apart. Slots outside the cache (-1) are
 * skipped; of a slot given twice, each 8 elements are either row's. */
int paged_append(const PagedCache *cache, const void *k, const void *v, int type,
                 long long row_stride, const int *slots, int tokens, struct ihipStream_t *stream);

/* The requests of paged_attention. Request r attends to its first lens[r]
 * tokens with the query in row rows[r] of q (row r where rows is null); a row
 * outside [0, n_rows) takes no part, and rows of `out` and `lse` that no
 * request names are left as they were. Query head h reads kv head
 * h / (heads / kv_heads). No row is named twice. A row of q and out is heads *
 * head_size elements of `type`: BMB_F32 with a cache of any type, or the cache's
 * own. Rows are multiples of 4 bytes apart.
 *
 * work: device memory of paged_attention_workspace() bytes for the partial
 * results of sequences that are split over their length, used by one call at
 * a time (two captured graphs that may run at once need one each); nothing in
 * it needs a value. With a null one the call leases from the library's pool,
 * as gemm() does, and is refused under graph capture if it needs any. */
typedef struct PagedBatch {
    int requests;
    int max_len;      /* no lens[r] is longer: the rest of a longer one is not read */
    int table_stride; /* columns of block_table, at least ceil(max_len / page_size) */
    int heads;        /* query heads, a multiple of kv_heads */
    int n_rows;       /* rows of q, out and lse */
    int type;
    float scale; /* of the scores, 1/sqrt(head_size) as a rule */
    long long q_stride, out_stride; /* elements from row to row */
    const int *block_table, *lens, *rows;
    void *work;
    size_t work_bytes;
} PagedBatch;

/* Bytes of workspace for a call of these sizes (its pointers are not looked
 * at); 0 if it needs none, or for arguments that the call would refuse. */
size_t paged_attention_workspace(const PagedCache *cache, const PagedBatch *batch);

/* out[row, h] = sum_j p_j v_j with p = softmax_j(scale q.k_j) over the
 * request's tokens; lse[row, h] (n_rows * heads floats, or null) is the natural
 * log-sum-exp of the scaled scores. A request without tokens, or whose every
 * score is -inf, gives 0 and -inf. Tokens in pages outside the cache count as
 * absent, and what lies in a page behind the last token has no influence.
 * Products and sums are fp32; with 16-bit queries a probability enters its
 * products as two 16-bit numbers, so there an infinite v_j gives NaN in its
 * element of the result. What they lose is at most 2^-17 of a probability in
 * bf16, and in fp16 2^-23 of it or, if that is more, 2^-40 of the request's
 * largest. */
int paged_attention(const PagedCache *cache, const PagedBatch *batch, void *out, float *lse,
                    const void *q, struct ihipStream_t *stream);

#pragma GCC visibility pop
#ifdef __cplusplus
}
#endif
#endif
