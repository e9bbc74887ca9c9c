/*
 * paged_b200.h — C ABI of libgptq_b200.so, continued: serving from a key / value cache in pages on NVIDIA B200 (sm_100a).
 * Block tables and slot maps from request lengths, rotation of queries and keys with the store of the new rows, attention of the
 * new tokens of every request over its pages.
 *
 * Every pointer inside the argument blocks is a DEVICE pointer.  Entry points are asynchronous on `stream`, never synchronise,
 * allocate or free, keep nothing between calls, and return 0 or a negative GPTQ_ERR_* code (gptq_b200.h).  Lengths are read on the
 * device only, and the launches do not depend on them: a captured graph serves other lengths of as many requests and rows.
 *
 * dtype: 0 = bf16, 1 = fp32, 2 = fp16 (queries, cache and results alike; sums and softmax statistics are fp32).
 * A cache tensor is [pages, kv_heads, page, dim] with the rows of a page contiguous; pages and heads may lie further apart.
 */
#ifndef PAGED_B200_H
#define PAGED_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define PAGED_MAX_REQUESTS 8192
#define PAGED_MAX_DIM 256
#define PAGED_MAX_PAGE (1 << 24)      /* positions count up to 2^30 */
/* bits of the status word, none of them a code of gptq_b200.h with another meaning (a run that meets one goes on without touching memory that is not its own) */
#define PAGED_BAD_INDEX 4              /* a page, position or slot outside the cache or the tables, or a negative length */
#define PAGED_NO_ROOM 8                /* pages of the pool, columns of the table or rows ran out, or a request has more than max_fresh new tokens; or the
                                          requests see more keys than the work lists count (2^30 blocks of 16): the attention then computes nothing */
#define PAGED_TIMED_OUT 16             /* a wait inside the attention's kernel for chunks ran out */

/* The plan of one step.  Request r has past[r] tokens in the cache and gets fresh[r] new ones (0 is allowed).  Rows are the new
 * tokens, request after request; rows behind the last one get slot -1 and position 0.
 *   pages:  full(r) = ceil((past + fresh) / page).  With a pool, entries ceil(past / page) .. full(r) - 1 of table row r become
 *           pool[*head ..], requests in order; *next_head = *head + the number taken.  Without, the table is complete.
 *   slots:  table[r, p / page] * page + p % page of position p = past + i.
 * `work` is the distribution of the attention's work over the processors, for `heads` query heads (PAGED_WORK of it). */
typedef struct {
	int requests, rows, table_width, page, pages, pool_size;
	int64_t table_ld;
	const int32_t *past, *fresh;
	int32_t *table;
	const int32_t *pool, *head;        /* NULL: no pages are taken */
	int32_t *next_head;                /* not *head itself */
	int32_t *row_start;                /* [requests + 1] */
	int32_t *lens;                     /* [requests]: past + fresh */
	int32_t *positions;                /* [rows] */
	int64_t *slots;                    /* [rows] */
	int heads, kv_heads, dim;
	int max_fresh;                     /* no request has more new tokens (rows, if nothing is known); one that has sets PAGED_NO_ROOM */
	int32_t *work;
	int *status;
} paged_plan_t;

/* q_out = rotated q; rotated k and v to their slots.  Rotation: the first rot entries of a head, pairs (i, i + rot / 2), by row
 * positions[m] of the tables [max_pos, rot] (rot = 0: none).  A row with slot -1 is rotated but not stored. */
typedef struct {
	int rows, heads, kv_heads, dim, rot, max_pos, page, pages;
	const void *q, *k, *v;             /* [rows, heads, dim] */
	int64_t q_row, q_head, k_row, k_head, v_row, v_head;          /* strides in elements */
	const void *cos_t, *sin_t;         /* [max_pos, rot] in the type of q */
	const int32_t *positions;
	const int64_t *slots;
	void *q_out;                       /* [rows, heads, dim] contiguous */
	void *k_cache, *v_cache;
	int64_t k_page, k_kv, v_page, v_kv;                            /* strides of pages and heads in elements, a page's rows (page * dim) at least */
	int *status;
} paged_append_t;

/* table, row_start, lens and work are those of a plan of the same requests, rows, heads, kv_heads, dim, page, pages, table_width, max_fresh and dtype.
 * out[row] = softmax over positions 0 .. p of scale * q . k, times v; p = position of the row.  Rows that belong to no request
 * (behind the last one) are left as they are. */
typedef struct {
	int requests, rows, heads, kv_heads, dim, page, pages, table_width, max_fresh;
	int64_t table_ld;
	float scale;                       /* positive */
	const void *q;                     /* [rows, heads, dim] */
	int64_t q_row, q_head;
	const void *k_cache, *v_cache;
	int64_t k_page, k_kv, v_page, v_kv;
	const int32_t *table, *row_start, *lens, *work;
	void *out;                         /* [rows, heads, dim] contiguous */
	void *scratch;                     /* paged_attention_scratch bytes, no initial value; 16-byte aligned */
	size_t scratch_bytes;
	int *status;
} paged_attention_t;

int paged_version(void);
int paged_last_cuda_error(void);
/* int32 values of paged_plan_t.work; -1: no plan has these sizes (rows below 2^30, rows times query heads of a key head below 2^31) */
int64_t paged_work_ints(int requests, int rows, int heads, int kv_heads);
int paged_plan(const paged_plan_t *args, int dtype, void *stream);
int paged_append(const paged_append_t *args, int dtype, void *stream);
int64_t paged_attention_scratch(const paged_attention_t *args, int dtype);
int paged_attention(const paged_attention_t *args, int dtype, void *stream);

#ifdef __cplusplus
}
#endif
#endif
