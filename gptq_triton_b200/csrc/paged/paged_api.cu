// C ABI of the paged cache: checks of arguments and the choice of kernels.
#include "paged.cuh"

namespace gptq {
// All the shared memory that a kernel may have, asked for once per kernel and device.
int pg_smem_opt_in(const void *kernel) {
	static std::atomic<const void *> kernels[32];
	static std::atomic<unsigned long long> devices[32];
	int dev = 0, i = 0;
	if (int rc = cuda_status(cudaGetDevice(&dev))) return rc;
	for (; i < 32; ++i) {
		const void *seen = kernels[i].load();
		if (!seen && kernels[i].compare_exchange_strong(seen, kernel)) seen = kernel;
		if (seen == kernel) break;
	}
	const bool kept = i < 32 && dev < 64;
	if (kept && devices[i].load() >> dev & 1) return GPTQ_OK;
	cudaFuncAttributes attr;
	if (int rc = cuda_status(cudaFuncGetAttributes(&attr, kernel))) return rc;
	if (int rc = cuda_status(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024 - (int)attr.sharedSizeBytes))) return rc;
	if (kept) devices[i].fetch_or(1ull << dev);
	return GPTQ_OK;
}
}

using namespace gptq;

namespace {

bool known(int dtype) { return dtype == PG_BF16 || dtype == PG_F32 || dtype == PG_F16; }
int size_of(int dtype) { return dtype == PG_F32 ? 4 : 2; }
bool page_ok(int page) { return page >= 1 && page <= PAGED_MAX_PAGE; }
bool heads_ok(int heads, int kv_heads) { return kv_heads >= 1 && heads >= kv_heads && heads % kv_heads == 0 && heads <= 65535; }
// heads and pages start on 16 bytes
bool steps_ok(int64_t a, int64_t b, int dtype) { return a * size_of(dtype) % 16 == 0 && b * size_of(dtype) % 16 == 0; }
// pages, and key heads within them, are places of their own
template <typename P>
bool places_ok(const P &p) {
	const int64_t least = (int64_t)p.page * p.dim;
	return !(p.pages > 1 && (p.k_page < least || p.v_page < least)) && !(p.kv_heads > 1 && (p.k_kv < least || p.v_kv < least));
}

bool tiles(const paged_attention_t &p, int dtype) { return p.pages > 0 && pg_tiles_serve(dtype, p.dim, p.page, p.max_fresh, p.heads, p.kv_heads); }

}   // namespace

extern "C" {

int paged_version(void) { return 100; }
int paged_last_cuda_error(void) { return g_last_cuda_error; }

int64_t paged_work_ints(int requests, int rows, int heads, int kv_heads) {
	if (requests < 0 || requests > PAGED_MAX_REQUESTS || rows < 0 || rows >= 1 << 30 || !heads_ok(heads, kv_heads) || (int64_t)rows * (heads / kv_heads) >= (int64_t)1 << 31) return -1;
	return pg_work(nullptr, requests, rows, heads, kv_heads).ints;
}

int paged_plan(const paged_plan_t *p, int dtype, void *stream) {
	if (!p || !known(dtype) || p->requests < 0 || p->requests > PAGED_MAX_REQUESTS || p->rows < 0 || !page_ok(p->page) || p->pages < 0 || p->table_width < 1 || p->table_ld < p->table_width ||
		!heads_ok(p->heads, p->kv_heads) || !p->row_start || !p->work || !p->status || p->max_fresh < 0 || paged_work_ints(p->requests, p->rows, p->heads, p->kv_heads) < 0)
		return GPTQ_ERR_INVALID;
	if (p->requests && (!p->past || !p->fresh || !p->table || !p->lens)) return GPTQ_ERR_INVALID;
	if (p->rows && (!p->positions || !p->slots)) return GPTQ_ERR_INVALID;
	if (p->pool && (!p->head || !p->next_head || p->head == p->next_head || p->pool_size < 0)) return GPTQ_ERR_INVALID;
	if (!aligned16(p->work)) return GPTQ_ERR_ALIGN;
	return pg_plan_launch(*p, dtype, (cudaStream_t)stream);
}

int paged_append(const paged_append_t *p, int dtype, void *stream) {
	if (!p || !known(dtype) || p->rows < 0 || !heads_ok(p->heads, p->kv_heads) || p->dim < 1 || p->rot < 0 || p->rot > p->dim || p->rot % 2 || !page_ok(p->page) || p->pages < 0 || !p->status)
		return GPTQ_ERR_INVALID;
	if (p->rows == 0) return GPTQ_OK;
	if (!p->q || !p->k || !p->v || !p->q_out || !p->k_cache || !p->v_cache || !p->slots || (p->rot && (!p->cos_t || !p->sin_t || !p->positions || p->max_pos < 1)) || !places_ok(*p))
		return GPTQ_ERR_INVALID;
	return pg_append_launch(*p, dtype, (cudaStream_t)stream);
}

int64_t paged_attention_scratch(const paged_attention_t *p, int dtype) {
	if (!p || !known(dtype) || p->dim < 1 || p->dim > PAGED_MAX_DIM) return -1;
	if (!heads_ok(p->heads, p->kv_heads) || !page_ok(p->page)) return -1;
	return pg_rows_scratch(*p) + (tiles(*p, dtype) ? pg_tiles_scratch(*p) : 0);
}

int paged_attention(const paged_attention_t *p, int dtype, void *stream) {
	if (!p || !known(dtype) || p->requests < 0 || p->requests > PAGED_MAX_REQUESTS || p->rows < 0 || !heads_ok(p->heads, p->kv_heads) || !page_ok(p->page) || p->pages < 0 || p->table_width < 1 ||
		p->table_ld < p->table_width || !(p->scale > 0.f) || !(p->scale <= 3.4e38f) || !p->status || p->max_fresh < 0 || paged_work_ints(p->requests, p->rows, p->heads, p->kv_heads) < 0)
		return GPTQ_ERR_INVALID;
	if (p->dim < 1 || p->dim > PAGED_MAX_DIM || p->dim % 8) return GPTQ_ERR_SHAPE;
	if (p->requests == 0 || p->rows == 0) return GPTQ_OK;
	if (!p->q || !p->k_cache || !p->v_cache || !p->table || !p->row_start || !p->lens || !p->work || !p->out) return GPTQ_ERR_INVALID;
	if (!places_ok(*p)) return GPTQ_ERR_INVALID;
	if (!steps_ok(p->k_page, p->k_kv, dtype) || !steps_ok(p->v_page, p->v_kv, dtype) || !steps_ok(p->q_row, p->q_head, dtype) || !aligned16(p->q) || !aligned16(p->k_cache) || !aligned16(p->v_cache) ||
		!aligned16(p->out))
		return GPTQ_ERR_ALIGN;
	if (!p->scratch || !aligned16(p->scratch) || (int64_t)p->scratch_bytes < paged_attention_scratch(p, dtype)) return GPTQ_ERR_WORKSPACE;
	const bool both = tiles(*p, dtype);
	char *tile_scratch = both ? (char *)p->scratch + pg_rows_scratch(*p) : nullptr;
	if (both)
		if (int rc = pg_tiles_launch(*p, dtype, tile_scratch, (cudaStream_t)stream)) return rc;
	if (int rc = pg_rows_launch(*p, dtype, both, (cudaStream_t)stream)) return rc;
	return pg_join_launch(*p, dtype, tile_scratch, (cudaStream_t)stream);
}

}   // extern "C"
