// Attention of few new tokens over a cache in pages.
#include "paged.cuh"

namespace gptq {

namespace {

// A warp serves one row and one query head: a lane holds entries lane, lane + 32 .. of the head; one key after the other with a running
// maximum and sum.
template <typename T>
__global__ void __launch_bounds__(128) simple_kernel(const paged_attention_t p) {
	const int lane = threadIdx.x & 31;
	const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
	const int m = (int)(at / p.heads), h = (int)(at % p.heads), kvh = h / (p.heads / p.kv_heads);
	if (m >= p.rows || m >= p.row_start[p.requests]) return;
	int lo = 0, hi = p.requests;
	while (hi - lo > 1) {
		const int mid = (lo + hi) >> 1;
		if (p.row_start[mid] <= m) lo = mid;
		else hi = mid;
	}
	const int r = lo, pos = p.lens[r] - (p.row_start[r + 1] - m);
	constexpr int N = PAGED_MAX_DIM / 32;
	float q[N], o[N], mx = -INFINITY, sum = 0.f;
#pragma unroll
	for (int i = 0; i < N; ++i) {
		const int d = lane + 32 * i;
		q[i] = d < p.dim ? PgElem<T>::get(reinterpret_cast<const T *>(p.q)[m * p.q_row + h * p.q_head + d]) * p.scale : 0.f;
		o[i] = 0.f;
	}
	bool bad = false;
	for (int j = 0; j <= pos; ++j) {
		const int c = j / p.page;
		const int id = c < p.table_width ? p.table[r * p.table_ld + c] : -1;
		const bool there = id >= 0 && id < p.pages;
		bad |= !there;
		const T *k = reinterpret_cast<const T *>(p.k_cache) + id * p.k_page + kvh * p.k_kv + (int64_t)(j - c * p.page) * p.dim;
		const T *v = reinterpret_cast<const T *>(p.v_cache) + id * p.v_page + kvh * p.v_kv + (int64_t)(j - c * p.page) * p.dim;
		float s = 0.f;
#pragma unroll
		for (int i = 0; i < N; ++i)
			if (there && lane + 32 * i < p.dim) s = fmaf(q[i], PgElem<T>::get(k[lane + 32 * i]), s);
#pragma unroll
		for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
		const float next = fmaxf(mx, s), keep = mx == -INFINITY ? 0.f : __expf(mx - next), w = __expf(s - next);
		sum = sum * keep + w;
#pragma unroll
		for (int i = 0; i < N; ++i) o[i] = fmaf(w, there && lane + 32 * i < p.dim ? PgElem<T>::get(v[lane + 32 * i]) : 0.f, o[i] * keep);
		mx = next;
	}
	if (bad && lane == 0) atomicOr(p.status, PAGED_BAD_INDEX);
#pragma unroll
	for (int i = 0; i < N; ++i)
		if (lane + 32 * i < p.dim) reinterpret_cast<T *>(p.out)[((int64_t)m * p.heads + h) * p.dim + lane + 32 * i] = PgElem<T>::put(pos < 0 ? 0.f : o[i] / sum);
}

}   // namespace

int pg_attend_simple(const paged_attention_t &p, int dtype, cudaStream_t stream) {
	const unsigned ctas = (unsigned)(((int64_t)p.rows * p.heads + 3) / 4);
	if (dtype == PG_F32) simple_kernel<float><<<ctas, 128, 0, stream>>>(p);
	else if (dtype == PG_BF16) simple_kernel<bf16><<<ctas, 128, 0, stream>>>(p);
	else simple_kernel<__half><<<ctas, 128, 0, stream>>>(p);
	return cuda_status(cudaGetLastError());
}

}   // namespace gptq
