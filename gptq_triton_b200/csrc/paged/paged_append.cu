// Rotation of the new queries and keys, and the store of the new key and value rows into their slots.
//   q' = q cos + turn(q) sin per head, turn(x) = (-x[rot/2 ..], x[.. rot/2]); the same for k; v is copied.  fp32 inside, one rounding.
// Every row is read and written once: bound by HBM for prompts, by the launch for a step.
#include "paged.cuh"

namespace gptq {

namespace {

// Thread: entries [e, e + VEC) of the first half of a head's rotated part and their partners, or VEC entries that are not rotated.
template <typename T>
__global__ void __launch_bounds__(256) append_kernel(const paged_append_t p, int units) {
	const int head_count = p.heads + 2 * p.kv_heads;
	const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x, total = (int64_t)p.rows * head_count * units;
	if (at >= total) return;
	const int unit = (int)(at % units), h = (int)(at / units % head_count), m = (int)(at / units / head_count);
	const int kind = h < p.heads ? 0 : h < p.heads + p.kv_heads ? 1 : 2, hh = kind == 0 ? h : kind == 1 ? h - p.heads : h - p.heads - p.kv_heads;
	const T *src = kind == 0   ? reinterpret_cast<const T *>(p.q) + (int64_t)m * p.q_row + (int64_t)hh * p.q_head
				   : kind == 1 ? reinterpret_cast<const T *>(p.k) + (int64_t)m * p.k_row + (int64_t)hh * p.k_head
							   : reinterpret_cast<const T *>(p.v) + (int64_t)m * p.v_row + (int64_t)hh * p.v_head;
	const int half = p.rot / 2;
	int pos = 0;
	bool bad = false;
	if (p.rot) {
		pos = p.positions[m];
		if (pos < 0 || pos >= p.max_pos) {          // rotated as position 0, not stored
			bad = true;
			pos = 0;
		}
	}
	T *dst = nullptr;
	if (kind == 0) {
		dst = reinterpret_cast<T *>(p.q_out) + ((int64_t)m * p.heads + hh) * p.dim;
	} else {
		const int64_t slot = p.slots[m];
		if (slot >= (int64_t)p.pages * p.page) bad = true;
		if (slot >= 0 && !bad) {
			const int64_t page = slot / p.page, row = slot - page * p.page;
			dst = kind == 1 ? reinterpret_cast<T *>(p.k_cache) + page * p.k_page + hh * p.k_kv + row * p.dim : reinterpret_cast<T *>(p.v_cache) + page * p.v_page + hh * p.v_kv + row * p.dim;
		}
	}
	if (bad) atomicOr(p.status, PAGED_BAD_INDEX);
	if (!dst) return;
	if (kind < 2 && unit < half) {
		const T *c = reinterpret_cast<const T *>(p.cos_t) + (int64_t)pos * p.rot, *s = reinterpret_cast<const T *>(p.sin_t) + (int64_t)pos * p.rot;
		const float a = PgElem<T>::get(src[unit]), b = PgElem<T>::get(src[unit + half]);
		dst[unit] = PgElem<T>::put(a * PgElem<T>::get(c[unit]) - b * PgElem<T>::get(s[unit]));
		dst[unit + half] = PgElem<T>::put(b * PgElem<T>::get(c[unit + half]) + a * PgElem<T>::get(s[unit + half]));
	} else if (kind == 2 || unit >= 2 * half) {
		dst[unit] = src[unit];
	}
}

}   // namespace

int pg_append_launch(const paged_append_t &p, int dtype, cudaStream_t stream) {
	const int64_t total = (int64_t)p.rows * (p.heads + 2 * p.kv_heads) * p.dim;
	const unsigned ctas = (unsigned)((total + 255) / 256);
	if (dtype == PG_F32) append_kernel<float><<<ctas, 256, 0, stream>>>(p, p.dim);
	else if (dtype == PG_BF16) append_kernel<bf16><<<ctas, 256, 0, stream>>>(p, p.dim);
	else append_kernel<__half><<<ctas, 256, 0, stream>>>(p, p.dim);
	return cuda_status(cudaGetLastError());
}

}   // namespace gptq
