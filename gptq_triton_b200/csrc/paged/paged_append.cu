// Rotation of the new queries and keys, and the store of the new key and value rows into their slots.
//   q' = q cos + turn(q) sin per head, turn(x) = (-x[rot/2 ..], x[.. rot/2]); the same for k; v is copied.  fp32 inside, one rounding.
// Every row is read and written once: bound by HBM for prompts, by the launch for a step.
#include <climits>

#include "paged.cuh"

namespace gptq {

namespace {

constexpr int AP_THREADS = 128;          // 4 806 rows of 80 heads of 128, us: 128 threads 37.0, 256 39.0, 320 40.8, 512 49.1; with 256, heads per thread 1 39.2, 2 39.0, 4 57.0

// Position (of the tables), page and row of the page of row m; a position outside the tables: position 0, no page (-1).
struct Place {
	int pos, page, row;
	__device__ __forceinline__ Place(const paged_append_t &p, int m) : pos(0), page(-1), row(0) {
		const int64_t slot = __ldcg(p.slots + m);
		bool bad = false;
		if (p.rot) {
			pos = __ldcg(p.positions + m);
			if (pos < 0 || pos >= p.max_pos) {
				bad = true;
				pos = 0;
			}
		}
		if (slot >= (int64_t)p.pages * p.page) bad = true;
		if (bad) {
			atomicOr(p.status, PAGED_BAD_INDEX);
		} else if (slot >= 0) {
			page = slot <= INT_MAX ? (int)((unsigned)slot / (unsigned)p.page) : (int)(slot / p.page);
			row = (int)(slot - (int64_t)page * p.page);
		}
	}
};

// Where head h (queries, keys, values in this order) of row m comes from and goes to; dst NULL: nowhere.
template <typename T>
struct Route {
	const T *src;
	T *dst;
	bool turned;
	__device__ __forceinline__ Route(const paged_append_t &p, int m, int h, const Place &at) {
		turned = h < p.heads + p.kv_heads;
		if (h < p.heads) {
			src = reinterpret_cast<const T *>(p.q) + (int64_t)m * p.q_row + (int64_t)h * p.q_head;
			dst = reinterpret_cast<T *>(p.q_out) + ((int64_t)m * p.heads + h) * p.dim;
			return;
		}
		const int g = h - p.heads - (turned ? 0 : p.kv_heads);
		src = turned ? reinterpret_cast<const T *>(p.k) + (int64_t)m * p.k_row + (int64_t)g * p.k_head : reinterpret_cast<const T *>(p.v) + (int64_t)m * p.v_row + (int64_t)g * p.v_head;
		T *cache = reinterpret_cast<T *>(turned ? p.k_cache : p.v_cache);
		dst = at.page < 0 ? nullptr : cache + at.page * (turned ? p.k_page : p.v_page) + g * (turned ? p.k_kv : p.v_kv) + (int64_t)at.row * p.dim;
	}
};

template <typename T>
__device__ __forceinline__ T fetch(const T *p) {          // through L2
	if constexpr (sizeof(T) == 2) {
		const unsigned short v = __ldcg(reinterpret_cast<const unsigned short *>(p));
		return *reinterpret_cast<const T *>(&v);
	} else {
		return __ldcg(p);
	}
}

// Any sizes and strides: a thread per entry (and its partner).
template <typename T>
__global__ void __launch_bounds__(256) append_entries_kernel(const paged_append_t p) {
	pdl_wait();
	pdl_trigger();
	const int head_count = p.heads + 2 * p.kv_heads;
	const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x, total = (int64_t)p.rows * head_count * p.dim;
	if (at >= total) return;
	const int unit = (int)(at % p.dim), h = (int)(at / p.dim % head_count), m = (int)(at / p.dim / head_count), half = p.rot / 2;
	const Place at_row(p, m);
	const Route<T> r(p, m, h, at_row);
	if (!r.dst) return;
	if (r.turned && unit < half) {
		const T *c = reinterpret_cast<const T *>(p.cos_t) + (int64_t)at_row.pos * p.rot, *s = reinterpret_cast<const T *>(p.sin_t) + (int64_t)at_row.pos * p.rot;
		const float a = PgElem<T>::get(fetch(r.src + unit)), b = PgElem<T>::get(fetch(r.src + unit + half));
		r.dst[unit] = PgElem<T>::put(a * PgElem<T>::get(c[unit]) - b * PgElem<T>::get(s[unit]));
		r.dst[unit + half] = PgElem<T>::put(b * PgElem<T>::get(c[unit + half]) + a * PgElem<T>::get(s[unit + half]));
	} else if (!r.turned || unit >= 2 * half) {
		r.dst[unit] = fetch(r.src + unit);
	}
}

// 16 bytes at a time.  A CTA works on a row, a thread on two runs of 16 bytes, VEC entries and their partners (or two runs that are only
// copied), of HEADS heads, whose cosines and sines it reads once.
template <typename T, int HEADS>
__global__ void __launch_bounds__(AP_THREADS) append_kernel(const paged_append_t p, int units, int pairs) {
	pdl_wait();
	pdl_trigger();
	constexpr int VEC = 16 / sizeof(T);
	const int at = blockIdx.y * AP_THREADS + threadIdx.x, m = blockIdx.x;
	if (at >= pairs) return;
	const int g = (int)((unsigned)at / (unsigned)units), unit = at - g * units, head_count = p.heads + 2 * p.kv_heads, h0 = g * HEADS;
	union Run {
		uint4 raw;
		T v[VEC];
	};
	const int turned = p.rot / 2 / VEC;                    // pairs of runs that are rotated
	const bool turn = unit < turned;
	const int a = turn ? unit : 2 * turned + 2 * (unit - turned), b = turn ? unit + turned : a + 1, last = p.dim / VEC;
	const Place place(p, m);
	Run x[HEADS][2], c[2], s[2];
	T *to[HEADS];
	bool rotate[HEADS];
#pragma unroll
	for (int i = 0; i < HEADS; ++i) {
		to[i] = nullptr;
		if (h0 + i < head_count) {
			const Route<T> r(p, m, h0 + i, place);
			to[i] = r.dst;
			rotate[i] = turn && r.turned;
			const uint4 *src = reinterpret_cast<const uint4 *>(r.src);
			x[i][0].raw = __ldcg(src + a);
			if (b < last) x[i][1].raw = __ldcg(src + b);
		}
	}
	if (turn) {
		const uint4 *ct = reinterpret_cast<const uint4 *>(reinterpret_cast<const T *>(p.cos_t) + (int64_t)place.pos * p.rot), *st = reinterpret_cast<const uint4 *>(reinterpret_cast<const T *>(p.sin_t) + (int64_t)place.pos * p.rot);
		c[0].raw = __ldg(ct + a);
		c[1].raw = __ldg(ct + b);
		s[0].raw = __ldg(st + a);
		s[1].raw = __ldg(st + b);
	}
#pragma unroll
	for (int i = 0; i < HEADS; ++i)
		if (to[i]) {
			if (rotate[i]) {
#pragma unroll
				for (int k = 0; k < VEC; ++k) {
					const float u = PgElem<T>::get(x[i][0].v[k]), w = PgElem<T>::get(x[i][1].v[k]);
					x[i][0].v[k] = PgElem<T>::put(u * PgElem<T>::get(c[0].v[k]) - w * PgElem<T>::get(s[0].v[k]));
					x[i][1].v[k] = PgElem<T>::put(w * PgElem<T>::get(c[1].v[k]) + u * PgElem<T>::get(s[1].v[k]));
				}
			}
			uint4 *dst = reinterpret_cast<uint4 *>(to[i]);
			dst[a] = x[i][0].raw;
			if (b < last) dst[b] = x[i][1].raw;
		}
}

template <typename T>
int launch(const paged_append_t &p, cudaStream_t stream) {
	constexpr int VEC = 16 / sizeof(T);
	const int head_count = p.heads + 2 * p.kv_heads;
	bool wide = p.dim % VEC == 0 && p.rot % (2 * VEC) == 0;
	for (int64_t s : {p.q_row, p.q_head, p.k_row, p.k_head, p.v_row, p.v_head, p.k_page, p.k_kv, p.v_page, p.v_kv}) wide = wide && s % VEC == 0;
	for (const void *q : {p.q, p.k, p.v, (const void *)p.q_out, (const void *)p.k_cache, (const void *)p.v_cache, p.cos_t, p.sin_t}) wide = wide && aligned16(q);
	if (!wide) {
		const int64_t total = (int64_t)p.rows * head_count * p.dim;
		return pg_launch(append_entries_kernel<T>, dim3((unsigned)((total + 255) / 256)), 256, 0, stream, p);
	}
	const int units = p.rot / 2 / VEC + ((p.dim - p.rot) / VEC + 1) / 2;
	// several heads per thread where that leaves a full wave of threads
	constexpr int MANY = 2;
	const int many = (head_count + MANY - 1) / MANY;
	auto go = [&](auto kernel, int pairs) { return pg_launch(kernel, dim3((unsigned)p.rows, (unsigned)((pairs + AP_THREADS - 1) / AP_THREADS)), AP_THREADS, 0, stream, p, units, pairs); };
	return (int64_t)p.rows * many * units >= 148 * 2048 ? go(append_kernel<T, MANY>, many * units) : go(append_kernel<T, 1>, head_count * units);
}

}   // namespace

int pg_append_launch(const paged_append_t &p, int dtype, cudaStream_t stream) { return dtype == PG_F32 ? launch<float>(p, stream) : dtype == PG_BF16 ? launch<bf16>(p, stream) : launch<__half>(p, stream); }

}   // namespace gptq
