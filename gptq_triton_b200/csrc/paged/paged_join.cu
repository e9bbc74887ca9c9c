// Joins the partial results of tiles whose keys are spread over several slots of an attention kernel: numerators, maxima (base 2) and sums
// of a row, in the order of the slots.
//   m = max m_i,  l = sum l_i 2^(m_i - m),  out = (sum a_i 2^(m_i - m)) / l
#include "paged.cuh"

namespace gptq {

namespace {

constexpr int JN_THREADS = 256, JN_CTAS = 296;
__host__ __device__ constexpr int jn_rows(int kind) { return kind ? 32 : 4; }          // rows of a tile that a CTA joins at a time

template <typename T> __device__ __forceinline__ void store_four(T *dst, float4 v) { *reinterpret_cast<uint2 *>(dst) = make_uint2(pack2<T>(v.x, v.y), pack2<T>(v.z, v.w)); }
template <> __device__ __forceinline__ void store_four<float>(float *dst, float4 v) { *reinterpret_cast<float4 *>(dst) = v; }

// kind 0: tiles of PG_ROWS rows, 1: of PG_TILE rows; DP: columns of a partial result
template <typename T, int DP>
__device__ void join(const paged_attention_t &p, int kind, int slot, int row0, const float *scratch, const PgStart &s, int more) {
	const int group = p.heads / p.kv_heads, tile_rows = kind ? PG_TILE : PG_ROWS;
	const PgEntry &e = s.job;
	auto part = [&](int i) { return scratch + (int64_t)(i == 0 ? 2 * slot + 1 : 2 * (slot + i)) * tile_rows * (DP + 2); };
	// Several threads share an entry of the result where there are enough of them, each takes every `shares`-th partial result.
	__shared__ float s_m[JN_THREADS], s_l[JN_THREADS];
	__shared__ float4 s_a[JN_THREADS];
	const int rows = (int)min((int64_t)jn_rows(kind), (int64_t)e.fresh * group - (int64_t)e.tile * tile_rows - row0), items = rows * (DP / 4);
	if (rows <= 0) return;
	const int shares = items >= JN_THREADS ? 1 : min(JN_THREADS / items, more + 1);
	for (int base = 0; base < items; base += JN_THREADS) {
		const int x = shares > 1 ? threadIdx.x % items : base + threadIdx.x, share = shares > 1 ? threadIdx.x / items : 0;
		const int row = row0 + x / (DP / 4), col = x % (DP / 4) * 4;
		const bool mine = x < items && share < shares && col < p.dim;
		float m = -INFINITY, l = 0.f;
		float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
		constexpr int BATCH = 8;                             // partial results that are asked for at once
		if (mine)
			for (int i0 = share; i0 <= more; i0 += BATCH * shares) {
				float2 ml[BATCH];
				float4 y[BATCH];
#pragma unroll
				for (int i = 0; i < BATCH; ++i)
					if (i0 + i * shares <= more) {
						ml[i] = __ldcg(reinterpret_cast<const float2 *>(part(i0 + i * shares) + (int64_t)tile_rows * DP) + row);
						y[i] = __ldcg(reinterpret_cast<const float4 *>(part(i0 + i * shares) + (int64_t)row * DP + col));
					}
				float top = m;
#pragma unroll
				for (int i = 0; i < BATCH; ++i)
					if (i0 + i * shares <= more) top = fmaxf(top, ml[i].x);
				const float keep = m == -INFINITY ? 0.f : ex2(m - top);
				m = top;
				l *= keep;
				a = make_float4(a.x * keep, a.y * keep, a.z * keep, a.w * keep);
#pragma unroll
				for (int i = 0; i < BATCH; ++i)
					if (i0 + i * shares <= more) {
						const float f = ml[i].x == -INFINITY ? 0.f : ex2(ml[i].x - top);
						l = fmaf(ml[i].y, f, l);
						a = make_float4(fmaf(y[i].x, f, a.x), fmaf(y[i].y, f, a.y), fmaf(y[i].z, f, a.z), fmaf(y[i].w, f, a.w));
					}
			}
		if (shares > 1) {
			__syncthreads();                                   // (the values of the job before have been read)
			s_m[threadIdx.x] = m;
			s_l[threadIdx.x] = l;
			s_a[threadIdx.x] = a;
			__syncthreads();
			if (share > 0) continue;
			float top = m;
			for (int i = 1; i < shares; ++i) top = fmaxf(top, s_m[x + i * items]);
			const float keep = m == -INFINITY ? 0.f : ex2(m - top);
			l *= keep;
			a = make_float4(a.x * keep, a.y * keep, a.z * keep, a.w * keep);
			for (int i = 1; i < shares; ++i) {
				const float f = s_m[x + i * items] == -INFINITY ? 0.f : ex2(s_m[x + i * items] - top);
				const float4 y = s_a[x + i * items];
				l = fmaf(s_l[x + i * items], f, l);
				a = make_float4(fmaf(y.x, f, a.x), fmaf(y.y, f, a.y), fmaf(y.z, f, a.z), fmaf(y.w, f, a.w));
			}
		}
		if (!mine) continue;
		const int64_t at = (int64_t)e.tile * tile_rows + row;
		const int token = (int)(at / group), head = (int)(at - (int64_t)token * group);
		const bool blind = e.len - e.fresh + token < 0;          // a row that sees nothing
		const float f = 1.f / l;
		store_four<T>(reinterpret_cast<T *>(p.out) + ((int64_t)(e.row + token) * p.heads + s.kv * group + head) * p.dim + col,
					  blind ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(a.x * f, a.y * f, a.z * f, a.w * f));
	}
}

// CTAs go over the jobs that were cut (the plan lists the slots in which they begin), a few rows at a time.
template <typename T, int DP>
__global__ void __launch_bounds__(JN_THREADS, 3) join_kernel(const paged_attention_t p, const PgWork work, const float *tile_scratch) {
	const PgList few = read_list(work.list);               // (the plan was complete before the attention kernels could start this one)
	PgList many = {};
	if (tile_scratch) many = read_list(work.list + 1);
	pdl_wait();
	pdl_trigger();
	for (int kind = 0; kind < 2; ++kind) {
		const PgList &list = kind ? many : few;
		const int slots = kind ? PG_TILE_SLOTS : PG_SLOTS, groups = (kind ? PG_TILE : PG_ROWS) / jn_rows(kind), count = list.cuts[0] + list.cuts[1];
		if (kind && DP > 128) break;
		for (int x = blockIdx.x; x < count * groups; x += gridDim.x) {
			const int i = x % count, row0 = x / count * jn_rows(kind);
			const int slot = __ldcg(work.cuts[kind] + (i < list.cuts[0] ? i : slots + i - list.cuts[0]));
			const PgStart s = read_start(work.starts[kind] + slot + 1);
			if (row0 >= (int64_t)s.job.fresh * (p.heads / p.kv_heads) - (int64_t)s.job.tile * (kind ? PG_TILE : PG_ROWS)) continue;
			const int more = (int)((s.job.blocks - s.block + list.per - 1) / list.per);          // further slots that the job runs through
			join<T, DP>(p, kind, slot, row0, kind ? tile_scratch : reinterpret_cast<const float *>(p.scratch), s, more);
		}
	}
}

template <typename T>
int launch(const paged_attention_t &p, const float *tile_scratch, cudaStream_t stream) {
	const PgWork work = pg_work(const_cast<int32_t *>(p.work), p.requests, p.rows, p.heads, p.kv_heads);
	const dim3 grid(JN_CTAS);
	if (p.dim <= 64) return pg_launch(join_kernel<T, 64>, grid, JN_THREADS, 0, stream, p, work, tile_scratch);
	if (p.dim <= 128) return pg_launch(join_kernel<T, 128>, grid, JN_THREADS, 0, stream, p, work, tile_scratch);
	return pg_launch(join_kernel<T, 256>, grid, JN_THREADS, 0, stream, p, work, tile_scratch);
}

}   // namespace

int pg_join_launch(const paged_attention_t &p, int dtype, char *tile_scratch, cudaStream_t stream) {
	const float *t = reinterpret_cast<const float *>(tile_scratch);
	return dtype == PG_BF16 ? launch<bf16>(p, t, stream) : dtype == PG_F16 ? launch<__half>(p, t, stream) : launch<float>(p, t, stream);
}

}   // namespace gptq
