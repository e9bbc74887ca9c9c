// Joins the partial results of tiles whose keys are spread over several slots of an attention kernel: numerators, maxima (base 2) and sums
// of a row, in the order of the slots.
//   m = max m_i,  l = sum l_i 2^(m_i - m),  out = (sum a_i 2^(m_i - m)) / l
// A tile that is spread begins in exactly one slot: CTA c looks whether one begins in slot c and ends in a later one.
#include "paged.cuh"

namespace gptq {

namespace {

constexpr int JN_THREADS = 128, JN_ROWS = 16;            // rows of a tile that a CTA joins

template <typename T> __device__ __forceinline__ void store_four(T *dst, float4 v) { *reinterpret_cast<uint2 *>(dst) = make_uint2(pack2<T>(v.x, v.y), pack2<T>(v.z, v.w)); }
template <> __device__ __forceinline__ void store_four<float>(float *dst, float4 v) { *reinterpret_cast<float4 *>(dst) = v; }

// kind 0: tiles of PG_ROWS rows, 1: of PG_TILE rows; DP: columns of a partial result.  Further slots that the job which begins in `slot`
// runs through (0: there is none), and its start in the next one.
__device__ __forceinline__ int cut(const PgWork &work, int kind, int slot, PgStart &s) {
	const int slots = kind ? PG_TILE_SLOTS : PG_SLOTS;
	if (read_list(work.list + kind).whole) return 0;
	const PgStart *starts = work.starts[kind];
	s = read_start(starts + slot + 1);
	const PgStart before = read_start(starts + slot);
	if (s.entry < 0 || s.block == 0 || (before.in_job(s.entry, s.kv) && before.block > 0)) return 0;
	for (int more = 1;; more += 32) {
		const int c = slot + 1 + more + (threadIdx.x & 31);
		bool inside = false;
		if (c <= slots) {
			const int4 n = __ldcg(reinterpret_cast<const int4 *>(starts + c));
			inside = n.x == s.entry && n.y == s.kv && n.z > 0;
		}
		const unsigned gone = ~__ballot_sync(0xffffffffu, inside);
		if (gone) return more + __ffs(gone) - 1;
	}
}

template <typename T, int DP>
__device__ void join(const paged_attention_t &p, int kind, int slot, int row0, const float *scratch, const PgStart &s, int more) {
	const int group = p.heads / p.kv_heads, tile_rows = kind ? PG_TILE : PG_ROWS;
	const PgEntry &e = s.job;
	auto part = [&](int i) { return scratch + (int64_t)(i == 0 ? 2 * slot + 1 : 2 * (slot + i)) * tile_rows * (DP + 2); };
	for (int x = threadIdx.x; x < JN_ROWS * (DP / 4); x += JN_THREADS) {
		const int row = row0 + x / (DP / 4), col = x % (DP / 4) * 4;
		const int64_t at = (int64_t)e.tile * tile_rows + row;
		if (at >= (int64_t)e.fresh * group || col >= p.dim) continue;
		float m = -INFINITY, l = 0.f;
		float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
		constexpr int BATCH = 8;                             // partial results that are asked for at once
		for (int i0 = 0; i0 <= more; i0 += BATCH) {
			float2 ml[BATCH];
			float4 y[BATCH];
#pragma unroll
			for (int i = 0; i < BATCH; ++i)
				if (i0 + i <= more) {
					ml[i] = __ldcg(reinterpret_cast<const float2 *>(part(i0 + i) + (int64_t)tile_rows * DP) + row);
					y[i] = __ldcg(reinterpret_cast<const float4 *>(part(i0 + i) + (int64_t)row * DP + col));
				}
			float top = m;
#pragma unroll
			for (int i = 0; i < BATCH; ++i)
				if (i0 + i <= more) top = fmaxf(top, ml[i].x);
			const float keep = m == -INFINITY ? 0.f : ex2(m - top);
			m = top;
			l *= keep;
			a = make_float4(a.x * keep, a.y * keep, a.z * keep, a.w * keep);
#pragma unroll
			for (int i = 0; i < BATCH; ++i)
				if (i0 + i <= more) {
					const float f = ml[i].x == -INFINITY ? 0.f : ex2(ml[i].x - top);
					l = fmaf(ml[i].y, f, l);
					a = make_float4(fmaf(y[i].x, f, a.x), fmaf(y[i].y, f, a.y), fmaf(y[i].z, f, a.z), fmaf(y[i].w, f, a.w));
				}
		}
		const int token = (int)(at / group), head = (int)(at - (int64_t)token * group);
		const bool blind = e.len - e.fresh + token < 0;          // a row that sees nothing
		const float f = 1.f / l;
		store_four<T>(reinterpret_cast<T *>(p.out) + ((int64_t)(e.row + token) * p.heads + s.kv * group + head) * p.dim + col,
					  blind ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(a.x * f, a.y * f, a.z * f, a.w * f));
	}
}

template <typename T, int DP>
__global__ void __launch_bounds__(JN_THREADS) join_kernel(const paged_attention_t p, const PgWork work, const float *tile_scratch) {
	const bool few = blockIdx.x < PG_SLOTS;
	const int x = blockIdx.x - (few ? 0 : PG_SLOTS), slot = few ? x : x % PG_TILE_SLOTS;
	PgStart s;
	const int more = cut(work, few ? 0 : 1, slot, s);      // (the plan was complete before the attention kernels could start this one)
	pdl_wait();
	pdl_trigger();
	if (more == 0) return;
	if (few) join<T, DP>(p, 0, slot, 0, reinterpret_cast<const float *>(p.scratch), s, more);
	else if (DP <= 128) join<T, DP>(p, 1, slot, x / PG_TILE_SLOTS * JN_ROWS, tile_scratch, s, more);
}

template <typename T>
int launch(const paged_attention_t &p, const float *tile_scratch, cudaStream_t stream) {
	const PgWork work = pg_work(const_cast<int32_t *>(p.work), p.requests, p.rows, p.heads, p.kv_heads);
	const dim3 grid(PG_SLOTS + (tile_scratch ? PG_TILE_SLOTS * (PG_TILE / JN_ROWS) : 0));
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
