// Joins the partial results of tiles whose keys are spread over several slots of an attention kernel: numerators, maxima (base 2) and sums
// of a row.
//   m = max m_i,  l = sum l_i 2^(m_i - m),  out = (sum a_i 2^(m_i - m)) / l
// The order of the additions is fixed by the sizes alone, so that results repeat bit by bit: a group of lanes (all 32; 16 for heads of up to 64)
// takes every n-th partial result in the order of the slots, the second half of a warp is added to the first, warp 1, 2 .. to warp 0.
#include "paged.cuh"

namespace gptq {

namespace {

constexpr int JN_THREADS = 256, JN_WARPS = JN_THREADS / 32, JN_CTAS = 296;

template <typename T> __device__ __forceinline__ void store_four(T *dst, float4 v) { *reinterpret_cast<uint2 *>(dst) = make_uint2(pack2<T>(v.x, v.y), pack2<T>(v.z, v.w)); }
template <> __device__ __forceinline__ void store_four<float>(float *dst, float4 v) { *reinterpret_cast<float4 *>(dst) = v; }

struct Sum {                           // of partial results, for four columns of a row
	float m, l;
	float4 a;
};
__device__ __forceinline__ void fold(Sum &s, float m, float l, float4 a) {
	const float top = fmaxf(s.m, m), keep = s.m == -INFINITY ? 0.f : ex2(s.m - top), f = m == -INFINITY ? 0.f : ex2(m - top);
	s.m = top;
	s.l = fmaf(l, f, s.l * keep);
	s.a = make_float4(fmaf(a.x, f, s.a.x * keep), fmaf(a.y, f, s.a.y * keep), fmaf(a.z, f, s.a.z * keep), fmaf(a.w, f, s.a.w * keep));
}

struct Cut {                           // a job that is cut: the slot in which it begins, where it goes on, how many further slots it runs through
	PgStart s;
	int slot, more;
};
__device__ __forceinline__ Cut read_cut(const PgWork &work, int kind, const PgList &list, int i) {
	Cut c;
	c.slot = __ldcg(work.cuts[kind] + (i < list.cuts[0] ? i : (kind ? PG_TILE_SLOTS : PG_SLOTS) + i - list.cuts[0]));
	c.s = read_start(work.starts[kind] + c.slot + 1);
	c.more = (int)((c.s.job.blocks - c.s.block + list.per - 1) / list.per);
	return c;
}

// A warp adds up ROWS rows from `row0` on of the partial results first, first + step ..; lanes take four columns each, and where a row has
// fewer than 128 every second partial result.  The sum of all is in the first DP / 4 lanes; their partners, which fold the same the other way round,
// have another rounding of it.
template <int DP, int ROWS>
__device__ __forceinline__ void add_up(const Cut &c, int tile_rows, int row0, int rows, const float *scratch, int col0, int first, int step, Sum (&sum)[ROWS]) {
	constexpr int LANES = DP / 4 < 32 ? DP / 4 : 32, SHARE = 32 / LANES, BATCH = ROWS > 1 ? 2 : 8;
	const int lane = threadIdx.x & 31, col = col0 + lane % LANES * 4;
	auto part = [&](int i) { return scratch + (int64_t)(i == 0 ? 2 * c.slot + 1 : 2 * (c.slot + i)) * tile_rows * (DP + 2); };
	for (int i0 = first * SHARE + lane / LANES; i0 <= c.more; i0 += BATCH * step * SHARE) {
		float2 ml[BATCH][ROWS];
		float4 y[BATCH][ROWS];
#pragma unroll
		for (int i = 0; i < BATCH; ++i)
#pragma unroll
			for (int r = 0; r < ROWS; ++r)
				if (i0 + i * step * SHARE <= c.more && r < rows) {          // (all asked for before the first is used)
					const float *q = part(i0 + i * step * SHARE);
					ml[i][r] = __ldcg(reinterpret_cast<const float2 *>(q + (int64_t)tile_rows * DP) + row0 + r);
					y[i][r] = __ldcg(reinterpret_cast<const float4 *>(q + (int64_t)(row0 + r) * DP + col));
				}
#pragma unroll
		for (int i = 0; i < BATCH; ++i)
#pragma unroll
			for (int r = 0; r < ROWS; ++r)
				if (i0 + i * step * SHARE <= c.more && r < rows) fold(sum[r], ml[i][r].x, ml[i][r].y, y[i][r]);
	}
#pragma unroll
	for (int d = LANES; d < 32; d *= 2)
#pragma unroll
		for (int r = 0; r < ROWS; ++r) {
			const Sum &s = sum[r];
			const float m = __shfl_xor_sync(0xffffffffu, s.m, d), l = __shfl_xor_sync(0xffffffffu, s.l, d);
			const float4 a = make_float4(__shfl_xor_sync(0xffffffffu, s.a.x, d), __shfl_xor_sync(0xffffffffu, s.a.y, d), __shfl_xor_sync(0xffffffffu, s.a.z, d), __shfl_xor_sync(0xffffffffu, s.a.w, d));
			fold(sum[r], m, l, a);
		}
}

template <typename T, int DP>
__device__ __forceinline__ void write(const paged_attention_t &p, const Cut &c, int tile_rows, int row, int col, const Sum &sum) {
	const int group = p.heads / p.kv_heads;
	const PgEntry &e = c.s.job;
	const int64_t at = (int64_t)e.tile * tile_rows + row;
	const int token = (int)(at / group), head = (int)(at - (int64_t)token * group);
	const bool blind = e.len - e.fresh + token < 0;          // a row that sees nothing
	const float f = 1.f / sum.l;
	if (col < p.dim && (threadIdx.x & 31) < DP / 4)          // (the lanes that hold the sum)
		store_four<T>(reinterpret_cast<T *>(p.out) + ((int64_t)(e.row + token) * p.heads + c.s.kv * group + head) * p.dim + col,
					  blind ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(sum.a.x * f, sum.a.y * f, sum.a.z * f, sum.a.w * f));
}
__device__ __forceinline__ int rows_of(const paged_attention_t &p, const Cut &c, int tile_rows) {
	return (int)min((int64_t)tile_rows, (int64_t)c.s.job.fresh * (p.heads / p.kv_heads) - (int64_t)c.s.job.tile * tile_rows);
}

// A unit is a row of a cut job of the kernel for few rows (four rows of one of the tile kernel).  Where there are fewer units than CTAs
// a CTA takes one, its warps share the partial results (a job of one request may run through hundreds of slots); else a warp takes one.
// few_rows, many_rows: rows that a tile has at most.
template <typename T, int DP>
__global__ void __launch_bounds__(JN_THREADS, 2) join_kernel(const paged_attention_t p, const PgWork work, const float *tile_scratch, int few_rows, int many_rows) {
	constexpr int COLS = DP / 128 > 1 ? DP / 128 : 1;          // runs of 128 columns
	__shared__ Sum s_sum[JN_WARPS][32];
	const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, col = lane % (DP / 4 < 32 ? DP / 4 : 32) * 4;
	const PgList few = read_list(work.list);               // (the plan was complete before the attention kernels could start this one)
	PgList many = {};
	if (tile_scratch) many = read_list(work.list + 1);
	const float *scratch = reinterpret_cast<const float *>(p.scratch);
	const int jobs = few.cuts[0] + few.cuts[1], units = jobs * few_rows;
	const bool together = units <= JN_CTAS;
	int u = together ? blockIdx.x : blockIdx.x * JN_WARPS + warp;
	Cut c = {};
	if (u < units) c = read_cut(work, 0, few, u / few_rows);
	pdl_wait();
	pdl_trigger();
	while (u < units) {
		const int row = u % few_rows;
		if (row < rows_of(p, c, PG_ROWS)) {
#pragma unroll
			for (int x = 0; x < COLS; ++x) {
				Sum sum[1] = {{-INFINITY, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)}};
				add_up<DP, 1>(c, PG_ROWS, row, 1, scratch, 128 * x, together ? warp : 0, together ? JN_WARPS : 1, sum);
				if (together) {
					__syncthreads();
					s_sum[warp][lane] = sum[0];
					__syncthreads();
					if (warp == 0) {
#pragma unroll
						for (int w = 1; w < JN_WARPS; ++w) fold(sum[0], s_sum[w][lane].m, s_sum[w][lane].l, s_sum[w][lane].a);
					}
				}
				if (!together || warp == 0) write<T, DP>(p, c, PG_ROWS, row, col + 128 * x, sum[0]);
			}
		}
		u += together ? gridDim.x : gridDim.x * JN_WARPS;
		if (u < units) c = read_cut(work, 0, few, u / few_rows);
	}
	if (DP > 128 || !tile_scratch) return;
	const int warps = gridDim.x * JN_WARPS, tiles = many.cuts[0] + many.cuts[1], first = blockIdx.x * JN_WARPS + warp;
	auto go = [&](auto rows_each) {
		constexpr int ROWS = decltype(rows_each)::value;
		const int groups = (many_rows + ROWS - 1) / ROWS, sets = tiles * groups;
		for (int x = first; x < sets; x += warps) {
			const int row0 = x % groups * ROWS;
			const Cut d = read_cut(work, 1, many, x / groups);
			const int rows = rows_of(p, d, PG_TILE) - row0;
			if (rows <= 0) continue;
			Sum sum[ROWS];
#pragma unroll
			for (int r = 0; r < ROWS; ++r) sum[r] = {-INFINITY, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
			add_up<DP, ROWS>(d, PG_TILE, row0, rows, tile_scratch, 0, 0, 1, sum);
#pragma unroll
			for (int r = 0; r < ROWS; ++r)
				if (r < rows) write<T, DP>(p, d, PG_TILE, row0 + r, col, sum[r]);
		}
	};
	// few jobs run through many slots each: more partial results of a row at once; many jobs: more rows
	if (tiles * many_rows <= 2 * warps) go(std::integral_constant<int, 1>());
	else go(std::integral_constant<int, 4>());
}

template <typename T>
int launch(const paged_attention_t &p, const float *tile_scratch, cudaStream_t stream) {
	const PgWork work = pg_work(const_cast<int32_t *>(p.work), p.requests, p.rows, p.heads, p.kv_heads);
	const int64_t rows = (int64_t)p.max_fresh * (p.heads / p.kv_heads);
	const int few = (int)(rows < PG_ROWS ? rows : PG_ROWS), many = (int)(rows < PG_TILE ? rows : PG_TILE);
	auto go = [&](auto kernel) { return pg_launch(kernel, dim3(JN_CTAS), JN_THREADS, 0, stream, p, work, tile_scratch, few, many); };
	return p.dim <= 64 ? go(join_kernel<T, 64>) : p.dim <= 128 ? go(join_kernel<T, 128>) : go(join_kernel<T, 256>);
}

}   // namespace

int pg_join_launch(const paged_attention_t &p, int dtype, char *tile_scratch, cudaStream_t stream) {
	const float *t = reinterpret_cast<const float *>(tile_scratch);
	return dtype == PG_BF16 ? launch<bf16>(p, t, stream) : dtype == PG_F16 ? launch<__half>(p, t, stream) : launch<float>(p, t, stream);
}

}   // namespace gptq
