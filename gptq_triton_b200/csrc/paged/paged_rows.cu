// Attention of few new tokens over a cache in pages.
#include "paged.cuh"

namespace gptq {

namespace {

// ---- fp16 and bf16 ------------------------------------------------------------------------------------------------------------
// Keys and values stream past up to 16 rows (new tokens times the query heads of a key head), which are the M of the MMAs whether or
// not all of them are in use: S = Q K^T, weights, O += P V, fp32 sums, maximum and sum per row kept while the keys pass.  Bound by HBM: the
// MMAs take a quarter of the time that the keys take from memory.
// A warp is a slot of the work list: it copies 16 keys and their values at a time for itself (cp.async, a ring of its own) and meets no
// other warp, so that there is no barrier, the copies run ahead over the ends of jobs, and many short jobs do not wait for one another.
// (Four warps that shared a job and joined their results in shared memory took 86 us for 48 requests of 1 to 12 000 keys: some slots
// had twenty jobs of a block each.)  Cut jobs leave numerator, maximum and sum of the rows in use, which join_kernel adds up.
constexpr int RW_THREADS = 128, RW_WARPS = 4;

template <int DP> struct RowsShape {
	static constexpr int UNITS = DP / 8;                            // 16-byte units of a row
	static constexpr int HALF = PG_KEYS * DP * 2;                   // bytes of the keys of a block, and of their values
	static constexpr int STAGES = DP == 64 ? 6 : 3;
	static constexpr int SMEM = RW_WARPS * STAGES * 2 * HALF;
};

struct Walk {                          // a block of a slot's jobs
	int entry, kv, block;
	PgEntry e;
	__device__ __forceinline__ bool start(const PgStart &s, const PgStart &end) {
		entry = s.entry;
		kv = s.kv;
		block = s.block;
		if (entry < 0 || (end.in_job(entry, kv) && end.block <= block)) return false;
		e = s.job;
		return true;
	}
	__device__ __forceinline__ bool step(const PgStart &end, const PgEntry *entries, int entry_count, int kv_heads) {          // false: no block is left
		if (++block == e.blocks) {
			block = 0;
			if (++kv == kv_heads) {
				kv = 0;
				if (++entry == entry_count) return false;
				e = read_entry(entries + entry);
			}
		}
		return !(end.in_job(entry, kv) ? block >= end.block : block == 0 && end.before(entry, kv));
	}
};

// EVEN: pages of a multiple of 16 rows, so that the keys of a block lie in one page, one behind the other
template <typename T, int DP, bool EVEN>
__global__ void __launch_bounds__(RW_THREADS, DP <= 128 ? 2 : 1) rows_kernel(const paged_attention_t p, const PgWork work, int beside) {
	using S = RowsShape<DP>;
	extern __shared__ __align__(128) unsigned char rw_smem[];
	const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gid = lane >> 2, tig = lane & 3;
	constexpr float LIFT = std::is_same<T, __half>::value ? 7.f : 0.f;          // fp16 weights up to 2^15: small ones stay above its subnormal range
	// Beside the tile kernel this one needs nothing of it and runs as soon as SMs are free: what came before the tile kernel is complete
	// when that triggers, and the wait is at the end, so that whoever waits for this kernel waits for both.
	if (!beside) pdl_wait();
	pdl_trigger();
	const int slot = blockIdx.x * RW_WARPS + warp;
	const PgEntry *entries = work.entries[0];
	const int entry_count = read_list(work.list).entries;
	const PgStart begin = read_start(work.starts[0] + slot), end = read_start(work.starts[0] + slot + 1);
	Walk at;
	if (!at.start(begin, end)) {
		if (beside) pdl_wait();
		return;
	}
	Walk ahead = at;                                     // what is copied next
	const int group = p.heads / p.kv_heads;
	const uint32_t ring = smem_u32(rw_smem) + warp * S::STAGES * 2 * S::HALF;
	const float to_base2 = p.scale * PG_LOG2E;
	const int units = p.dim / 8;
	int bad = 0;

	bool more = true;
	int next_id = -1, next_row = 0;                      // page (-1: no key there) and row in it: of the block (EVEN), of key (lane & 15) of it
	auto look_up = [&]() {
		const int key = ahead.block * PG_KEYS + (EVEN ? 0 : lane & 15);
		next_id = -1;
		next_row = 0;
		if (key < ahead.e.seen) {
			const int c = key / p.page;
			next_row = key - c * p.page;
			next_id = c < p.table_width ? max(__ldcg(p.table + (int64_t)ahead.e.request * p.table_ld + c), -1) : -1;
			if (next_id < 0) next_id = -2;                 // a key without a page
		}
	};
	auto copy = [&](int stage) {
		const bool there = next_id >= 0 && next_id < p.pages;
		if (next_id != -1 && !there) bad = PAGED_BAD_INDEX;
		const uint32_t dst = ring + stage * 2 * S::HALF;
		constexpr int LANES = S::UNITS < 32 ? S::UNITS : 32, ROWS = 32 / LANES;      // a row is 16 bytes times LANES lanes
		const int unit = lane % LANES, sub = lane / LANES;
		if (EVEN) {
			const int rows = there ? min(PG_KEYS, ahead.e.seen - ahead.block * PG_KEYS) : 0;
			const int64_t first = (int64_t)next_row * p.dim + unit * 8;
			const T *k = reinterpret_cast<const T *>(p.k_cache), *v = reinterpret_cast<const T *>(p.v_cache);
			if (there) {
				k += next_id * p.k_page + ahead.kv * p.k_kv + first;
				v += next_id * p.v_page + ahead.kv * p.v_kv + first;
			}
			const uint32_t base = dst + sub * DP * 2 + ((unit ^ sub) << 4);          // (ROWS divides 8: row r + sub is swizzled by r ^ sub)
			if (rows == PG_KEYS && units == S::UNITS) {
#pragma unroll
				for (int r = 0; r < PG_KEYS; r += ROWS) {
					const uint32_t to = (base ^ ((r & 7) << 4)) + r * DP * 2;
					cp_async16(to, k + sub * DP + r * DP);
					cp_async16(to + S::HALF, v + sub * DP + r * DP);
				}
			} else
#pragma unroll
			for (int r = 0; r < PG_KEYS; r += ROWS) {
				const int row = r + sub;
				const bool real = row < rows && unit < units;
				const uint32_t to = dst + row * DP * 2 + ((unit ^ (row & 7)) << 4);
				const int64_t from = real ? (int64_t)row * p.dim : 0;
				cp_async16_or_zero(to, real ? k + from : reinterpret_cast<const T *>(p.k_cache), real ? 16 : 0);
				cp_async16_or_zero(to + S::HALF, real ? v + from : reinterpret_cast<const T *>(p.v_cache), real ? 16 : 0);
			}
		} else {
			// The lower half of the warp knows where the 16 keys are, the upper half where their values are.
			const T *cache = reinterpret_cast<const T *>(lane < 16 ? p.k_cache : p.v_cache);
			const T *src = there ? cache + next_id * (lane < 16 ? p.k_page : p.v_page) + ahead.kv * (lane < 16 ? p.k_kv : p.v_kv) + (int64_t)next_row * p.dim : cache;
			const unsigned long long mine = reinterpret_cast<unsigned long long>(src) | (there ? 1ull : 0ull);          // (addresses are even)
#pragma unroll
			for (int r = 0; r < 2 * PG_KEYS; r += ROWS) {
				const int row = r + sub;                   // 16 ..: values
				const unsigned long long theirs = __shfl_sync(0xffffffffu, mine, row);
				const bool real = (theirs & 1ull) && unit < units;
				cp_async16_or_zero(dst + row * DP * 2 + ((unit ^ (row & 7)) << 4), reinterpret_cast<const unsigned char *>(theirs & ~1ull) + (real ? unit * 16 : 0), real ? 16 : 0);
			}
		}
		more = ahead.step(end, entries, entry_count, p.kv_heads);
		if (more) look_up();
	};
	look_up();
#pragma unroll
	for (int s = 0; s < S::STAGES; ++s) {
		if (more) copy(s);
		cp_async_commit();
	}

	uint32_t q[DP / 16][4];
	float o[DP / 8][4], mx[2], sum[2];
	int seen[2];                                          // keys that rows gid and gid + 8 see
	int least = 0, count = 0;                             // ... and that the row with the fewest of them sees; rows in use
	bool fresh = true;
	int first_block = at.block;
	for (int stage = 0;;) {
		if (fresh) {                                      // a new job: its queries
			fresh = false;
			first_block = at.block;
			count = min(PG_ROWS, at.e.fresh * group - at.e.tile * PG_ROWS);
			least = at.e.len - at.e.fresh + at.e.tile * PG_ROWS / group + 1;
#pragma unroll
			for (int i = 0; i < 2; ++i) {
				const int row = gid + 8 * i, token = (at.e.tile * PG_ROWS + row) / group, head = at.kv * group + (at.e.tile * PG_ROWS + row) - token * group;
				seen[i] = row < count ? at.e.len - at.e.fresh + token + 1 : 0;
				const T *src = reinterpret_cast<const T *>(p.q) + (int64_t)(at.e.row + token) * p.q_row + (int64_t)head * p.q_head;
#pragma unroll
				for (int k = 0; k < DP / 16; ++k) {
					const int d = 16 * k + 2 * tig;
					q[k][i] = row < count && d < p.dim ? __ldcg(reinterpret_cast<const uint32_t *>(src + d)) : 0u;
					q[k][2 + i] = row < count && d + 8 < p.dim ? __ldcg(reinterpret_cast<const uint32_t *>(src + d + 8)) : 0u;
				}
				mx[i] = -INFINITY;
				sum[i] = 0.f;
			}
#pragma unroll
			for (int i = 0; i < DP / 8; ++i)
#pragma unroll
				for (int j = 0; j < 4; ++j) o[i][j] = 0.f;
		}
		cp_async_wait<S::STAGES - 1>();
		__syncwarp();
		const uint32_t sk = ring + (uint32_t)stage * 2 * S::HALF, sv = sk + S::HALF;
		const int key0 = at.block * PG_KEYS;
		{
			// two chains of MMAs per eight keys
			float s[2][4] = {}, s2[2][4] = {};
			const int kr = (lane >> 4) * 8 + (lane & 7), ku = (lane >> 3) & 1;
			const uint32_t ka = sk + kr * DP * 2 + ((ku ^ (kr & 7)) << 4);          // (16-byte units are swizzled by their row: unit 2 k + ku lies at this address ^ 32 k)
#pragma unroll
			for (int k = 0; k < DP / 16; k += 2) {
				uint32_t b[4], c[4];
				ldsm4(b, ka ^ (32 * k));
				ldsm4(c, ka ^ (32 * k + 32));
				mma16<T>(s[0], q[k], b[0], b[1]);
				mma16<T>(s[1], q[k], b[2], b[3]);
				mma16<T>(s2[0], q[k + 1], c[0], c[1]);
				mma16<T>(s2[1], q[k + 1], c[2], c[3]);
			}
			const bool edge = key0 + PG_KEYS > least;
			float top[2];
#pragma unroll
			for (int i = 0; i < 2; ++i) {
#pragma unroll
				for (int t = 0; t < 2; ++t)
#pragma unroll
					for (int j = 0; j < 2; ++j) {
						float &x = s[t][2 * i + j];
						x = (x + s2[t][2 * i + j]) * to_base2;
						if (edge && key0 + 8 * t + 2 * tig + j >= seen[i]) x = -INFINITY;
					}
				float m = fmaxf(fmaxf(s[0][2 * i], s[0][2 * i + 1]), fmaxf(s[1][2 * i], s[1][2 * i + 1]));
				m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
				top[i] = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
			}
			// the reference point of a row follows its maximum only when that has grown by more than 2^8
			if (__any_sync(0xffffffffu, top[0] > mx[0] + 8.f || top[1] > mx[1] + 8.f)) {
#pragma unroll
				for (int i = 0; i < 2; ++i) {
					const float next = fmaxf(mx[i], top[i]), keep = mx[i] == -INFINITY ? 0.f : ex2(mx[i] - next);
					mx[i] = next;
					sum[i] *= keep;
#pragma unroll
					for (int t = 0; t < DP / 8; ++t) {
						o[t][2 * i] *= keep;
						o[t][2 * i + 1] *= keep;
					}
				}
			}
			uint32_t w[4];
#pragma unroll
			for (int i = 0; i < 2; ++i) {
				const float ref = mx[i] == -INFINITY ? 0.f : mx[i] - LIFT;
				const float a = ex2(s[0][2 * i] - ref), b = ex2(s[0][2 * i + 1] - ref), c = ex2(s[1][2 * i] - ref), d = ex2(s[1][2 * i + 1] - ref);
				sum[i] += (a + b) + (c + d);
				// weights in the type of the values: what the MMA multiplies; their sum is taken before the rounding
				w[i] = pack2<T>(a, b);
				w[2 + i] = pack2<T>(c, d);
			}
			const int vr = ((lane >> 3) & 1) * 8 + (lane & 7), vu = lane >> 4;
			const uint32_t va = sv + vr * DP * 2 + ((vu ^ (vr & 7)) << 4);
#pragma unroll
			for (int t = 0; t < DP / 16; ++t) {
				uint32_t b[4];
				ldsm4_t(b, va ^ (32 * t));
				mma16<T>(o[2 * t], w, b[0], b[1]);
				mma16<T>(o[2 * t + 1], w, b[2], b[3]);
			}
		}
		__syncwarp();
		if (more) copy(stage);
		cp_async_commit();
		stage = stage + 1 == S::STAGES ? 0 : stage + 1;

		const int blocks = at.e.blocks, last = at.block, entry_row = at.e.row, before = at.e.len - at.e.fresh, tile = at.e.tile, kv = at.kv;
		const bool tile_ends = last + 1 == blocks, go_on = at.step(end, entries, entry_count, p.kv_heads);
		if (!tile_ends && go_on) continue;
		// ---- the job, or this slot's part of it, is done ----
		fresh = true;
		const bool whole = first_block == 0 && tile_ends;
		float *part = reinterpret_cast<float *>(p.scratch) + (int64_t)(2 * slot + (first_block == 0)) * PG_ROWS * (DP + 2);
#pragma unroll
		for (int i = 0; i < 2; ++i) {
			const int row = gid + 8 * i;
			sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 1);
			sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 2);
			if (row >= count) continue;
			if (whole) {
				const int token = (tile * PG_ROWS + row) / group, head = kv * group + tile * PG_ROWS + row - token * group;
				const bool blind = before + token < 0;       // a row that sees nothing
				const float f = 1.f / sum[i];
				T *dst = reinterpret_cast<T *>(p.out) + ((int64_t)(entry_row + token) * p.heads + head) * p.dim + 2 * tig;
#pragma unroll
				for (int t = 0; t < DP / 8; ++t)
					if (8 * t < p.dim) *reinterpret_cast<uint32_t *>(dst + 8 * t) = blind ? 0u : pack2<T>(o[t][2 * i] * f, o[t][2 * i + 1] * f);
			} else {
				if (tig == 0) __stcg(reinterpret_cast<float2 *>(part + PG_ROWS * DP) + row, make_float2(mx[i], sum[i]));
#pragma unroll
				for (int t = 0; t < DP / 8; ++t) __stcg(reinterpret_cast<float2 *>(part + row * DP + 8 * t + 2 * tig), make_float2(o[t][2 * i], o[t][2 * i + 1]));
			}
		}
		if (!go_on) break;
	}
	if (bad) atomicOr(p.status, bad);
	if (beside) pdl_wait();
}

// ---- fp32 ---------------------------------------------------------------------------------------------------------------------
// The same walk without reduced-precision products.  Scores: a lane takes one of the 16 keys and half of the head's entries, the queries come
// from shared memory; products with the values: a lane takes four entries of the head (or of every second key, for heads of 64), weights
// come by shuffles.  ROWS: rows of a tile that the code provides for.
template <int DP, int ROWS> struct FloatShape {
	static constexpr int UNITS = DP / 4;
	static constexpr int HALF = PG_KEYS * DP * 4;
	static constexpr int STAGES = DP == 256 ? 1 : DP == 64 && ROWS > 4 ? 2 : 3;
	static constexpr int Q_ROW = DP + 8;                             // the halves of a query 4 floats further apart: other banks
	static constexpr int RING = RW_WARPS * STAGES * 2 * HALF;
	static constexpr int SMEM = RING + RW_WARPS * ROWS * Q_ROW * 4;
};

template <int DP, int ROWS, bool EVEN>
__global__ void __launch_bounds__(RW_THREADS, DP == 64 ? 2 : 1) rows_f32_kernel(const paged_attention_t p, const PgWork work) {
	using S = FloatShape<DP, ROWS>;
	extern __shared__ __align__(128) unsigned char rf_smem[];
	const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
	pdl_wait();
	pdl_trigger();
	const int slot = blockIdx.x * RW_WARPS + warp;
	const PgEntry *entries = work.entries[0];
	const int entry_count = read_list(work.list).entries;
	const PgStart begin = read_start(work.starts[0] + slot), end = read_start(work.starts[0] + slot + 1);
	Walk at;
	if (!at.start(begin, end)) return;
	Walk ahead = at;
	const int group = p.heads / p.kv_heads;
	const uint32_t ring = smem_u32(rf_smem) + warp * S::STAGES * 2 * S::HALF;
	const float *ring_f = reinterpret_cast<const float *>(rf_smem + warp * S::STAGES * 2 * S::HALF);
	float *s_q = reinterpret_cast<float *>(rf_smem + S::RING) + warp * ROWS * S::Q_ROW;
	const float to_base2 = p.scale * PG_LOG2E;
	int bad = 0, next_id = -1, next_row = 0;
	bool more = true;
	auto look_up = [&]() {
		const int key = ahead.block * PG_KEYS + (EVEN ? 0 : lane & 15);
		next_id = -1;
		next_row = 0;
		if (key < ahead.e.seen) {
			const int c = key / p.page;
			next_row = key - c * p.page;
			next_id = c < p.table_width ? max(__ldcg(p.table + (int64_t)ahead.e.request * p.table_ld + c), -1) : -1;
			if (next_id < 0) next_id = -2;                 // a key without a page
		}
	};
	auto copy = [&](int stage) {
		const bool there = next_id >= 0 && next_id < p.pages;
		if (next_id != -1 && !there) bad = PAGED_BAD_INDEX;
		const int left = ahead.e.seen - ahead.block * PG_KEYS;
		// place of this lane's key (of the first one: EVEN) and of its values
		const float *k = reinterpret_cast<const float *>(p.k_cache), *v = reinterpret_cast<const float *>(p.v_cache);
		if (there) {
			k += next_id * p.k_page + ahead.kv * p.k_kv + (int64_t)next_row * p.dim;
			v += next_id * p.v_page + ahead.kv * p.v_kv + (int64_t)next_row * p.dim;
		}
		const uint32_t dst = ring + stage * 2 * S::HALF;
#pragma unroll 4
		for (int x = lane; x < PG_KEYS * S::UNITS; x += 32) {
			const int row = x / S::UNITS, unit = x % S::UNITS;
			unsigned long long kp = reinterpret_cast<unsigned long long>(k), vp = reinterpret_cast<unsigned long long>(v);
			bool real = there;
			if (EVEN) {
				kp += (unsigned long long)row * p.dim * 4;
				vp += (unsigned long long)row * p.dim * 4;
				real = real && row < left;
			} else {
				kp = __shfl_sync(0xffffffffu, kp, row);
				vp = __shfl_sync(0xffffffffu, vp, row);
				real = __shfl_sync(0xffffffffu, (int)there, row);
			}
			real = real && 4 * unit < p.dim;
			const uint32_t to = dst + row * DP * 4 + ((unit ^ (row & 7)) << 4);
			cp_async16_or_zero(to, real ? reinterpret_cast<const void *>(kp + unit * 16) : p.k_cache, real ? 16 : 0);
			cp_async16_or_zero(to + S::HALF, real ? reinterpret_cast<const void *>(vp + unit * 16) : p.v_cache, real ? 16 : 0);
		}
		more = ahead.step(end, entries, entry_count, p.kv_heads);
		if (more) look_up();
	};
	look_up();
#pragma unroll
	for (int s = 0; s < S::STAGES; ++s) {
		if (more) copy(s);
		cp_async_commit();
	}

	constexpr int V4 = DP >= 128 ? DP / 128 : 1, SPLIT = DP >= 128 ? 1 : 2;          // float4 of a lane, lanes that share entries
	float4 o[ROWS][V4];
	float mx[ROWS], sum[ROWS];
	int count = 0, least = 0, seen = 0, first_block = 0;      // seen: keys that row (lane & 15) sees
	bool fresh = true;
	const int key = lane & 15, side = lane >> 4;
	for (int stage = 0;;) {
		if (fresh) {
			fresh = false;
			first_block = at.block;
			count = min(PG_ROWS, at.e.fresh * group - at.e.tile * PG_ROWS);
			least = at.e.len - at.e.fresh + at.e.tile * PG_ROWS / group + 1;
			const int mine = at.e.tile * PG_ROWS + key;
			seen = key < count ? at.e.len - at.e.fresh + mine / group + 1 : 0;
			__syncwarp();
			for (int x = lane; x < ROWS * S::UNITS; x += 32) {
				const int row = x / S::UNITS, d = x % S::UNITS * 4, token = (at.e.tile * PG_ROWS + row) / group, head = at.kv * group + (at.e.tile * PG_ROWS + row) - token * group;
				float4 q = make_float4(0.f, 0.f, 0.f, 0.f);
				if (row < count && d < p.dim) q = __ldcg(reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(p.q) + (int64_t)(at.e.row + token) * p.q_row + (int64_t)head * p.q_head + d));
				*reinterpret_cast<float4 *>(s_q + row * S::Q_ROW + d + (d >= DP / 2 ? 4 : 0)) = q;
			}
			__syncwarp();
#pragma unroll
			for (int r = 0; r < ROWS; ++r) {
				mx[r] = -INFINITY;
				sum[r] = 0.f;
#pragma unroll
				for (int i = 0; i < V4; ++i) o[r][i] = make_float4(0.f, 0.f, 0.f, 0.f);
			}
		}
		cp_async_wait<S::STAGES - 1>();
		__syncwarp();
		const float *sk = ring_f + stage * 2 * (S::HALF / 4), *sv = sk + S::HALF / 4;
		const int key0 = at.block * PG_KEYS;
		float w[ROWS];
#pragma unroll
		for (int r = 0; r < ROWS; ++r) w[r] = 0.f;
		// (rows in groups of four, whose chains run side by side)
#pragma unroll 4
		for (int u = 0; u < DP / 8; ++u) {
			const float4 k = *reinterpret_cast<const float4 *>(sk + key * DP + (((side * (DP / 8) + u) ^ (key & 7)) << 2));
#pragma unroll
			for (int g = 0; g < ROWS; g += 4)
				if (g < count) {
#pragma unroll
					for (int r = g; r < g + 4; ++r) {
						const float4 q = *reinterpret_cast<const float4 *>(s_q + r * S::Q_ROW + side * (DP / 2 + 4) + 4 * u);
						w[r] = fmaf(q.x, k.x, fmaf(q.y, k.y, fmaf(q.z, k.z, fmaf(q.w, k.w, w[r]))));
					}
				}
		}
		const bool edge = key0 + PG_KEYS > least;
#pragma unroll
		for (int g = 0; g < ROWS; g += 4)
			if (g < count) {
				float top[4];
				bool grown = false;
#pragma unroll
				for (int i = 0; i < 4; ++i) {
					w[g + i] = (w[g + i] + __shfl_xor_sync(0xffffffffu, w[g + i], 16)) * to_base2;
					if (edge && key0 + key >= __shfl_sync(0xffffffffu, seen, g + i)) w[g + i] = -INFINITY;
					top[i] = w[g + i];
				}
#pragma unroll
				for (int d = 8; d > 0; d >>= 1)
#pragma unroll
					for (int i = 0; i < 4; ++i) top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], d));
#pragma unroll
				for (int i = 0; i < 4; ++i) grown = grown || top[i] > mx[g + i];
				if (grown) {                                   // (the same in all lanes)
#pragma unroll
					for (int i = 0; i < 4; ++i) {
						const float next = fmaxf(mx[g + i], top[i]), keep = mx[g + i] == -INFINITY ? 0.f : ex2(mx[g + i] - next);
						mx[g + i] = next;
						sum[g + i] *= keep;
#pragma unroll
						for (int x = 0; x < V4; ++x) o[g + i][x] = make_float4(o[g + i][x].x * keep, o[g + i][x].y * keep, o[g + i][x].z * keep, o[g + i][x].w * keep);
					}
				}
#pragma unroll
				for (int i = 0; i < 4; ++i) {
					w[g + i] = ex2(w[g + i] - (mx[g + i] == -INFINITY ? 0.f : mx[g + i]));
					sum[g + i] += w[g + i];
				}
			}
#pragma unroll 4
		for (int j = 0; j < PG_KEYS / SPLIT; ++j) {
			const int from = j * SPLIT + (SPLIT == 2 ? side : 0);
			float4 v[V4];
#pragma unroll
			for (int i = 0; i < V4; ++i) v[i] = *reinterpret_cast<const float4 *>(sv + from * DP + (((lane % S::UNITS + 32 * i) ^ (from & 7)) << 2));
#pragma unroll
			for (int g = 0; g < ROWS; g += 4)
				if (g < count) {
#pragma unroll
					for (int r = g; r < g + 4; ++r) {
						const float x = __shfl_sync(0xffffffffu, w[r], from);
#pragma unroll
						for (int i = 0; i < V4; ++i) o[r][i] = make_float4(fmaf(x, v[i].x, o[r][i].x), fmaf(x, v[i].y, o[r][i].y), fmaf(x, v[i].z, o[r][i].z), fmaf(x, v[i].w, o[r][i].w));
					}
				}
		}
		__syncwarp();
		if (more) copy(stage);
		cp_async_commit();
		stage = stage + 1 == S::STAGES ? 0 : stage + 1;

		const int blocks = at.e.blocks, last = at.block, entry_row = at.e.row, before = at.e.len - at.e.fresh, tile = at.e.tile, kv = at.kv;
		const bool tile_ends = last + 1 == blocks, go_on = at.step(end, entries, entry_count, p.kv_heads);
		if (!tile_ends && go_on) continue;
		fresh = true;
		const bool whole = first_block == 0 && tile_ends;
		float *part = reinterpret_cast<float *>(p.scratch) + (int64_t)(2 * slot + (first_block == 0)) * PG_ROWS * (DP + 2);
#pragma unroll
		for (int r = 0; r < ROWS; ++r)
			if (r < count) {
#pragma unroll
				for (int d = 8; d > 0; d >>= 1) sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], d);
				const int token = (tile * PG_ROWS + r) / group, head = kv * group + tile * PG_ROWS + r - token * group;
				const float f = !whole ? 1.f : before + token < 0 ? 0.f : 1.f / sum[r];
				if (!whole && lane == 0) __stcg(reinterpret_cast<float2 *>(part + PG_ROWS * DP) + r, make_float2(mx[r], sum[r]));
#pragma unroll
				for (int i = 0; i < V4; ++i) {
					float4 a = o[r][i];
					if (SPLIT == 2) {
						a.x += __shfl_xor_sync(0xffffffffu, a.x, 16);
						a.y += __shfl_xor_sync(0xffffffffu, a.y, 16);
						a.z += __shfl_xor_sync(0xffffffffu, a.z, 16);
						a.w += __shfl_xor_sync(0xffffffffu, a.w, 16);
					}
					const int d = (lane % S::UNITS + 32 * i) * 4;
					if (SPLIT == 2 && side) continue;
					const float4 y = make_float4(a.x * f, a.y * f, a.z * f, a.w * f);
					if (!whole) __stcg(reinterpret_cast<float4 *>(part + r * DP + d), y);
					else if (d < p.dim) *reinterpret_cast<float4 *>(reinterpret_cast<float *>(p.out) + ((int64_t)(entry_row + token) * p.heads + head) * p.dim + d) = y;
				}
			}
		if (!go_on) break;
	}
	if (bad) atomicOr(p.status, bad);
}

int rows_dp(int dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }

template <typename T, int DP>
int rows_launch(const paged_attention_t &p, const PgWork &work, bool beside, cudaStream_t stream) {
	constexpr int smem = RowsShape<DP>::SMEM;
	static_assert(smem + 1024 <= (DP <= 128 ? 114 : 228) * 1024 && smem <= 227 * 1024, "shared memory of an SM, 1 KB of it reserved per CTA");
	const dim3 grid(PG_SLOTS / RW_WARPS);
	if (p.page % PG_KEYS == 0) return pg_launch(rows_kernel<T, DP, true>, grid, RW_THREADS, smem, stream, p, work, (int)beside);
	return pg_launch(rows_kernel<T, DP, false>, grid, RW_THREADS, smem, stream, p, work, (int)beside);
}
template <typename T>
int rows_launch_dim(const paged_attention_t &p, const PgWork &work, bool beside, cudaStream_t stream) {
	switch (rows_dp(p.dim)) {
		case 64: return rows_launch<T, 64>(p, work, beside, stream);
		case 128: return rows_launch<T, 128>(p, work, beside, stream);
		default: return rows_launch<T, 256>(p, work, beside, stream);
	}
}

template <int DP, int ROWS>
int rows_f32_launch_rows(const paged_attention_t &p, const PgWork &work, cudaStream_t stream) {
	constexpr int smem = FloatShape<DP, ROWS>::SMEM;
	static_assert(smem + 1024 <= (DP == 64 ? 114 : 228) * 1024 && smem <= 227 * 1024, "shared memory of an SM, 1 KB of it reserved per CTA");
	if (p.page % PG_KEYS == 0) return pg_launch(rows_f32_kernel<DP, ROWS, true>, dim3(PG_SLOTS / RW_WARPS), RW_THREADS, smem, stream, p, work);
	return pg_launch(rows_f32_kernel<DP, ROWS, false>, dim3(PG_SLOTS / RW_WARPS), RW_THREADS, smem, stream, p, work);
}
template <int DP>
int rows_f32_launch(const paged_attention_t &p, const PgWork &work, cudaStream_t stream) {
	const bool few = (int64_t)p.max_fresh * (p.heads / p.kv_heads) <= 4;
	return few ? rows_f32_launch_rows<DP, 4>(p, work, stream) : rows_f32_launch_rows<DP, PG_ROWS>(p, work, stream);
}

}   // namespace

int64_t pg_rows_scratch(const paged_attention_t &p) { return (int64_t)2 * PG_SLOTS * PG_ROWS * (rows_dp(p.dim) + 2) * 4; }

int pg_rows_launch(const paged_attention_t &p, int dtype, bool beside, cudaStream_t stream) {
	const PgWork work = pg_work(const_cast<int32_t *>(p.work), p.requests, p.rows, p.heads, p.kv_heads);
	if (dtype == PG_F32) return p.dim <= 64 ? rows_f32_launch<64>(p, work, stream) : p.dim <= 128 ? rows_f32_launch<128>(p, work, stream) : rows_f32_launch<256>(p, work, stream);
	return dtype == PG_BF16 ? rows_launch_dim<bf16>(p, work, beside, stream) : rows_launch_dim<__half>(p, work, beside, stream);
}

}   // namespace gptq
