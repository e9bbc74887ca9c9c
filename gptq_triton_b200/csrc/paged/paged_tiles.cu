// Attention of chunks over a cache in pages on the 5th-generation tensor cores (fp16, bf16, heads of up to 128).
//
// A tile is 256 rows (new tokens times the query heads of a key head, token-major, so that short chunks with shared key heads fill it):
// two sides of 128, whose scores and outputs take the 512 columns of tensor memory.  Per block of 128 keys and side: S = Q K^T, online
// softmax, O += P V; while the softmax warps of one side work, the tensor cores work for the other.
//   softmax warps   four per side, a thread owns a row: 128 scores from tensor memory, mask where the block crosses what the row sees,
//                   weights in the type of the values back to the columns of the scores (they are the A operand of P V there)
//   TMA warp        key and value blocks through one ring; a lane knows the page of its part of a block, so pages of 8 rows and more serve, one
//                   lane issues; pages behind what the tile sees, or that do not exist, are asked for outside the tensor and arrive as zeros
//   MMA lane        both sides in turn: P V of this block in two halves, as the weights come, Q K^T of the next
// O is rescaled only when a row's maximum has grown by more than 2^8.  fp32 sums; weights are rounded to the type of the values, their
// sum is taken before that.  Values behind the last key seen are zeroed in shared memory: a weight of zero times NaN would be NaN.
// CTAs stay for the whole launch and take whole jobs, or equal shares of all (paged_plan); cut jobs leave partial results, which
// join_kernel adds up.  Every wait is bounded.
//
// 512 tokens behind 30 000, 64 heads over 8 of 128, bf16: 459 us in a graph that runs for some milliseconds (1 107 TFLOP/s), 529 us when
// called without a pause, under the power limit (960); 2 047 tokens of 32 heads 50 and 53 us, twelve prompts of 90 to 3 000 tokens 156 and
// 167 us.  Bound by the chain of a block (scores, maximum, weights, products; 3 450 cycles for two sides that take turns, of which the tensor
// cores are busy for 58 %) and the clock under this load: without the exponentials it takes 440 us, with next to no MMAs 377, with neither
// 298.  Measured against this form (452 to 466 us then, all in short graphs): MMAs behind `lane == 0` 565, two threads per row 473, an MMA warp
// per side 505 (both sides then fall into step), scores of 64 keys in two buffers 510, a quarter of the exponentials on the FMA units 468.
#include <mutex>

#include "../tcgen05.cuh"
#include "paged.cuh"

namespace gptq {

namespace {

constexpr int TL_SIDE = 128, TL_KEYS = PG_TILE_KEYS;
constexpr int TL_CHUNK = 128 * 128;                      // bytes of 128 rows of 64 columns
constexpr int TL_THREADS = 384, TL_TMA = 8, TL_MMA = 9;          // (warps 10 and 11 complete the third warpgroup)
// registers of a thread behind setmaxnreg; what the kernel is launched with has to cover them (tiles_launch looks)
constexpr int TL_REGS_SOFTMAX = 208, TL_REGS_OTHER = 88, TL_REGS_LAUNCH = (2 * TL_REGS_SOFTMAX + TL_REGS_OTHER) / 3;
constexpr uint32_t TL_SPIN = 1u << 24;                  // polls of a bounded wait

template <int DP> struct TileShape {
	static constexpr int CHUNKS = DP / 64;
	static constexpr int BLOCK = CHUNKS * TL_CHUNK;     // bytes of a side's queries, of a key block, of a value block
	static constexpr int RING = DP == 64 ? 8 : 5;       // key and value blocks in flight
	static constexpr int SMEM = (2 + RING) * BLOCK + 1024;
	static constexpr int O_AT = 2 * TL_KEYS;            // column of the outputs
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const void *tmap, int c0, int c1, int c2, int c3, uint32_t bar) {
	asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(tmap)), "r"(c0),
				 "r"(c1), "r"(c2), "r"(c3), "r"(bar)
				 : "memory");
}
__device__ __forceinline__ bool wait_slow(uint32_t bar, uint32_t parity, volatile int *abort_flag) { return !*abort_flag && mbar_wait_bounded(bar, parity, TL_SPIN); }
__device__ __forceinline__ bool wait_fast(uint32_t bar, uint32_t parity, volatile int *abort_flag) { return mbar_try_wait(bar, parity) || wait_slow(bar, parity, abort_flag); }
// registers loaded by tcgen05.ld may be used only behind the wait: tie them to it
template <int N>
__device__ __forceinline__ void tmem_settle(float (&v)[N]) {
#pragma unroll
	for (int i = 0; i < N; ++i) asm volatile("" : "+f"(v[i]));
}
__device__ __forceinline__ bool elect() {
	uint32_t r;
	asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
	return r != 0;
}
// Values as the B operand: their columns are its N and lie one behind the other; chunks of 64 columns TL_CHUNK apart, a chunk holds
// rows of 128 bytes (a key each) in groups of 8, 1024 bytes apart; 128-byte swizzle.
__device__ __forceinline__ uint64_t desc_values(uint32_t addr) {
	return (uint64_t)((addr & 0x3FFFFu) >> 4) | (uint64_t)(TL_CHUNK >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// two fp32 operations per instruction
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pair(float a, float b) {
	f32x2 r;
	asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
	return r;
}
__device__ __forceinline__ void parts(f32x2 v, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
	f32x2 r;
	asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
	return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
	f32x2 r;
	asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
	return r;
}

// What a slot works off: every role walks through it for itself.
struct Items {
	PgEntry e;
	int kv, j0, j1;                    // key head, blocks of keys
	const PgEntry *entries, *sorted;
	PgStart end;                       // where the next slot begins
	int slot, kv_heads, whole, entry, entry_count, turn;
	__device__ Items(const PgWork &w, int kvh, int s) : entries(w.entries[1]), sorted(w.sorted), slot(s), kv_heads(kvh) {
		// (asked for together: which of them count depends on the list)
		const PgList l = read_list(w.list + 1);
		const PgStart st = read_start(w.starts[1] + s);
		const PgEntry first = read_entry(w.sorted + min(s / kvh, w.cap[1] - 1));
		end = read_start(w.starts[1] + s + 1);
		whole = l.whole;
		entry_count = l.entries;
		turn = 0;
		kv = whole ? 0 : st.kv;
		j1 = whole ? 0 : st.block;
		entry = whole ? 0 : st.entry;
		e = whole ? first : st.job;
	}
	__device__ bool next() {
		if (whole) {                     // sorted by length, dealt out forwards and backwards in turn
			constexpr int slots = PG_TILE_SLOTS;
			const int i = turn & 1 ? (turn + 1) * slots - 1 - slot : turn * slots + slot, at = i / kv_heads;
			if (at >= entry_count) return false;
			kv = i - at * kv_heads;
			if (turn++) e = read_entry(sorted + at);
			j0 = 0;
			j1 = e.blocks;
			return true;
		}
		if (entry < 0) return false;
		if (turn++) {
			if (j1 < e.blocks) return false;          // the rest is the next slot's
			j1 = 0;
			if (++kv == kv_heads) {
				kv = 0;
				if (++entry == entry_count) return false;
				e = read_entry(entries + entry);
			}
		}
		if (end.before(entry, kv)) return false;
		j0 = j1;
		j1 = end.in_job(entry, kv) ? end.block : e.blocks;
		return j0 < j1;
	}
};

// Keys that row i (of the tile) sees; 0: there is no such row
__device__ __forceinline__ int row_sees(const PgEntry &e, int i, int group, int &token, int &head) {
	const int64_t at = (int64_t)e.tile * PG_TILE + i;
	if (at >= (int64_t)e.fresh * group) return 0;
	token = (int)(at / group);
	head = (int)(at - (int64_t)token * group);
	return max(e.len - e.fresh + token + 1, 0);
}
// blocks of keys that side s sees at all
__device__ __forceinline__ int side_blocks(const PgEntry &e, int s, int group) {
	const int64_t rows = (int64_t)e.fresh * group - (int64_t)e.tile * PG_TILE, n = min(rows, (int64_t)(s + 1) * TL_SIDE);
	if (n <= s * TL_SIDE) return 0;
	const int token = (int)(((int64_t)e.tile * PG_TILE + n - 1) / group);
	return (max(e.len - e.fresh + token + 1, 1) + TL_KEYS - 1) / TL_KEYS;
}

template <typename T, int DP>
__global__ void __launch_bounds__(TL_THREADS, 1) tiles_kernel(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv, const paged_attention_t p, const PgWork work) {
	using S = TileShape<DP>;
	constexpr bool F16 = sizeof(T) == 2 && !std::is_same<T, bf16>::value;
	extern __shared__ unsigned char tl_raw[];
	__shared__ uint64_t s_bars[2 * S::RING + 13];
	__shared__ uint32_t s_tmem;
	__shared__ int s_stop;
	const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, group = p.heads / p.kv_heads;
	const uint32_t sq = (smem_u32(tl_raw) + 1023u) & ~1023u, ring = sq + 2 * S::BLOCK;
	const uint32_t bars = smem_u32(s_bars), bar_full = bars, bar_free = bars + 8 * S::RING, bar_q = bars + 16 * S::RING, bar_s = bar_q + 16, bar_p = bar_q + 32, bar_o = bar_q + 48, bar_none = bar_q + 64, bar_p2 = bar_q + 80, bar_end = bar_q + 96;
	volatile int *stop = &s_stop;
	if (tid == 0) {
		for (int i = 0; i < S::RING; ++i) {
			mbar_init(bar_full + 8 * i, 1);
			mbar_init(bar_free + 8 * i, 1);
		}
		for (int i = 0; i < 2; ++i) {
			mbar_init(bar_q + 8 * i, TL_SIDE / 32);          // a lane per warp arrives: 128 arrivals at one barrier take longer than the wait for them
			mbar_init(bar_s + 8 * i, 1);
			mbar_init(bar_p + 8 * i, TL_SIDE / 32);
			mbar_init(bar_p2 + 8 * i, TL_SIDE / 32);
			mbar_init(bar_o + 8 * i, 1);
			mbar_init(bar_none + 8 * i, 1);
		}
		mbar_init(bar_end, 1);
		s_stop = 0;
		fence_mbar_init();
	}
	if (warp == TL_MMA) {
		tmem_alloc(smem_u32(&s_tmem), 512);
		tmem_relinquish();
	}
	pdl_wait();
	pdl_trigger();
	Items it(work, p.kv_heads, blockIdx.x);
	bool have = it.next();
	tc_fence_before();
	__syncthreads();
	tc_fence_after();
	const uint32_t tmem = s_tmem;
	if (!have) {
		if (warp == TL_MMA) tmem_dealloc(tmem, 512);
		return;
	}
	auto fail = [&]() {
		*stop = 1;
		atomicOr(p.status, PAGED_TIMED_OUT);
	};

	if (warp >= 8) {
		asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(TL_REGS_OTHER));
	if (warp == TL_TMA) {
		// lane: page `mine / CHUNKS` of a block, columns 64 (mine % CHUNKS) ..
		const int per_block = p.page < TL_KEYS ? TL_KEYS / p.page : 1, loads = per_block * S::CHUNKS, box = min(p.page, TL_KEYS);
		const int sub = lane / S::CHUNKS, chunk = lane % S::CHUNKS;
		int n = 0, bad = 0;
		bool ok = true;
		const bool one = elect();
		for (; have && ok; have = it.next()) {
			const int *row = p.table + (int64_t)it.e.request * p.table_ld;
			auto page_at = [&](int j) {                    // page and row in it of this lane's part of block j
				const int key = j * TL_KEYS + sub * box;
				if (sub >= per_block || key >= it.e.seen) return -1;
				const int c = key / p.page;
				const int id = c < p.table_width ? __ldcg(row + c) : -2;
				if (id < 0 || id >= p.pages) {
					bad = PAGED_BAD_INDEX;
					return -1;
				}
				return id;
			};
			int id = page_at(it.j0);
			for (int j = it.j0; j < it.j1 && ok; ++j) {
				const int r0 = (j * TL_KEYS + sub * box) % p.page, now = id;
				if (j + 1 < it.j1) id = page_at(j + 1);
				for (int v = 0; v < 2; ++v, ++n) {
					const int b = n % S::RING;
					ok = wait_fast(bar_free + 8 * b, ((n / S::RING) & 1) ^ 1, stop);
					if (!__all_sync(0xffffffffu, ok)) {
						ok = false;
						fail();
						break;
					}
					if (lane == 0) mbar_arrive_expect_tx(bar_full + 8 * b, S::BLOCK);
					__syncwarp();
					for (int x = 0; x < per_block; ++x) {
						const int page = __shfl_sync(0xffffffffu, now, x * S::CHUNKS), first = __shfl_sync(0xffffffffu, r0, x * S::CHUNKS);
						if (one) {
#pragma unroll
							for (int c = 0; c < S::CHUNKS; ++c) tma_load_4d(ring + b * S::BLOCK + c * TL_CHUNK + x * box * 128, v ? &tmv : &tmk, 64 * c, first, it.kv, page, bar_full + 8 * b);
						}
					}
				}
			}
		}
		// no copy may be in flight when the CTA ends
		for (int i = max(0, n - S::RING); i < n; ++i) mbar_wait_bounded(bar_full + 8 * (i % S::RING), (i / S::RING) & 1, TL_SPIN);
		if (bad) atomicOr(p.status, bad);
		__syncwarp();
	}
	if (warp == TL_MMA) {
		if (elect()) {
			constexpr uint32_t base = (1u << 4) | (F16 ? 0u : (1u << 7) | (1u << 10)) | ((uint32_t)(TL_SIDE >> 4) << 24);          // D fp32, M = 128
			constexpr uint32_t id_qk = base | ((uint32_t)(TL_KEYS >> 3) << 17), id_pv = base | (1u << 16) | ((uint32_t)(DP >> 3) << 17);      // values: N contiguous
			int n = 0;                                     // blocks of the ring consumed
			uint32_t nq = 0, np[2] = {0, 0};
			bool ok = true;
			auto wait = [&](uint32_t bar, uint32_t parity) {
				if (ok && !wait_fast(bar, parity & 1, stop)) {
					ok = false;
					fail();
				}
				return ok;
			};
			auto full = [&](int i) { return wait(bar_full + 8 * (i % S::RING), i / S::RING); };
			auto qk = [&](int s, int i) {
				const uint64_t qd = smem_desc_sw128(sq + s * S::BLOCK), kd = smem_desc_sw128(ring + (i % S::RING) * S::BLOCK);
#pragma unroll
				for (int k = 0; k < DP / 16; ++k) umma_f16(tmem + s * TL_KEYS, qd + (k >> 2) * (TL_CHUNK / 16) + 2 * (k & 3), kd + (k >> 2) * (TL_CHUNK / 16) + 2 * (k & 3), id_qk, k ? 1u : 0u);
				umma_commit(bar_s + 8 * s);
			};
			auto pv = [&](int s, int i, int half, bool first) {          // 64 of the 128 keys
				const uint64_t vd = desc_values(ring + (i % S::RING) * S::BLOCK);
				tc_fence_after();
#pragma unroll
				for (int k = half * (TL_KEYS / 32); k < (half + 1) * (TL_KEYS / 32); ++k) umma_f16_ts(tmem + S::O_AT + s * DP, tmem + s * TL_KEYS + 8 * k, vd + 128 * k, id_pv, first && k == 0 ? 0u : 1u);
			};
			for (; have && ok; have = it.next(), ++nq) {
				// side s: blocks it.j0 .. ends[s] - 1
				const int ends[2] = {min(it.j1, side_blocks(it.e, 0, group)), min(it.j1, side_blocks(it.e, 1, group))};
				if (!full(n)) break;
				for (int s = 0; s < 2; ++s) {
					if (!wait(bar_q + 8 * s, nq)) break;
					tc_fence_after();
					if (it.j0 < ends[s]) qk(s, n);
					else umma_commit(bar_none + 8 * s);
				}
				if (!ok) break;
				umma_commit(bar_free + 8 * (n % S::RING));
				for (int j = it.j0; j < it.j1; ++j, n += 2) {
					const bool again = j + 1 < it.j1;
					if (!full(n + 1) || (again && !full(n + 2))) break;
					for (int s = 0; s < 2 && ok; ++s) {
						if (j < ends[s]) {
							if (wait(bar_p + 8 * s, np[s])) pv(s, n + 1, 0, j == it.j0);
							if (wait(bar_p2 + 8 * s, np[s]++)) pv(s, n + 1, 1, false);
						}
						if (ok && j + 1 < ends[s]) qk(s, n + 2);
						if (ok && j + 1 == ends[s]) umma_commit(bar_o + 8 * s);
					}
					if (!ok) break;
					umma_commit(bar_free + 8 * ((n + 1) % S::RING));
					if (again) umma_commit(bar_free + 8 * ((n + 2) % S::RING));
				}
				if (!ok) break;
			}
			umma_commit(bar_end);                          // every MMA has completed before tensor memory goes back
			mbar_wait_bounded(bar_end, 0, TL_SPIN);
		}
		__syncwarp();
	}
	} else {
		asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(TL_REGS_SOFTMAX));
		const int side = warp >> 2, rl = (warp & 3) * 32 + lane, row = side * TL_SIDE + rl;
		const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16, ts = tmem + side * TL_KEYS + lane_base, to = tmem + S::O_AT + side * DP + lane_base;
		const float scale2 = p.scale * PG_LOG2E;
		constexpr float LIFT = F16 ? 7.f : 0.f;            // fp16 weights up to 2^15: small ones stay above its subnormal range
		const bool sectors = p.dim % 16 == 0 && (reinterpret_cast<uintptr_t>(p.out) & 31) == 0;          // rows in whole sectors of 32 bytes
		uint32_t ns = 0, no = 0, nn = 0;
		int blocks = 0;                                    // of the ring before this tile's
		bool ok = true;
		auto wait = [&](uint32_t bar, uint32_t parity) {
			ok = ok && wait_fast(bar, parity & 1, stop);
			if (!__all_sync(0xffffffffu, ok)) {
				ok = false;
				fail();
			}
			tc_fence_after();
			return ok;
		};
		int token = 0, head = 0, sees = 0;
		// The warp's 32 rows, to shared memory as the A operand: a row is 16 bytes times DP / 8 lanes, so that whole lines are read.
		auto queries = [&]() {
			sees = row_sees(it.e, row, group, token, head);
			const unsigned long long src = sees > 0 ? reinterpret_cast<unsigned long long>(reinterpret_cast<const T *>(p.q) + (int64_t)(it.e.row + token) * p.q_row + (int64_t)(it.kv * group + head) * p.q_head) : 0;
			constexpr int LANES = DP / 8, ROWS = 32 / LANES;
			const int u = lane % LANES, sub = lane / LANES;
			const uint32_t dst = sq + side * S::BLOCK + (u >> 3) * TL_CHUNK + (warp & 3) * 32 * 128;
			const bool column = 8 * u < p.dim;
#pragma unroll
			for (int r = 0; r < 32; r += ROWS) {
				const int x = r + sub;
				const unsigned long long from = __shfl_sync(0xffffffffu, src, x);
				cp_async16_or_zero(dst + x * 128 + (((u & 7) ^ (x & 7)) << 4), from && column ? reinterpret_cast<const void *>(from + 16 * u) : p.q, from && column ? 16 : 0);
			}
			cp_async_commit();
			cp_async_wait<0>();
			fence_proxy_async();
			__syncwarp();
			if (lane == 0) mbar_arrive(bar_q + 8 * side);
		};
		queries();
		while (have && ok) {
			const int end = min(it.j1, side_blocks(it.e, side, group));
			float ref = -INFINITY;
			f32x2 total = pair(0.f, 0.f);
			for (int j = it.j0; j < end; ++j) {
				if (!wait(bar_s + 8 * side, ns++)) break;
				float s[4][32];
#pragma unroll
				for (int c = 0; c < 4; ++c) tmem_ld32(ts + 32 * c, s[c]);
				tmem_ld_wait();
#pragma unroll
				for (int c = 0; c < 4; ++c) tmem_settle(s[c]);
				const int visible = sees - j * TL_KEYS;      // keys of this block
				if (__any_sync(0xffffffffu, visible < TL_KEYS)) {
#pragma unroll
					for (int k = 0; k < TL_KEYS; ++k)
						if (k >= visible) s[k >> 5][k & 31] = -INFINITY;
				}
				float m[4];
#pragma unroll
				for (int c = 0; c < 4; ++c) {
					m[c] = s[c][0];
#pragma unroll
					for (int k = 1; k < 31; k += 2) m[c] = fmaxf(m[c], fmaxf(s[c][k], s[c][k + 1]));
					m[c] = fmaxf(m[c], s[c][31]);
				}
				const float top = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])) * scale2;
				if (__any_sync(0xffffffffu, top > ref + 8.f)) {
					const float next = fmaxf(ref, top), keep = ref == -INFINITY ? 0.f : ex2(ref - next);
					ref = next;
					float a, b;
					parts(total, a, b);
					total = pair(a * keep, b * keep);
					if (j != it.j0) {                          // (the products before this block are complete: its scores came after them)
#pragma unroll 1
						for (int c = 0; c < DP; c += 32) {
							float o[32];
							tmem_ld32(to + c, o);
							tmem_ld_wait();
							tmem_settle(o);
#pragma unroll
							for (int k = 0; k < 32; ++k) o[k] *= keep;
							tmem_st32(to + c, reinterpret_cast<uint32_t(&)[32]>(o));
						}
					}
				}
				const float at = ref == -INFINITY ? 0.f : LIFT - ref;
				const f32x2 mul = pair(scale2, scale2), off = pair(at, at);
				f32x2 sums[4] = {total, pair(0.f, 0.f), pair(0.f, 0.f), pair(0.f, 0.f)};          // four chains of additions
#pragma unroll
				for (int h = 0; h < 2; ++h) {
					uint32_t w[32];
#pragma unroll
					for (int k = 0; k < 32; ++k) {
						const int c = 2 * h + (k >> 4), i = 2 * (k & 15);
						float a, b;
						parts(fma2(pair(s[c][i], s[c][i + 1]), mul, off), a, b);
						a = ex2(a);
						b = ex2(b);
						sums[k & 3] = add2(sums[k & 3], pair(a, b));
						w[k] = pack2<T>(a, b);
					}
					tmem_st32(ts + 32 * h, w);
					if (h == 0 && it.e.seen - j * TL_KEYS < TL_KEYS) {
						// The last block of a tile: values behind the last key seen become zeros before the weights are handed over (both sides write
						// the same, each before its own products).
						const int i = blocks + 2 * (j - it.j0) + 1, tail = it.e.seen - j * TL_KEYS;
						wait(bar_full + 8 * (i % S::RING), i / S::RING);
						const uint32_t v = ring + (i % S::RING) * S::BLOCK;
						for (int x = tid & (TL_SIDE - 1); x < (TL_KEYS - tail) * 8 * S::CHUNKS; x += TL_SIDE) {
							const int unit = x & 7, rest = x >> 3, c = rest % S::CHUNKS, r = tail + rest / S::CHUNKS;
							asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(v + c * TL_CHUNK + r * 128 + unit * 16), "r"(0) : "memory");
						}
						fence_proxy_async();
					}
					tmem_st_wait();
					tc_fence_before();
					__syncwarp();
					if (lane == 0) mbar_arrive((h ? bar_p2 : bar_p) + 8 * side);
				}
				total = add2(add2(sums[0], sums[1]), add2(sums[2], sums[3]));
			}
			if (!ok) break;
			// the next tile's queries go first: its scores are computed while this one's results are stored
			const PgEntry e = it.e;
			blocks += 2 * (it.j1 - it.j0);
			const int kv = it.kv, j0 = it.j0, j1 = it.j1, my_token = token, my_head = head, my_sees = sees;
			// A side without blocks in this tile must not run ahead of the MMA warp: a wait tells a phase from its neighbours only.  (Not bar_o:
			// the MMA warp may come to this while the results of the tile before still wait to be read.)
			if (j0 >= end && !wait(bar_none + 8 * side, nn++)) break;
			have = it.next();
			if (have) queries();
			float a, b;
			parts(total, a, b);
			const float sum = a + b;
			const bool any = j0 < end, whole = j0 == 0 && j1 == e.blocks;
			if (any && !wait(bar_o + 8 * side, no++)) break;
			const bool mine = (int64_t)e.tile * PG_TILE + row < (int64_t)e.fresh * group;
			const float f = sum > 0.f || my_sees > 0 ? 1.f / sum : 0.f;
			T *dst = reinterpret_cast<T *>(p.out) + ((int64_t)(e.row + my_token) * p.heads + kv * group + my_head) * p.dim;
			float *part = reinterpret_cast<float *>(p.scratch) + (int64_t)(2 * blockIdx.x + (j0 == 0)) * PG_TILE * (DP + 2);
			if (!whole && mine) __stcg(reinterpret_cast<float2 *>(part + PG_TILE * DP) + row, make_float2(any ? ref : -INFINITY, sum));
#pragma unroll 1
			for (int c = 0; c < DP; c += 32) {
				float o[32];
				if (any) {
					tmem_ld32(to + c, o);
					tmem_ld_wait();
					tmem_settle(o);
				} else {
#pragma unroll
					for (int k = 0; k < 32; ++k) o[k] = 0.f;
				}
				if (!mine) continue;
				if (whole) {
#pragma unroll
					for (int k = 0; k < 32; k += 16) {
						if (c + k >= p.dim) break;
						uint32_t v[8];
#pragma unroll
						for (int x = 0; x < 8; ++x) v[x] = my_sees > 0 ? pack2<T>(o[k + 2 * x] * f, o[k + 2 * x + 1] * f) : 0u;
						if (sectors) {
							asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst + c + k), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
						} else {
							*reinterpret_cast<uint4 *>(dst + c + k) = make_uint4(v[0], v[1], v[2], v[3]);
							if (c + k + 8 < p.dim) *reinterpret_cast<uint4 *>(dst + c + k + 8) = make_uint4(v[4], v[5], v[6], v[7]);
						}
					}
				} else {
#pragma unroll
					for (int k = 0; k < 32; k += 4) __stcg(reinterpret_cast<float4 *>(part + (int64_t)row * DP + c + k), make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]));
				}
			}
			tc_fence_before();
		}
	}
	tc_fence_before();
	__syncthreads();
	if (warp == TL_MMA) tmem_dealloc(tmem, 512);
}

EncodeTiledFn encoder() {
	static EncodeTiledFn fn = nullptr;
	static std::once_flag once;
	std::call_once(once, [] {
		void *ptr = nullptr;
		cudaDriverEntryPointQueryResult q;
		if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess) fn = reinterpret_cast<EncodeTiledFn>(ptr);
	});
	return fn;
}

// a cache tensor [pages, kv_heads, page, dim] in boxes of 64 columns of (part of) a page
int cache_map(const void *base, const paged_attention_t &p, int64_t page_step, int64_t kv_step, bool half, CUtensorMap *out) {
	EncodeTiledFn enc = encoder();
	if (!enc) return GPTQ_ERR_CUDA;
	const int64_t block = (int64_t)p.page * p.dim;
	const cuuint64_t dims[4] = {(cuuint64_t)p.dim, (cuuint64_t)p.page, (cuuint64_t)p.kv_heads, (cuuint64_t)p.pages};
	const cuuint64_t strides[3] = {(cuuint64_t)p.dim * 2, (cuuint64_t)(p.kv_heads > 1 ? kv_step : block) * 2, (cuuint64_t)(p.pages > 1 ? page_step : block) * 2};
	const cuuint32_t box[4] = {64, (cuuint32_t)(p.page < TL_KEYS ? p.page : TL_KEYS), 1, 1}, step[4] = {1, 1, 1, 1};
	const CUresult r = enc(out, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void *>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
						   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
	if (r != CUDA_SUCCESS) {
		g_last_cuda_error = (int)r;
		return GPTQ_ERR_CUDA;
	}
	return GPTQ_OK;
}

template <typename T, int DP>
int tiles_launch(const paged_attention_t &p, const PgWork &work, bool half, cudaStream_t stream) {
	alignas(64) CUtensorMap tmk, tmv;
	if (int rc = cache_map(p.k_cache, p, p.k_page, p.k_kv, half, &tmk)) return rc;
	if (int rc = cache_map(p.v_cache, p, p.v_page, p.v_kv, half, &tmv)) return rc;
	constexpr int smem = TileShape<DP>::SMEM;
	static_assert(smem + 1024 <= 227 * 1024, "shared memory of a CTA");
	static const int registers = [] {
		cudaFuncAttributes attr;
		return cudaFuncGetAttributes(&attr, tiles_kernel<T, DP>) == cudaSuccess ? attr.numRegs : 0;
	}();
	if (registers < TL_REGS_LAUNCH) return GPTQ_ERR_UNSUPPORTED;          // (the softmax warps would wait for registers that nobody gives back)
	return pg_launch(tiles_kernel<T, DP>, dim3(PG_TILE_SLOTS), TL_THREADS, smem, stream, tmk, tmv, p, work);
}

}   // namespace

int64_t pg_tiles_scratch(const paged_attention_t &p) { return (int64_t)2 * PG_TILE_SLOTS * PG_TILE * ((p.dim <= 64 ? 64 : 128) + 2) * 4; }

int pg_tiles_launch(const paged_attention_t &p, int dtype, char *scratch, cudaStream_t stream) {
	const PgWork work = pg_work(const_cast<int32_t *>(p.work), p.requests, p.rows, p.heads, p.kv_heads);
	paged_attention_t a = p;
	a.scratch = scratch;
	if (dtype == PG_BF16) return p.dim <= 64 ? tiles_launch<bf16, 64>(a, work, false, stream) : tiles_launch<bf16, 128>(a, work, false, stream);
	return p.dim <= 64 ? tiles_launch<__half, 64>(a, work, true, stream) : tiles_launch<__half, 128>(a, work, true, stream);
}

}   // namespace gptq
