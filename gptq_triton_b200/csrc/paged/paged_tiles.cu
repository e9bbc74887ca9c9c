// Attention of chunks over a cache in pages on the 5th-generation tensor cores (fp16, bf16, heads of up to 128).
//
// A tile is 256 rows (new tokens times the query heads of a key head, token-major, so that short chunks with shared key heads fill it):
// two sides of 128, whose scores and outputs take the 512 columns of tensor memory.  Per block of 128 keys and side: S = Q K^T, online
// softmax, O += P V; while the softmax warps of one side work, the tensor cores work for the other.
//   softmax warps   eight per side, two threads share a row (64 keys each, they exchange their maxima): scores from tensor memory, mask
//                   where the block crosses what the row sees, weights in the type of the values back to the columns of the scores (they
//                   are the A operand of P V there).  With a thread per row (16 KB less to exchange, 1.6 times the chain from the scores
//                   to the weights) tensor cores and exponentials stood at 41 % each.
//   TMA warp        key and value blocks through one ring; a lane per page and 64 columns of a block, so pages of 8 rows and more serve;
//                   pages behind what the tile sees, or that do not exist, are asked for outside the tensor and arrive as zeros
//   MMA warp        both sides in turn: P V of this block, Q K^T of the next
// O is rescaled only when a row's maximum has grown by more than 2^8.  fp32 sums; weights are rounded to the type of the values, their
// sum is taken before that.  Values behind the last key seen are zeroed in shared memory: a weight of zero times NaN would be NaN.
// CTAs stay for the whole launch and take tiles, or equal ranges of all key blocks (paged_plan); ranges that end inside a tile leave
// partial results, which tile_join_kernel adds up.  Every wait is bounded.
#include <mutex>

#include "../tcgen05.cuh"
#include "paged.cuh"

namespace gptq {

namespace {

constexpr int TL_SIDE = 128, TL_KEYS = PG_TILE_KEYS;
constexpr int TL_CHUNK = 128 * 128;                      // bytes of 128 rows of 64 columns
constexpr int TL_THREADS = 640, TL_TMA = 16, TL_MMA = 17;
constexpr int TL_HEAD = 3072;                            // shared memory ahead of the operands: exchange of the halves, barriers
constexpr uint32_t TL_SPIN = 1u << 24;                  // polls of a bounded wait

template <int DP> struct TileShape {
	static constexpr int CHUNKS = DP / 64;
	static constexpr int BLOCK = CHUNKS * TL_CHUNK;     // bytes of a side's queries, of a key block, of a value block
	static constexpr int RING = DP == 64 ? 8 : 5;       // key and value blocks in flight
	static constexpr int SMEM = TL_HEAD + (2 + RING) * BLOCK;
	static constexpr int BARS = 2 * RING + 13;
	static_assert(4 * TL_SIDE * 4 + 8 * BARS + 8 <= TL_HEAD, "room ahead of the operands");
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
// One lane of the warp, known to the compiler as one: operands of the instructions behind `lane == 0` are taken for different ones in
// every lane, and eight MMAs then took 450 cycles to issue.
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
	const PgEntry *entries;
	const int *order;
	int slot, slots, kv_heads, whole, entry;
	int left, turn, count;             // (a slot's share and the number of tiles are far below 2^31: the plan's sums stop at 2^30 per key head)
	__device__ Items(const PgWork &w, int kvh, int s) : entries(w.entries[1]), order(w.order), slot(s), slots(PG_TILE_SLOTS), kv_heads(kvh) {
		const PgList l = w.list[1];
		whole = l.whole;
		turn = 0;
		count = (int)min((int64_t)l.entries * kvh, (int64_t)1 << 30);
		left = (int)max(min(min(l.per, (int64_t)1 << 30), l.total - (int64_t)s * l.per), (int64_t)0);
		kv = j1 = 0;
		entry = 0;
		if (!whole && left > 0) {
			const PgStart st = w.starts[1][s];
			entry = st.entry;
			kv = st.kv;
			j1 = st.block;
			e = read(entry);
		}
	}
	__device__ PgEntry read(int i) const {
		const int4 a = __ldg(reinterpret_cast<const int4 *>(entries + i)), b = __ldg(reinterpret_cast<const int4 *>(entries + i) + 1);
		return PgEntry{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
	}
	__device__ bool next() {
		if (whole) {                     // sorted by length, dealt out forwards and backwards in turn
			const int i = turn & 1 ? (turn + 1) * slots - 1 - slot : turn * slots + slot;
			++turn;
			if (i >= count) return false;
			kv = i % kv_heads;
			e = read(__ldg(order + i / kv_heads));
			j0 = 0;
			j1 = e.blocks;
			return true;
		}
		if (left <= 0) return false;
		if (turn++ && j1 == e.blocks) {          // the tile before was finished
			j1 = 0;
			if (++kv == kv_heads) {
				kv = 0;
				e = read(++entry);
			}
		}
		j0 = j1;
		j1 = e.blocks - j0 < left ? e.blocks : j0 + left;
		left -= j1 - j0;
		return true;
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
	extern __shared__ __align__(1024) unsigned char tl_raw[];
	float *s_pass = reinterpret_cast<float *>(tl_raw);                      // [side][half][row]
	uint64_t *s_bars = reinterpret_cast<uint64_t *>(tl_raw + 4 * TL_SIDE * 4);
	uint32_t *s_tmem = reinterpret_cast<uint32_t *>(s_bars + S::BARS);
	volatile int *stop = reinterpret_cast<volatile int *>(s_tmem + 1);
	const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, group = p.heads / p.kv_heads;
	const uint32_t sq = smem_u32(tl_raw) + TL_HEAD, ring = sq + 2 * S::BLOCK;
	const uint32_t bars = smem_u32(s_bars), bar_full = bars, bar_free = bars + 8 * S::RING, bar_q = bars + 16 * S::RING, bar_s = bar_q + 16, bar_p = bar_q + 32, bar_o = bar_q + 48, bar_none = bar_q + 64, bar_p2 = bar_q + 80, bar_end = bar_q + 96;
	Items it(work, p.kv_heads, blockIdx.x);
	bool have = it.next();
	if (!have) return;
	if (sq & 1023u) {                                    // (swizzled operands; does not happen without static shared memory)
		if (tid == 0) atomicOr(p.status, 2);
		return;
	}
	if (tid == 0) {
		for (int i = 0; i < S::RING; ++i) {
			mbar_init(bar_full + 8 * i, 1);
			mbar_init(bar_free + 8 * i, 1);
		}
		for (int i = 0; i < 2; ++i) {
			mbar_init(bar_q + 8 * i, 2 * TL_SIDE);
			mbar_init(bar_s + 8 * i, 1);
			mbar_init(bar_p + 8 * i, TL_SIDE);
			mbar_init(bar_p2 + 8 * i, TL_SIDE);
			mbar_init(bar_o + 8 * i, 1);
			mbar_init(bar_none + 8 * i, 1);
		}
		mbar_init(bar_end, 1);
		*stop = 0;
		fence_mbar_init();
	}
	if (warp == TL_MMA) {
		tmem_alloc(smem_u32(s_tmem), 512);
		tmem_relinquish();
	}
	tc_fence_before();
	__syncthreads();
	tc_fence_after();
	const uint32_t tmem = *s_tmem;
	auto fail = [&]() {
		*stop = 1;
		atomicOr(p.status, 3);
	};

	if (warp == TL_TMA) {
		// lane: page `mine / CHUNKS` of a block, columns 64 (mine % CHUNKS) ..
		const int per_block = p.page < TL_KEYS ? TL_KEYS / p.page : 1, loads = per_block * S::CHUNKS, box = min(p.page, TL_KEYS);
		const int sub = lane / S::CHUNKS, chunk = lane % S::CHUNKS;
		int n = 0, bad = 0;
		bool ok = true;
		for (; have && ok; have = it.next()) {
			const int *row = p.table + (int64_t)it.e.request * p.table_ld;
			auto page_at = [&](int j) {                    // page and row in it of this lane's part of block j
				const int key = j * TL_KEYS + sub * box;
				if (sub >= per_block || key >= it.e.seen) return -1;
				const int c = key / p.page;
				const int id = c < p.table_width ? __ldg(row + c) : -2;
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
					if (lane < loads) tma_load_4d(ring + b * S::BLOCK + chunk * TL_CHUNK + sub * box * 128, v ? &tmv : &tmk, 64 * chunk, r0, it.kv, now, bar_full + 8 * b);
				}
			}
		}
		// no copy may be in flight when the CTA ends
		for (int i = max(0, n - S::RING); i < n; ++i) mbar_wait_bounded(bar_full + 8 * (i % S::RING), (i / S::RING) & 1, TL_SPIN);
		if (bad) atomicOr(p.status, bad);
		__syncwarp();
	} else if (warp == TL_MMA) {
		constexpr uint32_t base = (1u << 4) | (F16 ? 0u : (1u << 7) | (1u << 10)) | ((uint32_t)(TL_SIDE >> 4) << 24);          // D fp32, M = 128
		constexpr uint32_t id_qk = base | ((uint32_t)(TL_KEYS >> 3) << 17), id_pv = base | (1u << 16) | ((uint32_t)(DP >> 3) << 17);      // values: N contiguous
		const bool one = elect();
		int n = 0;                                         // blocks of the ring consumed
		uint32_t nq = 0, np[2] = {0, 0};
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
		auto full = [&](int i) { return wait(bar_full + 8 * (i % S::RING), i / S::RING); };
		auto qk = [&](int s, int i) {
			if (one) {
				const uint64_t qd = smem_desc_sw128(sq + s * S::BLOCK), kd = smem_desc_sw128(ring + (i % S::RING) * S::BLOCK);
#pragma unroll
				for (int k = 0; k < DP / 16; ++k) umma_f16(tmem + s * TL_KEYS, qd + (k >> 2) * (TL_CHUNK / 16) + 2 * (k & 3), kd + (k >> 2) * (TL_CHUNK / 16) + 2 * (k & 3), id_qk, k ? 1u : 0u);
				umma_commit(bar_s + 8 * s);
			}
			__syncwarp();
		};
		auto pv = [&](int s, int i, int half, bool first) {          // 64 of the 128 keys
			if (one) {
				const uint64_t vd = desc_values(ring + (i % S::RING) * S::BLOCK);
#pragma unroll
				for (int k = half * (TL_KEYS / 32); k < (half + 1) * (TL_KEYS / 32); ++k) umma_f16_ts(tmem + S::O_AT + s * DP, tmem + s * TL_KEYS + (k >> 2) * 64 + (k & 3) * 8, vd + 128 * k, id_pv, first && k == 0 ? 0u : 1u);
			}
			__syncwarp();
		};
		auto commit = [&](uint32_t bar) {
			if (one) umma_commit(bar);
			__syncwarp();
		};
		for (; have && ok; have = it.next(), ++nq) {
			// side s: blocks it.j0 .. ends[s] - 1
			const int ends[2] = {min(it.j1, side_blocks(it.e, 0, group)), min(it.j1, side_blocks(it.e, 1, group))};
			if (!full(n)) break;
			for (int s = 0; s < 2 && ok; ++s) {
				if (!wait(bar_q + 8 * s, nq)) break;
				if (it.j0 < ends[s]) qk(s, n);
				else commit(bar_none + 8 * s);
			}
			if (!ok) break;
			commit(bar_free + 8 * (n % S::RING));
			for (int j = it.j0; j < it.j1 && ok; ++j, n += 2) {
				if (!full(n + 1)) break;
				const int tail = it.e.seen - j * TL_KEYS;
				if (tail < TL_KEYS) {                      // (only the last block of a tile)
					const uint32_t v = ring + ((n + 1) % S::RING) * S::BLOCK;
					for (int x = lane; x < (TL_KEYS - tail) * 8 * S::CHUNKS; x += 32) {
						const int unit = x & 7, rest = x >> 3, c = rest % S::CHUNKS, r = tail + rest / S::CHUNKS;
						asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(v + c * TL_CHUNK + r * 128 + unit * 16), "r"(0) : "memory");
					}
					fence_proxy_async();
					__syncwarp();
				}
				const bool again = j + 1 < it.j1;
				if (again && !full(n + 2)) break;
				for (int s = 0; s < 2 && ok; ++s) {
					if (j < ends[s]) {
						if (wait(bar_p + 8 * s, np[s])) pv(s, n + 1, 0, j == it.j0);
						if (wait(bar_p2 + 8 * s, np[s]++)) pv(s, n + 1, 1, false);
					}
					if (ok && j + 1 < ends[s]) qk(s, n + 2);
					if (ok && j + 1 == ends[s]) commit(bar_o + 8 * s);
				}
				if (!ok) break;
				commit(bar_free + 8 * ((n + 1) % S::RING));
				if (again) commit(bar_free + 8 * ((n + 2) % S::RING));
			}
		}
		commit(bar_end);                                 // every MMA has completed before tensor memory goes back
		mbar_wait_bounded(bar_end, 0, TL_SPIN);
		__syncwarp();
	} else if (warp < TL_TMA) {
		const int side = warp >> 3, half = (warp >> 2) & 1, rl = (warp & 3) * 32 + lane, row = side * TL_SIDE + rl;
		const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16, ts = tmem + side * TL_KEYS + half * 64 + lane_base, to = tmem + S::O_AT + side * DP + half * (DP / 2) + lane_base;
		float *mine_s = s_pass + (2 * side + half) * TL_SIDE + rl, *other_s = s_pass + (2 * side + 1 - half) * TL_SIDE + rl;
		const float scale2 = p.scale * PG_LOG2E;
		constexpr float LIFT = F16 ? 7.f : 0.f;            // fp16 weights up to 2^15: small ones stay above its subnormal range
		// the two warps that share 32 rows
		auto meet = [&]() { asm volatile("bar.sync %0, 64;" ::"r"(1 + side * 4 + (warp & 3)) : "memory"); };
		uint32_t ns = 0, no = 0, nn = 0;
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
		auto queries = [&]() {                             // this thread's row, to shared memory as the A operand
			sees = row_sees(it.e, row, group, token, head);
			const uint32_t dst = sq + side * S::BLOCK + rl * 128;
			const T *src = reinterpret_cast<const T *>(p.q) + (int64_t)(it.e.row + token) * p.q_row + (int64_t)(it.kv * group + head) * p.q_head;
#pragma unroll
			for (int u = half * (DP / 16); u < (half + 1) * (DP / 16); ++u) {
				uint4 v = make_uint4(0u, 0u, 0u, 0u);
				if (sees > 0 && 8 * u < p.dim) v = __ldg(reinterpret_cast<const uint4 *>(src + 8 * u));
				asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(dst + (u >> 3) * TL_CHUNK + (((u & 7) ^ (rl & 7)) << 4)), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
			}
			fence_proxy_async();
			mbar_arrive(bar_q + 8 * side);
		};
		queries();
		while (have) {
			const int end = min(it.j1, side_blocks(it.e, side, group));
			float ref = -INFINITY;
			f32x2 total = pair(0.f, 0.f);
			for (int j = it.j0; j < end; ++j) {
				// (a wait that ran out does not leave the loop: the two warps of a row must keep meeting)
				wait(bar_s + 8 * side, ns++);
				float s[2][32];
				tmem_ld32(ts, s[0]);
				tmem_ld32(ts + 32, s[1]);
				tmem_ld_wait();
				tmem_settle(s[0]);
				tmem_settle(s[1]);
				const int visible = sees - j * TL_KEYS - half * 64;      // keys of this half of the block
				if (__any_sync(0xffffffffu, visible < 64)) {
#pragma unroll
					for (int k = 0; k < 64; ++k)
						if (k >= visible) s[k >> 5][k & 31] = -INFINITY;
				}
				float m[2];
#pragma unroll
				for (int c = 0; c < 2; ++c) {
					m[c] = s[c][0];
#pragma unroll
					for (int k = 1; k < 31; k += 2) m[c] = fmaxf(m[c], fmaxf(s[c][k], s[c][k + 1]));
					m[c] = fmaxf(m[c], s[c][31]);
				}
				float top = fmaxf(m[0], m[1]);
				*mine_s = top;
				meet();
				// (written again for the next block only: its scores come after both warps have handed over their weights of this one)
				top = fmaxf(top, *other_s) * scale2;
				if (__any_sync(0xffffffffu, top > ref + 8.f)) {          // the same rows, so the same decision in both warps
					const float next = fmaxf(ref, top), keep = ref == -INFINITY ? 0.f : ex2(ref - next);
					ref = next;
					float a, b;
					parts(total, a, b);
					total = pair(a * keep, b * keep);
					if (j != it.j0) {                          // (the products before this block are complete: its scores came after them)
#pragma unroll 1
						for (int c = 0; c < DP / 2; c += 16) {
							float o[16];
							tmem_ld16(to + c, o);
							tmem_ld_wait();
							tmem_settle(o);
#pragma unroll
							for (int k = 0; k < 16; ++k) o[k] *= keep;
							tmem_st16(to + c, o);
						}
						tmem_st_wait();
						meet();                                // neither half's weights may be multiplied into the other's columns before
					}
				}
				const float at = ref == -INFINITY ? 0.f : LIFT - ref;
				const f32x2 mul = pair(scale2, scale2), off = pair(at, at);
#pragma unroll
				for (int c = 0; c < 2; ++c) {
					uint32_t w[16];
#pragma unroll
					for (int k = 0; k < 16; ++k) {
						float a, b;
						parts(fma2(pair(s[c][2 * k], s[c][2 * k + 1]), mul, off), a, b);
						a = ex2(a);
						b = ex2(b);
						total = add2(total, pair(a, b));
						w[k] = pack2<T>(a, b);
					}
					tmem_st16(ts + 16 * c, reinterpret_cast<float(&)[16]>(w));
				}
				tmem_st_wait();
				tc_fence_before();
				mbar_arrive((half ? bar_p2 : bar_p) + 8 * side);
			}
			const bool any = it.j0 < end, whole = it.j0 == 0 && it.j1 == it.e.blocks, blind = sees <= 0;
			const bool mine = (int64_t)it.e.tile * PG_TILE + row < (int64_t)it.e.fresh * group;
			T *dst = reinterpret_cast<T *>(p.out) + ((int64_t)(it.e.row + token) * p.heads + it.kv * group + head) * p.dim;
			float *part = reinterpret_cast<float *>(p.scratch) + (int64_t)(2 * blockIdx.x + (it.j0 == 0)) * PG_TILE * (DP + 2);
			// A side without blocks in this tile must not run ahead of the MMA warp: a wait tells a phase from its neighbours only.  (Not bar_o:
			// the MMA warp may come to this while the results of the tile before still wait to be read.)
			if (!any) wait(bar_none + 8 * side, nn++);
			// the next tile's queries go first: its scores are computed while this one's results are stored
			have = it.next();
			if (have) queries();
			if (any) wait(bar_o + 8 * side, no++);
			float a, b;
			parts(total, a, b);
			const float mine_sum = ok ? a + b : -1.f;          // (sums are not negative: both warps of a row learn of a wait that ran out)
			*mine_s = mine_sum;
			meet();
			const float other_sum = *other_s, sum = half ? other_sum + mine_sum : mine_sum + other_sum;
			meet();
			if (__any_sync(0xffffffffu, mine_sum < 0.f || other_sum < 0.f)) break;
			const float f = 1.f / sum;
			if (!whole && mine && half == 0) __stcg(reinterpret_cast<float2 *>(part + PG_TILE * DP) + row, make_float2(any ? ref : -INFINITY, sum));
#pragma unroll 1
			for (int c = 0; c < DP / 2; c += 16) {
				float o[16];
				if (any) {
					tmem_ld16(to + c, o);
					tmem_ld_wait();
					tmem_settle(o);
				} else {
#pragma unroll
					for (int k = 0; k < 16; ++k) o[k] = 0.f;
				}
				const int col = half * (DP / 2) + c;
				if (!mine) continue;
				if (whole) {
#pragma unroll
					for (int k = 0; k < 16; k += 8) {
						if (col + k >= p.dim) break;
						uint4 v;
						v.x = pack2<T>(o[k] * f, o[k + 1] * f);
						v.y = pack2<T>(o[k + 2] * f, o[k + 3] * f);
						v.z = pack2<T>(o[k + 4] * f, o[k + 5] * f);
						v.w = pack2<T>(o[k + 6] * f, o[k + 7] * f);
						if (blind) v = make_uint4(0u, 0u, 0u, 0u);
						*reinterpret_cast<uint4 *>(dst + col + k) = v;
					}
				} else {
#pragma unroll
					for (int k = 0; k < 16; k += 4) __stcg(reinterpret_cast<float4 *>(part + (int64_t)row * DP + col + k), make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]));
				}
			}
			tc_fence_before();
		}
	}
	tc_fence_before();
	__syncthreads();
	if (warp == TL_MMA) tmem_dealloc(tmem, 512);
}

// CTA (c, g) joins rows 16 g .. of the tile whose keys begin in slot c and end in a later one.
template <typename T, int DP>
__global__ void __launch_bounds__(128) tile_join_kernel(const paged_attention_t p, const PgWork work) {
	const PgList list = work.list[1];
	const int slot = blockIdx.x, group = p.heads / p.kv_heads;
	if (list.whole || (slot + 1) * list.per >= list.total) return;
	const PgStart s = work.starts[1][slot + 1];
	if (s.block == 0 || s.block > list.per) return;
	const PgEntry e = work.entries[1][s.entry];
	const int more = (int)((e.blocks - s.block + list.per - 1) / list.per);
	const float *scratch = reinterpret_cast<const float *>(p.scratch);
	auto part = [&](int i) { return scratch + (int64_t)(i == 0 ? 2 * slot + 1 : 2 * (slot + i)) * PG_TILE * (DP + 2); };
	for (int x = threadIdx.x; x < 16 * (DP / 4); x += 128) {
		const int row = blockIdx.y * 16 + x / (DP / 4), col = x % (DP / 4) * 4;
		int token = 0, head = 0;
		if ((int64_t)e.tile * PG_TILE + row >= (int64_t)e.fresh * group || col >= p.dim) continue;
		const int sees = row_sees(e, row, group, token, head);
		float m = -INFINITY, l = 0.f;
		float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
		for (int i = 0; i <= more; ++i) {
			const float2 ml = __ldcg(reinterpret_cast<const float2 *>(part(i) + PG_TILE * DP) + row);
			const float4 y = __ldcg(reinterpret_cast<const float4 *>(part(i) + (int64_t)row * DP + col));
			const float top = fmaxf(m, ml.x), keep = m == -INFINITY ? 0.f : ex2(m - top), f = ml.x == -INFINITY ? 0.f : ex2(ml.x - top);
			m = top;
			l = fmaf(l, keep, ml.y * f);
			a = make_float4(fmaf(a.x, keep, y.x * f), fmaf(a.y, keep, y.y * f), fmaf(a.z, keep, y.z * f), fmaf(a.w, keep, y.w * f));
		}
		const float f = sees > 0 ? 1.f / l : 0.f;
		*reinterpret_cast<uint2 *>(reinterpret_cast<T *>(p.out) + ((int64_t)(e.row + token) * p.heads + s.kv * group + head) * p.dim + col) = make_uint2(pack2<T>(a.x * f, a.y * f), pack2<T>(a.z * f, a.w * f));
	}
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
	static_assert(smem <= 227 * 1024, "shared memory of a CTA");
	if (int rc = cuda_status(cudaFuncSetAttribute(tiles_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem))) return rc;
	tiles_kernel<T, DP><<<PG_TILE_SLOTS, TL_THREADS, smem, stream>>>(tmk, tmv, p, work);
	if (int rc = cuda_status(cudaGetLastError())) return rc;
	tile_join_kernel<T, DP><<<dim3(PG_TILE_SLOTS, PG_TILE / 16), 128, 0, stream>>>(p, work);
	return cuda_status(cudaGetLastError());
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
