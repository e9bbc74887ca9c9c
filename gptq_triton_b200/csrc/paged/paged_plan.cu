// Block tables, slot maps, positions and row offsets of a step from the request lengths, and the distribution of the attention's work.
//
// Every CTA scans the lengths of all requests into shared memory for itself (two sums per request: rows and pages taken), which is
// cheaper than a second launch or a barrier over the grid; then two or three lay out the attention's work, the others write pages and rows.
// A row finds its request by bisection in shared memory.  Table entries that are read (pages of old tokens) and written (pages taken
// now) are different ones, so the order of the CTAs does not matter, and a second run over the same inputs writes the same.
// The bytes are nothing; what counts is the chain launch - lengths - scan - table entry - store.
#include "paged.cuh"

namespace gptq {

namespace {

constexpr int PL_THREADS = 1024;

// sums that stop at a limit (associative for values of 0 .. limit; the sum of two limits of 2^30 is beyond an int)
__device__ __forceinline__ int add_to(int a, int b, int limit) { return (int)min((unsigned)a + (unsigned)b, (unsigned)limit); }
constexpr int PL_LIMIT = 1 << 30;

// exclusive scan over the CTA of two values per thread; returns the totals in (ta, tb).  s: 66 ints of shared memory
__device__ __forceinline__ void scan2(int &a, int &b, int limit_a, int limit_b, int &ta, int &tb, int *s) {
	const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
	int x = a, y = b;
#pragma unroll
	for (int d = 1; d < 32; d <<= 1) {
		const int u = __shfl_up_sync(0xffffffffu, x, d), v = __shfl_up_sync(0xffffffffu, y, d);
		if (lane >= d) {
			x = add_to(x, u, limit_a);
			y = add_to(y, v, limit_b);
		}
	}
	__syncthreads();
	if (lane == 31) {
		s[warp] = x;
		s[32 + warp] = y;
	}
	__syncthreads();
	int px = s[lane], py = s[32 + lane];          // (32 warps)
#pragma unroll
	for (int d = 1; d < 32; d <<= 1) {
		const int u = __shfl_up_sync(0xffffffffu, px, d), v = __shfl_up_sync(0xffffffffu, py, d);
		if (lane >= d) {
			px = add_to(px, u, limit_a);
			py = add_to(py, v, limit_b);
		}
	}
	ta = __shfl_sync(0xffffffffu, px, 31);
	tb = __shfl_sync(0xffffffffu, py, 31);
	const int bx = __shfl_sync(0xffffffffu, px, (warp + 31) & 31), by = __shfl_sync(0xffffffffu, py, (warp + 31) & 31);
	int ex = __shfl_up_sync(0xffffffffu, x, 1), ey = __shfl_up_sync(0xffffffffu, y, 1);
	if (lane == 0) ex = ey = 0;
	a = warp ? add_to(bx, ex, limit_a) : ex;
	b = warp ? add_to(by, ey, limit_b) : ey;
}

// the last i in [0, n) with v[i] <= x (v ascending, v[0] <= x)
__device__ __forceinline__ int find(const int *v, int n, int x) {
	int lo = 0, hi = n;
	while (hi - lo > 1) {
		const int mid = (lo + hi) >> 1;
		if (v[mid] <= x) lo = mid;
		else hi = mid;
	}
	return lo;
}

struct Lengths { int past, fresh, old, full; };

__device__ __forceinline__ Lengths lengths_of(const paged_plan_t &p, int r, int &bad) {
	Lengths l;
	l.past = __ldcg(p.past + r);
	l.fresh = __ldcg(p.fresh + r);
	if (l.past < 0 || l.past > PL_LIMIT || l.fresh < 0 || l.fresh > PL_LIMIT / 2) {
		bad |= PAGED_BAD_INDEX;
		l.past = min(max(l.past, 0), PL_LIMIT);
		l.fresh = min(max(l.fresh, 0), PL_LIMIT / 2);
	}
	l.old = (l.past + p.page - 1) / p.page;
	l.full = (l.past + l.fresh + p.page - 1) / p.page;
	if (p.pool == nullptr) l.full = l.old = 0;          // the table is complete
	return l;
}

// What the attention sees of a request is at most what its table can name.
__device__ __forceinline__ int length_seen(const paged_plan_t &p, const Lengths &l) { return (int)min((int64_t)l.past + l.fresh, min((int64_t)p.table_width * p.page, (int64_t)PL_LIMIT)); }

constexpr int PL_JOIN = 6;
constexpr int PL_KEEP = 4096;          // entries whose places and lengths are kept in shared memory
constexpr int PL_NEAR = 1024;          // ... and those that are kept there whole
constexpr int PL_PARTS = 2;            // CTAs that share the starts of the kernel for few rows

// (16 bytes at a time: word by word the stores of the lists take half of the kernel's time)
__device__ __forceinline__ void put(PgEntry *to, const PgEntry &x) {
	int4 *dst = reinterpret_cast<int4 *>(to);
	dst[0] = make_int4(x.request, x.tile, x.blocks, x.first);
	dst[1] = make_int4(x.row, x.fresh, x.len, x.seen);
}

// The work list of one kernel.  s_tiles [R + 1]: tiles of the requests before; s_len [R]; s_entry [PL_NEAR], s_first, s_sorted [PL_KEEP].
// The CTAs that share a list all form it, `part` 0 writes the entries, each its part of the starts.
__device__ void lay_out(const paged_plan_t &p, int kind, int part, int parts, const int *s_start, const int *s_len, const int *s_tiles, PgEntry *s_entry, int *s_first, int *s_sorted, int *s_scan,
						PgWork w) {
	const int tid = threadIdx.x, R = p.requests, tile_rows = kind ? PG_TILE : PG_ROWS, keys = kind ? PG_TILE_KEYS : PG_KEYS, group = p.heads / p.kv_heads;
	const int slots = kind ? PG_TILE_SLOTS : PG_SLOTS;
	int E = min(s_tiles[R], w.cap[kind]);
	int units = 0;
	for (int base = 0; base < E; base += PL_THREADS) {
		const int e = base + tid;
		PgEntry x = {};
		int n = 0, none = 0;
		if (e < E) {
			x.request = find(s_tiles, R, e);
			x.tile = e - s_tiles[x.request];
			x.row = s_start[x.request];
			x.fresh = s_start[x.request + 1] - x.row;
			x.len = s_len[x.request];
			const int last = (int)((min((int64_t)x.fresh * group, (int64_t)(x.tile + 1) * tile_rows) - 1) / group);
			x.seen = min(max(x.len - x.fresh + last + 1, 0), x.len);
			x.blocks = max((x.seen + keys - 1) / keys, 1);
			n = x.blocks + pg_begin(kind);
		}
		int total, unused;
		scan2(n, none, PL_LIMIT, PL_LIMIT, total, unused, s_scan);
		if (e < E) {
			x.first = add_to(units, n, PL_LIMIT);
			if (part == 0) put(w.entries[kind] + e, x);
			if (e < PL_NEAR) s_entry[e] = x;
			if (e < PL_KEEP) s_first[e] = x.first;
		}
		units = add_to(units, total, PL_LIMIT);
	}
	const bool over = units >= PL_LIMIT;                   // more keys than the lists count (10^9 blocks): an empty list
	if (over && tid == 0) atomicOr(p.status, PAGED_NO_ROOM);
	E = over ? 0 : E;
	units = over ? 0 : units;
	__syncthreads();
	if (E > PL_NEAR && part > 0) return;                   // (the other entries are in global memory, where part 0 has written them)
	if (E > PL_NEAR) parts = 1;
	auto blocks_of = [&](int e) { return e < PL_NEAR ? s_entry[e].blocks : w.entries[kind][e].blocks; };
	// A share is longer than what a job costs besides its blocks, so that no two slots begin at the same place, by one block (one token of 32
	// heads behind 100, us: 1 block 7.2, 2 8.0, 4 10.0; behind 2 100 11.7, 11.7, 11.8; 66 tokens of 28 heads over 4 behind 1 336, tiles: 1 block
	// 23.3, 2 30.1, 4 34.3).
	const int64_t total = (int64_t)units * p.kv_heads, per = max((total + slots - 1) / slots, (int64_t)(1 + pg_begin(kind)));
	int whole = 0;
	if (kind) {
		// Whole tiles, the longest first, dealt out to the slots forwards and backwards in turn, unless the longest slot would then work
		// PL_JOIN blocks longer than equal ranges take: that is what partial results and the kernel that joins them cost.
		__shared__ int s_most, s_span, s_hist[PL_THREADS];
		if (tid == 0) s_most = s_span = 0;
		s_hist[tid] = 0;
		__syncthreads();
		if (E <= PL_KEEP) {
			int most = 0;
			for (int e = tid; e < E; e += PL_THREADS) most = max(most, blocks_of(e));
			atomicMax(&s_most, most);
			__syncthreads();
			auto bucket = [&](int n) { return PL_THREADS - 1 - (int)((int64_t)n * (PL_THREADS - 1) / s_most); };
			for (int e = tid; e < E; e += PL_THREADS) atomicAdd(&s_hist[bucket(blocks_of(e))], 1);
			__syncthreads();
			int a = s_hist[tid], b = 0, ta, tb;
			scan2(a, b, PL_LIMIT, PL_LIMIT, ta, tb, s_scan);
			s_hist[tid] = a;
			__syncthreads();
			// (tiles of one length are in no particular order: which slot takes one changes no result)
			for (int e = tid; e < E; e += PL_THREADS) {
				const PgEntry x = e < PL_NEAR ? s_entry[e] : w.entries[1][e];
				const int at = atomicAdd(&s_hist[bucket(x.blocks)], 1);
				put(w.sorted + at, x);
				s_sorted[at] = x.blocks + pg_begin(1);
			}
		} else {
			for (int e = tid; e < E; e += PL_THREADS) put(w.sorted + e, w.entries[1][e]);
		}
		__syncthreads();
		const int64_t items = (int64_t)E * p.kv_heads;
		if (tid < slots) {
			int64_t sum = 0;
			for (int64_t turn = 0, i = tid; i < items; ++turn, i = turn & 1 ? (turn + 1) * slots - 1 - tid : turn * slots + tid) {
				const int at = items < PL_LIMIT ? (int)i / p.kv_heads : (int)(i / p.kv_heads);
				sum += E <= PL_KEEP ? s_sorted[at] : w.entries[1][at].blocks + pg_begin(1);
			}
			atomicMax(&s_span, (int)min(sum, (int64_t)PL_LIMIT));
		}
		__syncthreads();
		whole = s_span <= per + PL_JOIN;
	}
	if (tid == 0 && part == 0) {
		int4 *dst = reinterpret_cast<int4 *>(w.list + kind);          // (the counts of cuts follow)
		dst[0] = make_int4(E, whole, (int)(per & 0xffffffff), (int)(per >> 32));
		reinterpret_cast<int2 *>(dst)[2] = make_int2((int)(total & 0xffffffff), (int)(total >> 32));
		if (whole || parts == 1) w.list[kind].cuts[1] = 0;
		if (whole) w.list[kind].cuts[0] = 0;
	}
	if (whole) return;                                     // (nobody looks at the starts)
	int cuts = 0;
	for (int base = part * PL_THREADS; base <= slots; base += parts * PL_THREADS) {
		const int c = base + tid;
		const int64_t u = c * per;
		PgStart s = {-1, 0, 0, 0, {}};
		if (c <= slots && u < total) {
			const bool small = total < PL_LIMIT;
			const int x = small ? (int)u / p.kv_heads : (int)(u / p.kv_heads);
			int e;
			if (E <= PL_KEEP) {
				e = find(s_first, E, x);
			} else {
				int lo = 0, hi = E;
				while (hi - lo > 1) {
					const int mid = (lo + hi) >> 1;
					if (w.entries[kind][mid].first <= x) lo = mid;
					else hi = mid;
				}
				e = lo;
			}
			s.entry = e;
			s.job = e < PL_NEAR ? s_entry[e] : w.entries[kind][e];
			const int n = s.job.blocks + pg_begin(kind);
			const int64_t rest = u - (int64_t)s.job.first * p.kv_heads;
			s.kv = small ? (int)rest / n : (int)(rest / n);
			s.block = max((int)(rest - (int64_t)s.kv * n) - pg_begin(kind), 0);
		}
		if (c <= slots) {
			*reinterpret_cast<int4 *>(w.starts[kind] + c) = make_int4(s.entry, s.kv, s.block, 0);
			put(&w.starts[kind][c].job, s.job);
		}
		// the first cut of a job lies less than a share behind its begin
		int at = s.entry >= 0 && s.block > 0 && s.block <= per, none = 0, count, unused;
		const bool cut = at;
		scan2(at, none, PL_LIMIT, PL_LIMIT, count, unused, s_scan);
		if (cut) w.cuts[kind][part * slots + cuts + at] = c - 1;
		cuts += count;
	}
	if (tid == 0) w.list[kind].cuts[part] = cuts;
}

__global__ void __launch_bounds__(PL_THREADS) plan_kernel(const paged_plan_t p, int tiles) {
	extern __shared__ __align__(16) int pl_smem[];
	__shared__ int s_scan[64];
	int *s_start = pl_smem, *s_off = pl_smem + p.requests + 1;
	const int tid = threadIdx.x, R = p.requests;
	pdl_wait();
	pdl_trigger();
	int bad = 0, rows = 0, taken = 0;
	for (int base = 0; base < R; base += PL_THREADS) {
		const int r = base + tid;
		int a = 0, b = 0;
		if (r < R) {
			const Lengths l = lengths_of(p, r, bad);
			a = min(l.fresh, p.rows + 1);
			b = l.full - l.old;
		}
		int ta, tb;
		scan2(a, b, p.rows + 1, PL_LIMIT, ta, tb, s_scan);
		if (r < R) {
			s_start[r] = min(add_to(rows, a, p.rows + 1), p.rows);
			s_off[r] = add_to(taken, b, PL_LIMIT);
		}
		rows = add_to(rows, ta, p.rows + 1);
		taken = add_to(taken, tb, PL_LIMIT);
	}
	if (tid == 0) s_start[R] = min(rows, p.rows);
	if (rows > p.rows) bad |= PAGED_NO_ROOM;
	__syncthreads();
	const int head = p.pool ? __ldcg(p.head) : 0, used = s_start[R];
	if (p.pool && (head < 0 || head > p.pool_size || taken > p.pool_size - head)) bad |= head < 0 || head > p.pool_size ? PAGED_BAD_INDEX : PAGED_NO_ROOM;

	// the page that entry c of request r names; -1: none
	auto page_of = [&](int r, int c, int old) {
		int id;
		if (p.pool && c >= old) {
			const long long at = (long long)head + s_off[r] + (c - old);
			id = at >= 0 && at < p.pool_size ? __ldcg(p.pool + at) : -1;
		} else {
			id = c < p.table_width ? __ldcg(p.table + (int64_t)r * p.table_ld + c) : -1;
		}
		return id;
	};

	const int planners = PL_PARTS + (tiles ? 1 : 0);
	if ((int)blockIdx.x < planners) {
		for (int r = tid; r < R; r += PL_THREADS) {
			const Lengths l = lengths_of(p, r, bad);
			const int len = length_seen(p, l);
			s_off[r] = len;                                // (the pages taken before are of no use here)
			if (blockIdx.x == 0) {
				p.row_start[r] = s_start[r];
				p.lens[r] = len;
				if (len < l.past + l.fresh || l.fresh > p.max_fresh) bad |= PAGED_NO_ROOM;
			}
		}
		if (tid == 0 && blockIdx.x == 0) {
			p.row_start[R] = used;
			if (p.pool) *p.next_head = min(max(head, 0), p.pool_size) + min(taken, p.pool_size - min(max(head, 0), p.pool_size));
		}
		int *s_few = s_off + R + 1, *s_many = s_few + R + 1, *s_first = s_many + R + 1, *s_sorted = s_first + PL_KEEP;
		PgEntry *s_entry = reinterpret_cast<PgEntry *>(pl_smem + (4 * (R + 1) + 2 * PL_KEEP + 3) / 4 * 4);
		const int group = p.heads / p.kv_heads;
		int few = 0, many = 0;
		for (int base = 0; base < R; base += PL_THREADS) {
			const int r = base + tid;
			int a = 0, b = 0;
			if (r < R) {
				const int64_t n = (int64_t)(s_start[r + 1] - s_start[r]) * group;
				if (tiles && n > pg_few(group)) b = (int)((n + PG_TILE - 1) / PG_TILE);
				else a = (int)((n + PG_ROWS - 1) / PG_ROWS);
			}
			int ta, tb;
			scan2(a, b, PL_LIMIT, PL_LIMIT, ta, tb, s_scan);
			if (r < R) {
				s_few[r] = few + a;
				s_many[r] = many + b;
			}
			few += ta;
			many += tb;
		}
		if (tid == 0) {
			s_few[R] = few;
			s_many[R] = many;
		}
		__syncthreads();
		const PgWork w = pg_work(p.work, R, p.rows, p.heads, p.kv_heads);
		if (blockIdx.x < PL_PARTS) lay_out(p, 0, blockIdx.x, PL_PARTS, s_start, s_off, s_few, s_entry, s_first, s_sorted, s_scan, w);
		else lay_out(p, 1, 0, 1, s_start, s_off, s_many, s_entry, s_first, s_sorted, s_scan, w);
	} else {
		// pages that are taken now: a warp per request
		const int others = gridDim.x - planners, me = blockIdx.x - planners, warps = others * (PL_THREADS / 32), lane = tid & 31;
		if (p.pool)
			for (int r = me * (PL_THREADS / 32) + (tid >> 5); r < R; r += warps) {
				const Lengths l = lengths_of(p, r, bad);
				if (l.full > p.table_width) bad |= PAGED_NO_ROOM;
				for (int c = l.old + lane; c < min(l.full, p.table_width); c += 32) p.table[(int64_t)r * p.table_ld + c] = page_of(r, c, l.old);
			}
		for (int m = me * PL_THREADS + tid; m < p.rows; m += others * PL_THREADS) {
			int pos = 0;
			int64_t slot = -1;
			if (m < used) {
				const int r = find(s_start, R, m);
				const int past = min(max(__ldcg(p.past + r), 0), PL_LIMIT);
				pos = past + m - s_start[r];
				const int c = pos / p.page;
				const int id = page_of(r, c, (past + p.page - 1) / p.page);
				if (c >= p.table_width) bad |= PAGED_NO_ROOM;
				else if (id >= 0 && id < p.pages) slot = (int64_t)id * p.page + (pos - c * p.page);
				else bad |= PAGED_BAD_INDEX;
			}
			p.positions[m] = pos;
			p.slots[m] = slot;
		}
	}
	if (bad) atomicOr(p.status, bad);
}

}   // namespace

int pg_plan_launch(const paged_plan_t &p, int dtype, cudaStream_t stream) {
	const int tiles = p.pages > 0 && pg_tiles_serve(dtype, p.dim, p.page, p.max_fresh, p.heads, p.kv_heads);
	const size_t smem = (size_t)(4 * (p.requests + 1) + 2 * PL_KEEP + 3) * sizeof(int) + PL_NEAR * sizeof(PgEntry);
	static_assert((4 * (PAGED_MAX_REQUESTS + 1) + 2 * PL_KEEP) * sizeof(int) + PL_NEAR * sizeof(PgEntry) + 6144 <= 227 * 1024, "shared memory");
	const int fill = (int)((p.rows + (int64_t)PL_THREADS - 1) / PL_THREADS), ctas = PL_PARTS + (tiles ? 1 : 0) + (fill < 1 ? 1 : fill > 288 ? 288 : fill);
	return pg_launch(plan_kernel, dim3(ctas), PL_THREADS, smem, stream, p, tiles);
}

}   // namespace gptq
