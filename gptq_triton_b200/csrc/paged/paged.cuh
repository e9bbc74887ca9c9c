// Shared pieces of the paged cache: argument blocks, element access, the layout of the attention's work lists.
#pragma once

#include <atomic>
#include <type_traits>
#include <utility>

#include <cuda_bf16.h>

#include "../common.cuh"
#include "../../../include/paged_b200.h"

namespace gptq {

typedef __nv_bfloat16 bf16;

enum { PG_BF16, PG_F32, PG_F16 };

template <typename T> struct PgElem;
template <> struct PgElem<float> {
	static __device__ __forceinline__ float get(float v) { return v; }
	static __device__ __forceinline__ float put(float v) { return v; }
};
template <> struct PgElem<bf16> {
	static __device__ __forceinline__ float get(bf16 v) { return __bfloat162float(v); }
	static __device__ __forceinline__ bf16 put(float v) { return __float2bfloat16_rn(v); }
};
template <> struct PgElem<__half> {
	static __device__ __forceinline__ float get(__half v) { return __half2float(v); }
	static __device__ __forceinline__ __half put(float v) { return __float2half_rn(v); }
};

// ---- how the attention's work is laid out (paged_plan_t.work) ---------------------------------------------------------------
// The rows of a request under one key head are its new tokens times the query heads of that key head, token-major.  A tile is a run
// of them: PG_ROWS rows for the kernel that streams keys past few rows, PG_TILE for the tensor-core kernel; its keys come in blocks of
// PG_KEYS, PG_TILE_KEYS.  A job is one tile under one key head.  Entries list the tiles; jobs follow one another entry by entry, key head
// by key head.  Laid end to end, each as long as its blocks and PG_BEGIN (what a job costs besides: queries, results), they are cut
// into equal lengths for the slots (warps of one kernel, CTAs of the other): whatever the lengths of the requests, no slot has more to
// do than another.  A cut inside a job leaves partial results, which are joined; slot c works from starts[c] to starts[c + 1].
constexpr int PG_ROWS = 16, PG_KEYS = 16, PG_SLOTS = 1184;
// Requests of up to so many rows per key head go to the kernel for few rows.  us, few rows / tiles (inside a graph, four sets of inputs in turn): 16 requests
// behind 300 to 5 000 tokens, 32 heads over 8, 20 rows 39 / 45, 32 rows 41 / 46, 40 rows 53 / 48, heads of 64 31 / 36, 32 / 36, 42 / 37; one request behind
// 3 000 13 / 20, 13 / 19, 19 / 20.  A key head of its own for every head is another matter, there is twice the cache to read for two tiles: 16 rows
// 79 / 138, 20 rows 135 / 137, 32 rows 140 / 113.
inline __host__ __device__ int pg_few(int group) { return group > 1 ? 32 : PG_ROWS; }
constexpr int PG_TILE = 256, PG_TILE_KEYS = 128, PG_TILE_SLOTS = 148;
inline __host__ __device__ int pg_begin(int kind) { return kind ? 2 : 1; }

struct PgList {                        // of one of the two kernels; behind it in `work`: starts, entries, sorted
	int entries;
	int whole;                          // slots take whole jobs in the order of `sorted` instead (tile kernel)
	int64_t per, total;                 // length of a slot's share, of all jobs
	int cuts[2];                        // slots in which a job begins that ends in a later one: how many, in the two parts of the list
};
struct alignas(16) PgEntry {
	int request, tile, blocks, first;   // blocks of keys that the tile sees; length of the entries before, per key head
	int row, fresh, len, seen;          // first row and new tokens of the request, its tokens, those that the tile's last row sees
};
struct alignas(16) PgStart {                       // entry -1: behind the last job
	int entry, kv, block, pad;
	PgEntry job;                        // entries[entry]
	__device__ bool in_job(int e, int k) const { return entry == e && kv == k; }
	__device__ bool before(int e, int k) const { return entry >= 0 && (entry < e || (entry == e && kv < k)); }          // its job comes before
};

// Everything that an earlier kernel wrote is read through L2: under programmatic dependent launch a line may have come to L1 before.
__device__ __forceinline__ PgList read_list(const PgList *p) {
	const int2 a = __ldcg(reinterpret_cast<const int2 *>(p));
	const long long b = __ldcg(reinterpret_cast<const long long *>(p) + 1), c = __ldcg(reinterpret_cast<const long long *>(p) + 2);
	const int2 d = __ldcg(reinterpret_cast<const int2 *>(p) + 3);
	return PgList{a.x, a.y, b, c, {d.x, d.y}};
}
__device__ __forceinline__ PgStart read_start(const PgStart *p) {
	const int4 a = __ldcg(reinterpret_cast<const int4 *>(p)), b = __ldcg(reinterpret_cast<const int4 *>(p) + 1), c = __ldcg(reinterpret_cast<const int4 *>(p) + 2);
	return PgStart{a.x, a.y, a.z, a.w, PgEntry{b.x, b.y, b.z, b.w, c.x, c.y, c.z, c.w}};
}
__device__ __forceinline__ PgEntry read_entry(const PgEntry *p) {
	const int4 a = __ldcg(reinterpret_cast<const int4 *>(p)), b = __ldcg(reinterpret_cast<const int4 *>(p) + 1);
	return PgEntry{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
}

struct PgWork {
	PgList *list;                       // [2]
	PgStart *starts[2];                 // [slots + 1]
	PgEntry *entries[2];
	PgEntry *sorted;                    // of the tile kernel, the longest first
	int *cuts[2];                       // [2 PG_SLOTS], [2 PG_TILE_SLOTS]: the slots of both parts
	int cap[2];
	int64_t ints;
};
inline __host__ __device__ PgWork pg_work(int32_t *base, int requests, int rows, int heads, int kv_heads) {
	PgWork w;
	const int64_t r = (int64_t)rows * (heads / kv_heads);
	w.cap[0] = (int)(r / PG_ROWS) + requests;
	w.cap[1] = (int)(r / PG_TILE) + requests;
	int64_t at = 16;
	w.list = reinterpret_cast<PgList *>(base);
	w.starts[0] = reinterpret_cast<PgStart *>(base + at);
	at += 12 * (PG_SLOTS + 1);
	w.starts[1] = reinterpret_cast<PgStart *>(base + at);
	at += 12 * (PG_TILE_SLOTS + 1);
	w.entries[0] = reinterpret_cast<PgEntry *>(base + at);
	at += 8 * (int64_t)w.cap[0];
	w.entries[1] = reinterpret_cast<PgEntry *>(base + at);
	at += 8 * (int64_t)w.cap[1];
	w.sorted = reinterpret_cast<PgEntry *>(base + at);
	at += 8 * (int64_t)w.cap[1];
	w.cuts[0] = base + at;
	at += 2 * PG_SLOTS;
	w.cuts[1] = base + at;
	w.ints = at + 2 * PG_TILE_SLOTS;
	return w;
}
// Whether the tensor-core kernel serves these sizes; which requests it then takes (more rows than PG_ROWS) is decided on the device.
inline bool pg_tiles_serve(int dtype, int dim, int page, int max_fresh, int heads, int kv_heads) {
	return dtype != PG_F32 && dim <= 128 && dim % 8 == 0 && (page == 8 || page == 16 || page == 32 || page == 64 || page % PG_TILE_KEYS == 0) && (int64_t)max_fresh * (heads / kv_heads) > pg_few(heads / kv_heads);
}

// cp.async of 16 bytes; `bytes` 0 writes zeros and reads nothing
__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void *src, int bytes) {
	asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ float ex2(float x) {
	float r;
	asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
	return r;
}
constexpr float PG_LOG2E = 1.44269504088896341f;

template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<bf16>(float lo, float hi) {
	__nv_bfloat162 a = __floats2bfloat162_rn(lo, hi);
	return *reinterpret_cast<uint32_t *>(&a);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
	__half2 a = __floats2half2_rn(lo, hi);
	return *reinterpret_cast<uint32_t *>(&a);
}
// D(16x8) += A(16x16, row) * B(16x8, col); fragment ownership as in mma16816
template <typename T> __device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma16<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) { mma16816(d, a[0], a[1], a[2], a[3], b0, b1); }
template <> __device__ __forceinline__ void mma16<bf16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
	asm volatile(
		"mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
		: "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
		: "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
	asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
	asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

// Launch with programmatic stream serialisation: every kernel here touches nothing that an earlier one wrote, and writes
// nothing, before its pdl_wait(), and triggers its successor behind it.  (The kernel for few rows is the exception, see there.)
int pg_smem_opt_in(const void *kernel);
template <typename... KArgs, typename... Args>
int pg_launch(void (*kernel)(KArgs...), dim3 grid, int threads, size_t smem, cudaStream_t stream, Args &&...args) {
	if (smem > 16 * 1024)          // (static shared memory comes on top)
		if (int rc = pg_smem_opt_in(reinterpret_cast<const void *>(kernel))) return rc;
	cudaLaunchConfig_t cfg = {};
	cfg.gridDim = grid;
	cfg.blockDim = dim3(threads);
	cfg.dynamicSmemBytes = smem;
	cfg.stream = stream;
	cudaLaunchAttribute attr;
	attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
	attr.val.programmaticStreamSerializationAllowed = 1;
	cfg.attrs = &attr;
	cfg.numAttrs = 1;
	return cuda_status(cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...));
}

int pg_plan_launch(const paged_plan_t &p, int dtype, cudaStream_t stream);
int pg_append_launch(const paged_append_t &p, int dtype, cudaStream_t stream);
int64_t pg_rows_scratch(const paged_attention_t &p);
int pg_rows_launch(const paged_attention_t &p, int dtype, bool beside, cudaStream_t stream);          // beside: the tile kernel runs too
int pg_join_launch(const paged_attention_t &p, int dtype, char *tile_scratch, cudaStream_t stream);          // of both kernels
int64_t pg_tiles_scratch(const paged_attention_t &p);
int pg_tiles_launch(const paged_attention_t &p, int dtype, char *scratch, cudaStream_t stream);

}   // namespace gptq
