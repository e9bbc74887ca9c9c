// Shared pieces of the paged-cache library: argument blocks, element access, the layout of the attention's work lists.
#pragma once

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
// of them: PG_ROWS rows for the kernel that streams keys past few rows, PG_TILE for the tensor-core kernel; a unit is one tile, one
// key head and a block of keys (PG_KEYS, PG_TILE_KEYS).  Entries list the tiles, units are counted entry by entry, key head by key head,
// keys ascending.  Slot c of a kernel works off units [c * per, (c + 1) * per): every slot has as much to do as any other, whatever the
// lengths, and a tile's keys may be spread over neighbouring slots, whose partial results are then joined.
constexpr int PG_ROWS = 16, PG_KEYS = 64, PG_SLOTS = 296;
constexpr int PG_TILE = 256, PG_TILE_KEYS = 128, PG_TILE_SLOTS = 148;

struct PgList {                        // of one of the two kernels; behind it in `work`: starts, entries, order
	int entries, per, total;            // total: units of all key heads
	int whole;                          // slots take whole tiles by `order` instead (tile kernel)
};
struct PgEntry { int request, tile, blocks, first; };          // blocks of keys that the tile sees; first: units of the entries before, per key head
struct PgStart { int entry, kv, block, pad; };                 // entry -1: nothing to do

struct PgWork {
	PgList *list;                       // [2]
	PgStart *starts[2];                 // [slots + 1]
	PgEntry *entries[2];
	int *order;
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
	at += 4 * (PG_SLOTS + 1);
	w.starts[1] = reinterpret_cast<PgStart *>(base + at);
	at += 4 * (PG_TILE_SLOTS + 1);
	w.entries[0] = reinterpret_cast<PgEntry *>(base + at);
	at += 4 * (int64_t)w.cap[0];
	w.entries[1] = reinterpret_cast<PgEntry *>(base + at);
	at += 4 * (int64_t)w.cap[1];
	w.order = base + at;
	w.ints = at + w.cap[1];
	return w;
}
// Whether the tensor-core kernel serves these sizes; which requests it then takes (more rows than PG_ROWS) is decided on the device.
inline bool pg_tiles_serve(int dtype, int dim, int page, int max_fresh, int heads, int kv_heads) {
	return false;
}

int pg_plan_launch(const paged_plan_t &p, int dtype, cudaStream_t stream);
int pg_append_launch(const paged_append_t &p, int dtype, cudaStream_t stream);
int pg_attend_simple(const paged_attention_t &p, int dtype, cudaStream_t stream);

}   // namespace gptq
