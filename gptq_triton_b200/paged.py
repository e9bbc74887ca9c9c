"""Serving from a key / value cache in pages: requests of different lengths in one batch, memory that follows the lengths, prompts in
portions beside single tokens.

A cache is a pool of pages; one cache tensor is [pages, kv_heads, page, dim].  A request owns the pages that its row of the block table
names, in the order of its positions; position p lies in row p % page of page table[r, p // page].  Of a step with new[r] tokens for
request r behind past[r] cached ones

	plan = paged_plan(past, new, table, k_cache, rows, heads, pool=pool, head=head)      once: pages, positions, slots, the attention's work
	q = paged_append(q, k, v, k_cache, v_cache, plan, cos, sin)                           per layer: rotation, keys and values into their pages
	out = paged_attention(q, k_cache, v_cache, plan)                                      per layer

Rows are the new tokens, request after request.  Lengths stay on the device: a captured graph serves whatever they are at its replay.
The operators raise on arguments that the host can judge; what only the device sees (a page that does not exist, no pages left) sets
the status word (_lib.kernel_status(): 4, 8, 16) and touches no memory that is not its own; the results of such a step are not to be used.
There is no gradient.

Any page and any head size that is a multiple of 8 is served, but chunks run on tensor memory (several times faster) only in 16 bits, in heads
of up to 128, and in pages of 8, 16, 32, 64 or a multiple of 128 rows.
"""
from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass
from typing import Optional

import torch

from . import _paged
from ._lib import GptqB200Error, ptr, require_cuda, stream_ptr


@dataclass
class PagedPlan:
	"""What a step's operators share.  `serves`: heads, kv_heads, page, pages, dim, dtype of the layers that it was made for."""
	table: torch.Tensor           # int32 [requests, width]: the caller's block table
	row_start: torch.Tensor       # int32 [requests + 1]: first row of every request, and the number of rows in use
	lens: torch.Tensor            # int32 [requests]: cached tokens, the new ones included
	positions: torch.Tensor       # int32 [rows]; 0 behind the last row in use
	slots: torch.Tensor           # int64 [rows]: page * page_size + row of the page; -1 behind the last row in use
	head: Optional[torch.Tensor]  # int32 [1]: place in the pool behind the pages taken
	work: torch.Tensor            # the attention's distribution of work
	rows: int
	max_new: int
	serves: tuple
	native: tuple = ()            # the same for native code: type code, heads, kv_heads, page, pages, dim, rows, address of the status word


def _int32(t: torch.Tensor, name: str, dims: int, device):
	if t.dtype != torch.int32 or t.dim() != dims or t.device != device or (t.numel() and t.stride(-1) != 1):
		raise ValueError(f'{name} must be an int32 tensor of {dims} dimension(s) with neighbouring entries on {device}, got {t.dtype} {tuple(t.shape)} on {t.device}')


def _cache(t: torch.Tensor, name: str):
	if t.dim() != 4 or t.dtype not in _paged.DTYPE_CODE:
		raise ValueError(f'{name} must be [pages, kv_heads, page, dim] in fp16, bf16 or fp32, got {t.dtype} {tuple(t.shape)}')
	if t.numel() and (t.stride(3) != 1 or t.stride(2) != t.shape[3]):
		raise ValueError(f'{name}: the rows of a page must lie one behind the other (strides {t.stride()})')


class _On:
	"""Makes `device` the current one for a launch, where it is not."""

	def __init__(self, device):
		self.guard = None if device.index is None or device.index == torch.cuda.current_device() else torch.cuda.device(device)

	def __enter__(self):
		if self.guard is not None:
			self.guard.__enter__()

	def __exit__(self, *e):
		if self.guard is not None:
			self.guard.__exit__(*e)


def paged_plan(past: torch.Tensor, new: torch.Tensor, table: torch.Tensor, cache: torch.Tensor, rows: int, heads: int, pool: Optional[torch.Tensor] = None,
			   head: Optional[torch.Tensor] = None, max_new: Optional[int] = None) -> PagedPlan:
	"""The plan of a step in one launch.

	past, new: int32 [requests], tokens in the cache and new ones (0: the request waits).  table: int32 [requests, width]; with
	`pool` (int32, numbers of free pages) and `head` (int32 [1], place of the first one that is still free) the entries of the pages
	that the new tokens need are written into it in place, requests in order; plan.head is the place behind them (a tensor of its own,
	so the same call again gives the same plan).  Without, the table must name all pages.
	cache: a key cache tensor of the layers, for its sizes and type.  rows: rows of q, k and v, at least the sum of `new`; rows left over
	get slot -1.  heads: query heads.  max_new: no request has more new tokens (default: rows), which spares launches and time; one
	that has sets status 8.
	"""
	if cache.is_cuda:
		dt = cache.dtype
		code, most, status = _paged.DTYPE_CODE.get(dt), rows if max_new is None else min(max_new, rows), _paged.status_ptr(cache.get_device())
		served = _paged.native().paged_plan(past, new, table, cache, code, rows, heads, pool, head, most, status)
		if served is not None:
			pages, kv_heads, page, dim = cache.shape
			return PagedPlan(table, *served, rows, most, (heads, kv_heads, page, pages, dim, dt), (code, heads, kv_heads, page, pages, dim, rows, status))
	require_cuda(past, new, table, cache, pool, head)
	dev = cache.device
	_cache(cache, 'cache')
	pages, kv_heads, page, dim = cache.shape
	_int32(past, 'past', 1, dev)
	_int32(new, 'new', 1, dev)
	_int32(table, 'table', 2, dev)
	R, rows, heads = past.numel(), int(rows), int(heads)
	if new.numel() != R or table.shape[0] != R or R > _paged.MAX_REQUESTS:
		raise ValueError(f'past, new and table must speak of the same requests, at most {_paged.MAX_REQUESTS}: {R}, {new.numel()}, {table.shape[0]}')
	if rows < 0 or rows >= 1 << 30 or kv_heads < 1 or heads < 1 or heads % kv_heads or heads > 65535 or not 1 <= page <= _paged.MAX_PAGE or dim < 1 or table.shape[1] < 1:
		raise ValueError(f'paged_plan: {rows} rows, {heads} heads over {kv_heads} key heads, pages of {page} rows of {dim}, {table.shape[1]} table columns')
	if R > 1 and table.stride(0) < table.shape[1]:
		raise ValueError(f'table: rows that overlap (strides {table.stride()})')
	if (pool is None) != (head is None):
		raise ValueError('pool and head go together')
	if pool is not None:
		_int32(pool, 'pool', 1, dev)
		_int32(head, 'head', 1, dev)
		if head.numel() != 1:
			raise ValueError('head is one number')
	max_new = rows if max_new is None else min(int(max_new), rows)
	if max_new < 0:
		raise ValueError('max_new must not be negative')
	lib = _paged.lib()
	ints = R + 1 + R + rows + 1
	words = lib.paged_work_ints(R, rows, heads, kv_heads)
	if words < 0:
		raise ValueError('paged_plan: sizes out of range')
	# one allocation: slots first (8 bytes), then work (16-byte groups), then the rest
	at = 2 * rows + (2 * rows & 2)
	buf = torch.empty(at + words + ints, dtype=torch.int32, device=dev)
	slots, work = buf[:2 * rows].view(torch.int64), buf[at:at + words]
	row_start, lens, positions, nxt = buf[at + words:].split([R + 1, R, rows, 1])
	a = _paged.Plan()
	a.requests, a.rows, a.table_width, a.page, a.pages, a.pool_size = R, rows, table.shape[1], page, pages, 0 if pool is None else pool.numel()
	a.table_ld = max(table.stride(0), table.shape[1])
	a.past, a.fresh, a.table, a.pool, a.head = ptr(past), ptr(new), ptr(table), ptr(pool), ptr(head)
	a.next_head, a.row_start, a.lens, a.positions, a.slots = ptr(nxt) if pool is not None else None, ptr(row_start), ptr(lens), ptr(positions), ptr(slots)
	a.heads, a.kv_heads, a.dim, a.max_fresh, a.work, a.status = heads, kv_heads, dim, max_new, ptr(work), _paged.status_ptr(dev.index)
	with _On(dev):
		_paged.check(lib.paged_plan(ctypes.byref(a), _paged.DTYPE_CODE[cache.dtype], stream_ptr(dev)), 'paged_plan')
	return PagedPlan(table, row_start, lens, positions, slots, None if pool is None else nxt, work, rows, max_new, (heads, kv_heads, page, pages, dim, cache.dtype),
					 (_paged.DTYPE_CODE[cache.dtype], heads, kv_heads, page, pages, dim, rows, _paged.status_ptr(dev.index)))


def _caches(k_cache, v_cache, plan: PagedPlan, what: str):
	_cache(k_cache, 'k_cache')
	_cache(v_cache, 'v_cache')
	pages, kv_heads, page, dim = k_cache.shape
	if k_cache.shape != v_cache.shape or k_cache.dtype != v_cache.dtype or plan.serves[1:] != (kv_heads, page, pages, dim, k_cache.dtype):
		raise ValueError(f'{what}: k_cache {k_cache.dtype} {tuple(k_cache.shape)} and v_cache {v_cache.dtype} {tuple(v_cache.shape)}, the plan was made for {plan.serves}')


def _rows(t: torch.Tensor, name: str, plan: PagedPlan, heads: int):
	if t.dim() != 3 or t.shape != (plan.rows, heads, plan.serves[4]) or t.dtype != plan.serves[5] or t.device != plan.work.device:
		raise ValueError(f'{name} must be [{plan.rows}, {heads}, {plan.serves[4]}] {plan.serves[5]} on {plan.work.device}, got {tuple(t.shape)} {t.dtype} on {t.device}')
	if t.numel() and t.stride(2) != 1:
		raise ValueError(f'{name}: the entries of a head must be neighbours (strides {t.stride()})')


def _out(out: Optional[torch.Tensor], q: torch.Tensor) -> torch.Tensor:
	if out is None:
		return torch.empty(q.shape, dtype=q.dtype, device=q.device)
	if out.shape != q.shape or out.dtype != q.dtype or out.device != q.device or not out.is_contiguous():
		raise ValueError(f'out must be contiguous {tuple(q.shape)} {q.dtype} on {q.device}')
	return out


def paged_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, plan: PagedPlan, cos: Optional[torch.Tensor] = None,
				 sin: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
	"""Rotates the new queries and keys by their positions and stores key and value rows in their pages; returns the rotated queries.

	q: [rows, heads, dim], k, v: [rows, kv_heads, dim], any strides with neighbouring entries (columns of a fused projection).  cos, sin:
	[positions, rot] in the type of q, rotate-half convention as rope_tables() gives them; rot < dim turns the first entries of a head
	only; without tables nothing is turned.  Rows with slot -1 are not stored; a position outside the tables sets status 4, its row is
	turned as position 0 and not stored.  Slots are distinct unless the block table gives one page to two requests that write to it: which row
	such a place then holds is open.  `out` may be q itself (contiguous).
	"""
	served = _paged.native().paged_append(q, k, v, k_cache, v_cache, cos, sin, out, plan.positions, plan.slots, *plan.native)
	if served is not None:
		return served
	heads, kv_heads, page, pages, dim, dt = plan.serves
	require_cuda(q, k, v, k_cache, v_cache, cos, sin, out)
	_caches(k_cache, v_cache, plan, 'paged_append')
	_rows(q, 'q', plan, heads)
	_rows(k, 'k', plan, kv_heads)
	_rows(v, 'v', plan, kv_heads)
	dev = q.device
	if k_cache.device != dev or v_cache.device != dev:
		raise ValueError('paged_append: caches and rows must be on one device')
	if (cos is None) != (sin is None):
		raise ValueError('cos and sin go together')
	a = _paged.Append()
	if cos is not None:
		if cos.dim() != 2 or cos.shape != sin.shape or cos.dtype != dt or sin.dtype != dt or cos.device != dev or sin.device != dev or not (cos.is_contiguous() and sin.is_contiguous()) \
				or cos.shape[1] > dim or cos.shape[1] % 2 or cos.shape[0] < 1:
			raise ValueError(f'cos and sin must be contiguous [positions, rot] {dt} on {dev} with an even rot of at most {dim}: {tuple(cos.shape)} {cos.dtype}, {tuple(sin.shape)} {sin.dtype}')
		a.rot, a.max_pos, a.cos_t, a.sin_t = cos.shape[1], cos.shape[0], ptr(cos), ptr(sin)
	res = _out(out, q)
	a.rows, a.heads, a.kv_heads, a.dim, a.page, a.pages = plan.rows, heads, kv_heads, dim, page, pages
	a.q, a.k, a.v = ptr(q), ptr(k), ptr(v)
	a.q_row, a.q_head, a.k_row, a.k_head, a.v_row, a.v_head = q.stride(0), q.stride(1), k.stride(0), k.stride(1), v.stride(0), v.stride(1)
	a.positions, a.slots, a.q_out, a.k_cache, a.v_cache = ptr(plan.positions), ptr(plan.slots), ptr(res), ptr(k_cache), ptr(v_cache)
	a.k_page, a.k_kv, a.v_page, a.v_kv, a.status = k_cache.stride(0), k_cache.stride(1), v_cache.stride(0), v_cache.stride(1), _paged.status_ptr(dev.index)
	with _On(dev):
		_paged.check(_paged.lib().paged_append(ctypes.byref(a), _paged.DTYPE_CODE[dt], stream_ptr(dev)), 'paged_append')
	return res


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, plan: PagedPlan, scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
	"""softmax(scale q k^T) v of every new token over the positions up to its own, [rows, heads, dim].

	q: [rows, heads, dim] (rotated); query head h reads key head h // (heads // kv_heads).  scale: positive, default 1 / sqrt(dim).
	Rows behind the last one in use are left as they are (`out`, which may be q itself) or have no particular value.  Values of positions
	behind a request's last one do not count, whatever the pages hold there.  A value of a new token that is not finite can make earlier
	rows of the same step and request NaN (a weight of zero times it), as it does in the formula's products.
	"""
	heads, kv_heads, page, pages, dim, dt = plan.serves
	scale = 1.0 / math.sqrt(dim) if scale is None else float(scale)
	served = _paged.native().paged_attention(q, k_cache, v_cache, out, scale, plan.table, plan.row_start, plan.lens, plan.work, plan.max_new, *plan.native)
	if served is not None:
		return served
	require_cuda(q, k_cache, v_cache, out)
	_caches(k_cache, v_cache, plan, 'paged_attention')
	_rows(q, 'q', plan, heads)
	dev = q.device
	if k_cache.device != dev or v_cache.device != dev:
		raise ValueError('paged_attention: caches and queries must be on one device')
	if dim % 8 or dim > _paged.MAX_DIM:
		raise ValueError(f'paged_attention serves head sizes that are multiples of 8 up to {_paged.MAX_DIM}, not {dim}')
	if not (0.0 < scale < math.inf):
		raise ValueError('scale must be positive and finite')
	res = _out(out, q)
	lib, code = _paged.lib(), _paged.DTYPE_CODE[dt]
	a = _paged.Attention()
	a.requests, a.rows, a.heads, a.kv_heads, a.dim, a.page, a.pages, a.table_width, a.max_fresh = plan.lens.numel(), plan.rows, heads, kv_heads, dim, page, pages, plan.table.shape[1], plan.max_new
	a.table_ld, a.scale = max(plan.table.stride(0), plan.table.shape[1]), scale
	a.q, a.q_row, a.q_head, a.k_cache, a.v_cache = ptr(q), q.stride(0), q.stride(1), ptr(k_cache), ptr(v_cache)
	a.k_page, a.k_kv, a.v_page, a.v_kv = k_cache.stride(0), k_cache.stride(1), v_cache.stride(0), v_cache.stride(1)
	a.table, a.row_start, a.lens, a.work, a.out, a.status = ptr(plan.table), ptr(plan.row_start), ptr(plan.lens), ptr(plan.work), ptr(res), _paged.status_ptr(dev.index)
	need = lib.paged_attention_scratch(ctypes.byref(a), code)
	scratch = torch.empty(max(need, 16), dtype=torch.uint8, device=dev)
	a.scratch, a.scratch_bytes = ptr(scratch), scratch.numel()
	with _On(dev):
		_paged.check(lib.paged_attention(ctypes.byref(a), code, stream_ptr(dev)), 'paged_attention')
	return res
