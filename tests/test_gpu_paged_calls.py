"""Calls of the paged operators: refusals, native code and ctypes side by side, captured graphs over other lengths, streams, the three
operators as a step uses them, pages that do not exist."""
import random

import pytest
import torch

import gptq_triton_b200 as G
from gptq_triton_b200 import _lib, _paged
from oracle import paged_oracle as O
from paged_cases import DTYPES, Step, bound, ceil
from test_gpu_paged import DEV, healthy, make_plan, status, tables      # noqa: F401 (healthy: status is zero behind every test)

pytestmark = pytest.mark.gpu


@pytest.fixture
def step():
	return Step([20, 0, 130], [1, 40, 3], 8, 2, 64, 16, 'fp16', pad=2)


def on_gpu(s):
	k, v = s.k.to(DEV), s.v.to(DEV)
	return k, v, *(t for t in s.parts(s.qkv.to(DEV)))


def test_refusals_of_the_plan(step):
	k = step.k.to(DEV)
	i32 = step.ints
	ok = dict(past=i32(step.past), new=i32(step.new), table=i32(step.table), cache=k, rows=step.rows, heads=8)
	G.paged_plan(**ok)
	pool, head = i32([0, 1]), i32([0])
	for change, error in ((dict(past=i32(step.past).long()), ValueError), (dict(new=i32(step.new[:2])), ValueError), (dict(table=i32(step.table)[:2]), ValueError), (dict(table=i32(step.table).t()), ValueError),
						  (dict(heads=7), ValueError), (dict(heads=0), ValueError), (dict(rows=-1), ValueError), (dict(cache=k[0]), ValueError), (dict(cache=k.double()), ValueError),
						  (dict(cache=k.transpose(2, 3)), ValueError), (dict(cache=k[..., ::2]), ValueError), (dict(pool=pool), ValueError), (dict(head=head), ValueError), (dict(pool=pool, head=i32([0, 1])), ValueError),
						  (dict(pool=pool.long(), head=head), ValueError), (dict(max_new=-1), ValueError), (dict(past=torch.zeros(3, dtype=torch.int32)), _lib.GptqB200Error),
						  (dict(past=i32([0] * 8193), new=i32([0] * 8193), table=i32([[0]] * 8193)), ValueError), (dict(past=i32(step.past * 2)[::2]), ValueError), (dict(table=i32(step.table)[:1].expand(3, -1)), ValueError)):
		with pytest.raises(error):
			G.paged_plan(**{**ok, **change})


def test_refusals_of_append_and_attention(step):
	k, v, q, kn, vn = on_gpu(step)
	plan = make_plan(step, k)
	cos, sin = (t.to(DEV) for t in tables(64, 200, step.dtype))
	append = lambda **kw: G.paged_append(**{**dict(q=q, k=kn, v=vn, k_cache=k, v_cache=v, plan=plan, cos=cos, sin=sin), **kw})
	attend = lambda **kw: G.paged_attention(**{**dict(q=q, k_cache=k, v_cache=v, plan=plan), **kw})
	append(), attend()
	for kw in (dict(q=q[:-1]), dict(q=q[:, :4]), dict(q=q.bfloat16()), dict(q=q.transpose(1, 2)), dict(k=q), dict(v=vn[:, :1]), dict(k_cache=k[:-1]), dict(v_cache=v.float()), dict(cos=None), dict(cos=cos[:, :32]),
			   dict(cos=cos.float(), sin=sin.float()), dict(cos=cos[:0], sin=sin[:0]), dict(cos=cos[:, :63], sin=sin[:, :63]), dict(out=q), dict(out=torch.empty_like(q)[:-1]), dict(k_cache=k.transpose(0, 1))):
		with pytest.raises(ValueError):
			append(**kw)
	for kw in (dict(q=q[:-1]), dict(q=q.float()), dict(k_cache=k.bfloat16(), v_cache=v.bfloat16()), dict(v_cache=v[:-1]), dict(scale=0.0), dict(scale=-1.0), dict(scale=float('nan')), dict(scale=float('inf')), dict(out=q),
			   dict(k_cache=k[:1].expand(k.shape[0], -1, -1, -1)), dict(v_cache=v[:, :1].expand(-1, 2, -1, -1))):
		with pytest.raises(ValueError):
			attend(**kw)
	with pytest.raises(_lib.GptqB200Error):
		attend(q=q.cpu())
	odd = torch.empty((k.shape[0], 2, 16, 12), dtype=torch.float16, device=DEV)          # heads of 12: rows do not start on 16 bytes
	s = Step([3], [2], 2, 2, 12, 16, 'fp16', spare=k.shape[0] - 1)
	with pytest.raises(ValueError):
		G.paged_attention(s.parts(s.qkv.to(DEV))[0], odd, odd, make_plan(s, odd))
	wide = torch.empty((3, 2, 16, 264), dtype=torch.float16, device=DEV)
	s = Step([3], [2], 2, 2, 264, 16, 'fp16', spare=2)
	with pytest.raises(ValueError):
		G.paged_attention(s.parts(s.qkv.to(DEV))[0], wide, wide, make_plan(s, wide))


@pytest.mark.parametrize('dtype', list(DTYPES))
def test_native_code_and_ctypes_agree(monkeypatch, dtype):
	s = Step([20, 0, 130, 0], [1, 40, 3, 0], 8, 2, 64, 16, dtype, pad=2)
	k, v, q, kn, vn = on_gpu(s)
	cos, sin = (t.to(DEV) for t in tables(64, 200, s.dtype))

	def run():
		table = s.ints(s.table)
		table[1, 1:] = -1          # dealt out again from a pool
		pool = s.ints([9, *s.table[1][1:3], 0, 0])
		plan = G.paged_plan(s.ints(s.past), s.ints([1, 40, 3, 0]), table, k, s.rows, 8, max_new=40)
		dealt = G.paged_plan(s.ints([0, 16]), s.ints([0, 24]), table[:2], k, 30, 8, pool=pool, head=s.ints([1]))
		kc, vc = k.clone(), v.clone()
		out = G.paged_append(q, kn, vn, kc, vc, plan, cos, sin)
		return [table, plan.row_start, plan.lens, plan.positions, plan.slots, dealt.head, dealt.slots, dealt.row_start, out, kc, vc, G.paged_append(q, kn, vn, kc, vc, plan, out=torch.empty_like(out)),
				G.paged_attention(out, k, v, plan), G.paged_attention(q, k, v, plan, scale=0.3)]
	served = []
	native = _paged.native()
	assert native is not _paged._Ctypes

	class Counts:
		pass
	for name in ('paged_plan', 'paged_append', 'paged_attention'):
		setattr(Counts, name, staticmethod(lambda *a, f=getattr(native, name): served.append(f(*a)) or served[-1]))
	monkeypatch.setattr(_paged, '_native', Counts)
	new = run()
	assert len(served) == 6 and all(x is not None for x in served)
	monkeypatch.setattr(_paged, '_native', _paged._Ctypes)
	old = run()
	status()
	used = sum(s.new)
	for i, (a, b) in enumerate(zip(new, old)):
		a, b = (t[:used] if t.dim() == 3 and i >= 12 else t for t in (a, b))          # (attention: rows behind the last have no value)
		assert a.dtype == b.dtype and a.shape == b.shape and torch.equal(a.nan_to_num(7.0) if a.is_floating_point() else a, b.nan_to_num(7.0) if b.is_floating_point() else b), i


@pytest.mark.parametrize('dtype,heads,kv_heads,dim,page', [('fp16', 32, 8, 128, 16), ('bf16', 8, 8, 64, 32), ('fp32', 6, 2, 96, 24), ('bf16', 12, 4, 96, 128), ('fp16', 4, 1, 80, 7)])
def test_steps_of_a_server(dtype, heads, kv_heads, dim, page):
	"""Plan, append and attention over several steps from an empty cache: portions of prompts, single tokens, requests that wait; pages from a
	pool.  Against the restatement, which keeps its own cache."""
	rng = random.Random(dim)
	steps = [[30, 0, 7, 1], [40, 0, 1, 1], [1, 5, 1, 1], [1, 1, 0, 200], [1, 1, 1, 1]]
	R, past = 4, [0] * 4
	total = sum(ceil(sum(s[r] for s in steps), page) for r in range(R)) + 2
	pool = list(range(total))
	rng.shuffle(pool)
	width = max(ceil(sum(s[r] for s in steps), page) for r in range(R))
	k, v = (torch.full((total, kv_heads, page, dim), float('nan'), dtype=DTYPES[dtype], device=DEV) for _ in range(2))
	hk, hv = k.cpu(), v.cpu()
	i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
	d_table, d_pool, d_head = torch.full((R, width), -1, dtype=torch.int32, device=DEV), i32(pool), i32([0])
	table, head = [[-1] * width for _ in range(R)], 0
	cos, sin = tables(dim, 400, DTYPES[dtype])
	for n, new in enumerate(steps):
		pad = n % 3
		s = Step([0] * R, new, heads, kv_heads, dim, page, dtype, seed=n, pad=pad)          # (for its rows)
		start, lens, pos, slots, head = O.plan(past, new, table, page, s.rows, pool, head)
		plan = G.paged_plan(i32(past), i32(new), d_table, k, s.rows, heads, pool=d_pool, head=d_head, max_new=max(new))
		d_head = plan.head
		q, kn, vn = s.parts(s.qkv.to(DEV))
		q = G.paged_append(q, kn, vn, k, v, plan, cos.to(DEV), sin.to(DEV))
		out = G.paged_attention(q, k, v, plan)
		assert plan.slots.tolist() == slots and d_table.tolist() == table and int(d_head) == head
		# the cache that the attention read, kept by the restatement from the rows that the append made
		p = torch.tensor(slots[:start[-1]]) // page
		r = torch.tensor(slots[:start[-1]]) % page
		kc = k.cpu()
		rotated = O.rotate(s.parts()[1][:start[-1]], cos[torch.tensor(pos[:start[-1]])], sin[torch.tensor(pos[:start[-1]])])
		u = torch.finfo(DTYPES[dtype]).eps / 2
		assert ((kc[p, :, r].double() - rotated).abs() <= u * 1.01 * rotated.abs() + 2.0 ** -22 * 6 + 2.0 ** -25).all()
		hk[p, :, r], hv[p, :, r] = kc[p, :, r], s.parts()[2][:start[-1]]
		assert torch.equal(hk.nan_to_num(9.0), kc.nan_to_num(9.0)) and torch.equal(hv.nan_to_num(9.0), v.cpu().nan_to_num(9.0))
		want, absolute, score = O.attention(q.cpu(), hk, hv, table, start, lens)
		error = (out.cpu()[:start[-1]].double() - want).abs()
		assert (error <= bound(want, absolute, score, dim, max(lens), DTYPES[dtype])).all()
		past = lens


def test_captured_steps_follow_the_lengths():
	"""One captured step of plan, append and attention replayed for other lengths, while another graph of the same sizes is replayed on
	another stream: each owns its plan and its partial results."""
	R, heads, kv_heads, dim, page = 5, 8, 2, 128, 16
	cases = [[100, 3, 700, 0, 33], [1, 2000, 16, 15, 64], [0, 0, 0, 0, 0]]
	steps = [Step(past, [1] * R, heads, kv_heads, dim, page, 'fp16', seed=i, spare=0, fill=0.0) for i, past in enumerate(cases)]
	pages, width = max(s.pages for s in steps), max(s.width for s in steps)

	class Graph:
		def __init__(self):
			self.past, self.new, self.table = (torch.zeros(s, dtype=torch.int32, device=DEV) for s in ((R,), (R,), (R, width)))
			self.k, self.v = (torch.zeros((pages, kv_heads, page, dim), dtype=torch.float16, device=DEV) for _ in range(2))
			self.q = torch.zeros((R, heads, dim), dtype=torch.float16, device=DEV)
			self.g, self.stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
			self.new.fill_(1)
			torch.cuda.synchronize()
			with torch.cuda.stream(self.stream):
				self.body()
				self.stream.synchronize()
				with torch.cuda.graph(self.g, stream=self.stream):
					self.out = self.body()

		def body(self):
			plan = G.paged_plan(self.past, self.new, self.table, self.k, R, heads, max_new=1)
			return G.paged_attention(self.q, self.k, self.v, plan)

		def load(self, s):
			self.past.copy_(s.ints(s.past))
			self.table.zero_()
			self.table[:, :s.width] = s.ints(s.table)
			self.k[:s.pages] = s.k.to(DEV)
			self.v[:s.pages] = s.v.to(DEV)
			self.q.copy_(s.parts(s.qkv.to(DEV))[0])

	graphs = [Graph(), Graph()]
	for first, second in ((0, 1), (1, 2), (2, 0)):
		for g, i in zip(graphs, (first, second)):
			g.load(steps[i])
		torch.cuda.synchronize()
		for _ in range(3):
			for g in graphs:
				with torch.cuda.stream(g.stream):
					g.g.replay()
		torch.cuda.synchronize()
		for g, i in zip(graphs, (first, second)):
			s = steps[i]
			lens = [p + 1 for p in s.past]
			want, absolute, score = O.attention(s.parts()[0], s.k, s.v, s.table, list(range(R + 1)), lens)
			error = (g.out.cpu().double() - want).abs()
			assert (error <= bound(want, absolute, score, dim, max(lens), torch.float16)).all(), i
	status()


@pytest.mark.parametrize('new', [1, 100])
def test_cache_of_more_than_two_thousand_million_entries(new):
	"""Pages whose first entry lies beyond 2^31: rows that are stored and read there."""
	heads, dim, page = 4, 128, 16
	pages = (2 ** 31 + 2 ** 28) // (heads * page * dim)
	s = Step([40], [new], heads, heads, dim, page, 'fp16', filled=False, fill=0.0)
	k, v = (torch.empty((pages, heads, page, dim), dtype=torch.float16, device=DEV) for _ in range(2))
	used = -(-(40 + new) // page)
	own = [pages - 1 - 3 * i for i in range(used)]
	for i, mine in enumerate(own):
		k[mine], v[mine] = s.k[s.table[0][i]].to(DEV), s.v[s.table[0][i]].to(DEV)
	s.table = [own]
	q, kn, vn = s.parts(s.qkv.to(DEV))
	plan = G.paged_plan(s.ints([40]), s.ints([new]), s.ints([own]), k, s.rows, heads)
	assert plan.slots.tolist() == [own[p // page] * page + p % page for p in range(40, 40 + new)]
	G.paged_append(q, kn, vn, k, v, plan)
	out = G.paged_attention(q, k, v, plan)
	small_k, small_v = (torch.stack([t[m] for m in own]).cpu() for t in (k, v))
	j = torch.arange(40, 40 + new)
	assert torch.equal(small_k[j // page, :, j % page], s.parts()[1]) and torch.equal(small_v[j // page, :, j % page], s.parts()[2])
	want, absolute, score = O.attention(s.parts()[0], small_k, small_v, [list(range(used))], [0, new], [40 + new])
	assert ((out.cpu().double() - want).abs() <= bound(want, absolute, score, dim, 40 + new, torch.float16)).all()


@pytest.mark.parametrize('new', [[1, 1], [40, 70]])
def test_results_in_the_place_of_the_queries(new):
	s = Step([300, 20], new, 8, 2, 64, 16, 'bf16')
	k, v = s.k.to(DEV), s.v.to(DEV)
	q = s.parts(s.qkv.to(DEV))[0].contiguous()
	plan = make_plan(s, k)
	want = G.paged_attention(q, k, v, plan)
	assert G.paged_attention(q, k, v, plan, out=q) is q and torch.equal(q, want)


def test_a_page_in_two_tables():
	"""Requests that share the pages of a common beginning."""
	s = Step([64, 64], [1, 20], 8, 2, 64, 16, 'fp16')
	for c in range(4):
		s.table[1][c] = s.table[0][c]
	k, v = s.k.to(DEV), s.v.to(DEV)
	out = G.paged_attention(s.parts(s.qkv.to(DEV))[0], k, v, make_plan(s, k))
	want, absolute, score = O.attention(s.parts()[0], s.k, s.v, s.table, [0, 1, 21], [65, 84])
	assert ((out.cpu().double() - want).abs() <= bound(want, absolute, score, 64, 84, torch.float16)).all()


def test_another_stream(step):
	k, v, q, kn, vn = on_gpu(step)
	want = G.paged_attention(q, k, v, make_plan(step, k))
	torch.cuda.synchronize()
	s = torch.cuda.Stream()
	with torch.cuda.stream(s):
		got = G.paged_attention(q, k, v, make_plan(step, k))
	s.synchronize()
	used = sum(step.new)
	assert torch.equal(got[:used], want[:used])


@pytest.mark.parametrize('new', [[1, 1], [3, 300]])
@pytest.mark.parametrize('dtype', ['fp16', 'fp32'])
def test_pages_that_do_not_exist(new, dtype):
	"""The status says so, other requests are not touched by it, and nothing outside the cache is read."""
	s = Step([100, 90], new, 4, 2, 64, 16, dtype)
	k, v = s.k.to(DEV), s.v.to(DEV)
	q = s.parts(s.qkv.to(DEV))[0]
	want = G.paged_attention(q, k, v, make_plan(s, k))
	for wrong in (-1, s.pages, 2 ** 31 - 1, -2 ** 31):
		s.table[0][2] = wrong
		out = G.paged_attention(q, k, v, make_plan(s, k))
		torch.cuda.synchronize()
		assert torch.equal(out[new[0]:], want[new[0]:])
		assert status() == 4


def test_rows_that_see_nothing_and_masked_values():
	"""Infinite scores and values count where they are seen and only there."""
	s = Step([0, 40], [20, 1], 2, 2, 64, 16, 'fp32', fill=float('inf'))
	s.k[s.table[0][0], :, 0] = 0          # the first key of the first request: score 0 for everyone
	k, v, q, _, _ = on_gpu(s)
	v[s.table[0][1], :, 3] = float('inf')          # a value at position 19, which only the last row sees
	out = G.paged_attention(q, k, v, make_plan(s, k))
	assert torch.isinf(out[19]).all() or torch.isnan(out[19]).any()
	assert torch.isfinite(out[20]).all()
	big = s.qkv.clone()
	big[:, :2 * 64] = 1e4                  # scores far apart: one key takes all the weight
	q = s.parts(big.to(DEV))[0]
	k, v = s.k.to(DEV), s.v.to(DEV)
	out = G.paged_attention(q, k, v, make_plan(s, k))
	want, _, _ = O.attention(s.parts(big)[0], s.k, s.v, s.table, [0, 20, 21], [20, 41])
	assert (out.cpu().double() - want).abs().max() <= 1e-4


def test_numbers_beyond_the_c_types_are_refused(step):
	k = step.k.to(DEV)
	ok = dict(past=step.ints(step.past), new=step.ints(step.new), table=step.ints(step.table), cache=k, rows=step.rows, heads=8)
	for change in (dict(rows=1 << 30), dict(heads=1 << 16), dict(heads=(1 << 32) + 8)):
		with pytest.raises(ValueError):
			G.paged_plan(**{**ok, **change})
