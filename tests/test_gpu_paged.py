"""Operators of the cache in pages on the GPU, against the 64-bit restatement."""
import pytest
import torch

from oracle import paged_oracle as O
from paged_cases import DTYPES, Step, bound, ceil

pytestmark = pytest.mark.gpu
DEV = 'cuda'


def make_plan(s: Step, k, **kw):
	from gptq_triton_b200 import paged_plan
	return paged_plan(s.ints(s.past), s.ints(s.new), s.ints(s.table).view(len(s.past), -1), k, s.rows, s.heads, **kw)


def status():
	from gptq_triton_b200 import _lib
	torch.cuda.synchronize()
	st = _lib.kernel_status(torch.device('cuda', torch.cuda.current_device()))
	if st:
		_lib.clear_kernel_status()
	return st


@pytest.fixture(autouse=True)
def healthy():
	yield
	assert status() == 0


# ---- plan ------------------------------------------------------------------------------------------------------------------
PLANS = [
	([0], [1], 16, 0), ([5], [0], 16, 0), ([0, 0, 0], [0, 0, 0], 16, 2), ([15, 16, 17], [1, 1, 1], 16, 0), ([0, 7, 100], [33, 0, 64], 16, 5),
	([3, 0, 9, 2], [1, 2, 3, 4], 1, 1), ([100, 0], [41, 1], 7, 0), ([1000], [3000], 64, 0),
	([i * 37 % 900 for i in range(300)], [(i * 7) % 5 for i in range(300)], 32, 11), ([i % 65 for i in range(1025)], [1 + i % 3 for i in range(1025)], 8, 0),
	([i % 3 for i in range(8192)], [1] * 8192, 16, 1),
]


@pytest.mark.parametrize('past,new,page,pad', PLANS, ids=lambda v: None if isinstance(v, list) else str(v))
def test_plan(past, new, page, pad):
	from gptq_triton_b200 import paged_plan
	rows, R = sum(new) + pad, len(past)
	full = [ceil(p + n, page) for p, n in zip(past, new)]
	width, total = max(full) + 2, sum(full) + 4
	ids = list(range(total))
	import random
	random.Random(len(past)).shuffle(ids)
	table, at = [], 0
	for p in past:
		n = ceil(p, page)
		table.append(ids[at:at + n] + [-1] * (width - n))
		at += n
	pool = [7, 8, 9] + ids[at:]
	cache = torch.empty((total, 2, page, 8), dtype=torch.float16, device=DEV)
	i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
	wide = torch.full((R, width + 3), -5, dtype=torch.int32, device=DEV)          # the table is a part of it
	wide[:, :width] = i32(table)
	want = O.plan(past, new, table, page, rows, pool, 3)
	p_pool, p_head, p_past, p_new = i32(pool), i32([3]), i32(past), i32(new)
	for _ in range(2):          # the second run finds the pages written and writes them again
		plan = paged_plan(p_past, p_new, wide[:, :width], cache, rows, 4, pool=p_pool, head=p_head)
		assert wide[:, :width].tolist() == table and (wide[:, width:] == -5).all()
		assert (plan.row_start.tolist(), plan.lens.tolist(), plan.positions.tolist(), plan.slots.tolist(), int(plan.head)) == want
	assert p_head.tolist() == [3] and p_pool.tolist() == pool and p_past.tolist() == past and p_new.tolist() == new
	plan = paged_plan(p_past, p_new, wide[:, :width], cache, rows, 4, max_new=max(new))          # a complete table
	assert (plan.row_start.tolist(), plan.lens.tolist(), plan.positions.tolist(), plan.slots.tolist(), plan.head) == (*want[:4], None)


def test_plan_of_nothing():
	from gptq_triton_b200 import paged_plan
	e = torch.empty(0, dtype=torch.int32, device=DEV)
	cache = torch.empty((2, 1, 16, 8), dtype=torch.float16, device=DEV)
	plan = paged_plan(e, e, torch.empty((0, 4), dtype=torch.int32, device=DEV), cache, 3, 1)
	assert plan.row_start.tolist() == [0] and plan.slots.tolist() == [-1] * 3 and plan.positions.tolist() == [0] * 3
	plan = paged_plan(e, e, torch.empty((0, 4), dtype=torch.int32, device=DEV), cache, 0, 1)
	assert plan.row_start.tolist() == [0] and plan.slots.numel() == 0


@pytest.mark.parametrize('what,bits', [('pool', 8), ('table', 8), ('rows', 8), ('negative', 4), ('page', 4), ('head', 4), ('huge', 4), ('more', 8)])
def test_plan_without_room(what, bits):
	"""What only the device sees sets the status; slots of such tokens are -1 and nothing else is written."""
	from gptq_triton_b200 import paged_plan
	i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
	past, new, rows, page = [20, 3], [10, 30], 40, 16
	pool, head, width = [4, 5, 6, 7], [0], 3
	table = [[1, 2, -1], [3, -1, -1]]
	if what == 'pool':
		pool = pool[:1]
	elif what == 'table':
		new, rows = [10, 60], 70
	elif what == 'rows':
		rows = 25
	elif what == 'negative':
		past = [-1, 3]
	elif what == 'page':
		table[0][1] = 99
	elif what == 'head':
		head = [-3]
	elif what == 'huge':
		past = [2000000000, 3]
	cache = torch.empty((8, 1, page, 8), dtype=torch.float16, device=DEV)
	plan = paged_plan(i32(past), i32(new), i32(table), cache, rows, 1, pool=i32(pool), head=i32(head), max_new=20 if what == 'more' else None)
	torch.cuda.synchronize()
	assert status() & bits
	s = plan.slots.tolist()
	assert all(-1 <= x < 8 * page for x in s) and max(plan.row_start.tolist()) <= rows
	if what == 'pool':
		assert s[:10] == [2 * 16 + 4 + i for i in range(10)] and s[10:23] == [3 * 16 + 3 + i for i in range(13)] and s[23:39] == [4 * 16 + i for i in range(16)] and s[39:] == [-1]
	elif what == 'rows':
		assert plan.row_start.tolist() == [0, 10, 25]
	elif what == 'page':
		assert s[:10] == [-1] * 10 and s[10] == 3 * 16 + 3


# ---- append ----------------------------------------------------------------------------------------------------------------
def tables(rot, n, dtype):
	angle = torch.outer(torch.arange(n, dtype=torch.float64), 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot))
	full = torch.cat([angle, angle], 1)
	return full.cos().to(dtype), full.sin().to(dtype)


@pytest.mark.parametrize('dtype', list(DTYPES))
@pytest.mark.parametrize('heads,kv_heads,dim,rot,page,past,new,pad,together', [
	(32, 32, 128, 128, 16, [40], [1], 0, False), (8, 2, 64, 64, 32, [0, 31, 5], [7, 2, 0], 3, True), (5, 1, 80, 32, 16, [0], [50], 0, False), (3, 3, 24, 24, 8, [1, 2], [1, 9], 1, False),
	(4, 2, 7, 6, 3, [2, 0], [5, 1], 2, False), (2, 1, 128, 0, 16, [9], [20], 0, True), (1, 1, 1, 0, 1, [0], [3], 0, False), (4, 4, 20, 12, 5, [4], [3], 0, False), (16, 4, 256, 64, 64, [0, 100], [130, 1], 4, False)])
def test_append(dtype, heads, kv_heads, dim, rot, page, past, new, pad, together):
	from gptq_triton_b200 import paged_append
	s = Step(past, new, heads, kv_heads, dim, page, dtype, seed=dim, pad=pad, filled=False, fill=1.5, together=together)
	start, lens, pos, slots, _ = O.plan(past, new, s.table, page, s.rows)
	both = torch.stack([s.k, s.v], 1 if together else 0).to(DEV)
	k, v = (both[:, 0], both[:, 1]) if together else (both[0], both[1])
	plan = make_plan(s, k)
	qkv = s.qkv.to(DEV)
	q, kn, vn = s.parts(qkv)
	cos, sin = tables(rot, max(lens) + 1, s.dtype) if rot else (None, None)
	out = paged_append(q, kn, vn, k, v, plan, *([t.to(DEV) for t in (cos, sin)] if rot else []))
	hq, hk, hv = s.parts()
	pos_t = torch.tensor(pos)
	turn = (lambda x: O.rotate(x, cos[pos_t], sin[pos_t])) if rot else (lambda x: x.double())
	u = torch.finfo(s.dtype).eps / 2
	# two products and their sum in fp32, one rounding: u of the value, 2^-22 of the operands' sizes
	def close(got, want, size):
		assert ((got.double() - want).abs() <= u * 1.01 * want.abs() + 2.0 ** -22 * size + 2.0 ** -25).all()
	close(out.cpu(), turn(hq), hq.double().abs().amax())
	wk, wv = s.k.clone(), s.v.clone()
	used = start[-1]
	rk = turn(hk)
	for m in range(used):
		p, r = divmod(slots[m], page)
		close(k[p, :, r].cpu(), rk[m], hk.double().abs().amax())
		assert torch.equal(v[p, :, r].cpu(), hv[m])
		wk[p, :, r], wv[p, :, r] = k[p, :, r].cpu(), hv[m]
	assert torch.equal(k.cpu(), wk) and torch.equal(v.cpu(), wv)          # nothing else was written
	assert torch.equal(qkv.cpu(), s.qkv)
	q2 = q.contiguous()
	assert paged_append(q2, kn, vn, k, v, plan, *([t.to(DEV) for t in (cos, sin)] if rot else []), out=q2) is q2 and torch.equal(q2, out)


def test_append_outside_the_tables():
	from gptq_triton_b200 import paged_append
	s = Step([14], [4], 2, 1, 64, 16, 'fp16', filled=False, fill=1.0)
	k, v = s.k.to(DEV), s.v.to(DEV)
	plan = make_plan(s, k)
	cos, sin = (t.to(DEV) for t in tables(64, 16, s.dtype))          # positions 16 and 17 are not in it
	q, kn, vn = s.parts(s.qkv.to(DEV))
	out = paged_append(q, kn, vn, k, v, plan, cos, sin)
	assert status() == 4
	assert torch.equal(out[2:], q[2:])          # turned as position 0
	page = s.table[0][1]
	assert (k[page] == 1).all() and (v[page] == 1).all() and not (v[s.table[0][0], 0, 14:] == 1).all()


# ---- attention -------------------------------------------------------------------------------------------------------------
def check_attention(s: Step, scale=None, **kw):
	from gptq_triton_b200 import paged_attention
	k, v = s.k.to(DEV), s.v.to(DEV)
	if s.k.stride(0) != k.stride(0):
		both = torch.stack([s.k, s.v], 1).to(DEV)
		k, v = both[:, 0], both[:, 1]
	plan = make_plan(s, k, **kw)
	q = s.parts(s.qkv.to(DEV))[0]
	out = torch.full((s.rows, s.heads, s.dim), 7.0, dtype=s.dtype, device=DEV)
	assert paged_attention(q, k, v, plan, scale=scale, out=out) is out
	start, lens = [0], [p + n for p, n in zip(s.past, s.new)]
	for n in s.new:
		start.append(start[-1] + n)
	want, absolute, score = O.attention(s.parts()[0], s.k, s.v, s.table, start, lens, scale)
	got = out.cpu()
	assert (got[start[-1]:] == 7).all()          # rows behind the last one are left as they were
	error, allowed = (got[:start[-1]].double() - want).abs(), bound(want, absolute, score, s.dim, max(lens + [0]), s.dtype)
	assert torch.isfinite(got).all()
	assert (error <= allowed).all(), f'{(error / allowed).max():.3f} of the bound at {torch.nonzero(error > allowed)[:5].tolist()}'
	again = torch.full_like(out, 7.0)
	paged_attention(q, k, v, plan, scale=scale, out=again)
	assert torch.equal(out, again)          # the same sums in the same order
	return out


SINGLES = [([0], [1]), ([1], [1]), ([15], [1]), ([16], [1]), ([63], [1]), ([64], [1]), ([700], [1]), ([0, 1, 200, 64, 3, 0, 129], [1, 1, 1, 1, 1, 0, 1]), ([5000], [1])]


@pytest.mark.parametrize('dtype', list(DTYPES))
@pytest.mark.parametrize('past,new', SINGLES, ids=str)
@pytest.mark.parametrize('heads,kv_heads,dim,page', [(4, 4, 128, 16), (8, 1, 64, 32)])
def test_single_tokens(dtype, past, new, heads, kv_heads, dim, page):
	check_attention(Step(past, new, heads, kv_heads, dim, page, dtype, seed=len(past) + page))


@pytest.mark.parametrize('dtype', list(DTYPES))
@pytest.mark.parametrize('heads,kv_heads,dim,page', [(6, 2, 8, 1), (5, 1, 24, 3), (7, 7, 80, 24), (12, 4, 96, 64), (16, 1, 128, 128), (24, 1, 64, 256), (2, 2, 256, 16), (10, 2, 160, 5), (28, 4, 128, 8), (40, 1, 112, 16)])
def test_sizes(dtype, heads, kv_heads, dim, page):
	"""Head sizes, groups and pages of all kinds; single tokens, short and longer chunks in one batch."""
	check_attention(Step([37, 0, 0, 300, 90, 255], [1, 1, 0, 4, 17, 1], heads, kv_heads, dim, page, dtype, seed=dim, pad=3, together=True))


@pytest.mark.parametrize('dtype', list(DTYPES))
@pytest.mark.parametrize('past,new', [([0], [128]), ([0], [257]), ([64], [64]), ([1], [127]), ([3], [130]), ([500], [20]), ([1000], [300]), ([0, 0, 0], [1, 255, 256]), ([129, 0, 40, 0], [100, 1, 1, 310])], ids=str)
@pytest.mark.parametrize('heads,kv_heads,dim,page', [(2, 2, 128, 16), (8, 2, 64, 64), (6, 2, 96, 128), (5, 1, 128, 8)])
def test_chunks(dtype, past, new, heads, kv_heads, dim, page):
	check_attention(Step(past, new, heads, kv_heads, dim, page, dtype, seed=new[0]))


@pytest.mark.parametrize('seed', range(4))
@pytest.mark.parametrize('heads,kv_heads,dim', [(16, 16, 64), (12, 4, 128)])
def test_many_tiles(seed, heads, kv_heads, dim):
	"""Several tiles per processor one after the other, full ones, ones with rows on one side only, short and long ones."""
	import random
	rng = random.Random(seed)
	new = [rng.choice([1, 7, 20, 90, 128, 140, 256, 257, 300, 511]) for _ in range(24)]
	check_attention(Step([rng.choice([0, 0, 5, 130]) for _ in new], new, heads, kv_heads, dim, 32, 'bf16' if seed % 2 else 'fp16', seed=seed, pad=1))


def test_requests_that_all_wait():
	check_attention(Step([5, 0], [0, 0], 4, 2, 64, 16, 'fp16', pad=4))
