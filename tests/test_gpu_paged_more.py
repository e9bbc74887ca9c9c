"""Attention over work lists of more than a thousand and more than four thousand tiles, values and keys that are not finite in hidden places, rows that see nothing."""
import math

import pytest
import torch

import gptq_triton_b200 as G
from oracle import paged_oracle as O
from paged_cases import Step, bound
from test_gpu_paged import DEV, check_attention, healthy, make_plan, status      # noqa: F401 (healthy: status is zero behind every test)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('requests,new,longest,dtype', [
	(1100, 1, 70, 'fp16'), (1100, 1, 9000, 'fp32'), (5000, 1, 70, 'fp32'), (5000, 1, 9000, 'fp16'), (8192, 1, 9000, 'fp16'),
	(1100, 17, 70, 'fp16'), (1100, 17, 9000, 'fp16'), (4200, 17, 70, 'fp16'), (4200, 17, 9000, 'fp16'), (1500, 17, 9000, 'fp32')])
def test_many_requests(requests, new, longest, dtype):
	"""Two heads over one: a single token is a tile of the kernel for few rows, 17 tokens are one of the tile kernel (in fp32 three of the other);
	some long requests, whose jobs are cut."""
	past = [i * 7 % 61 if i % 900 != 450 else longest + i // 50 for i in range(requests)]
	counts = [new if i % 97 != 5 else 0 for i in range(requests)]
	check_attention(Step(past, counts, 2, 1, 8, 16, dtype, seed=requests + new, pad=3), max_new=new)


@pytest.mark.parametrize('dtype', ['fp16', 'bf16', 'fp32'])
@pytest.mark.parametrize('bad', [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize('past,new,at', [(0, 20, 19), (40, 16, 50), (0, 300, 290), (130, 400, 513)])
def test_hidden_keys_that_are_not_finite(past, new, at, bad, dtype):
	"""A key at position `at` counts for the rows that see it and for no other."""
	s = Step([past, 33], [new, 1], 4, 2, 64, 16, dtype)
	k, v = s.k.to(DEV), s.v.to(DEV)
	q = s.parts(s.qkv.to(DEV))[0]
	plan = make_plan(s, k)
	want = G.paged_attention(q, k, v, plan)
	k[s.table[0][at // 16], :, at % 16] = bad
	out = G.paged_attention(q, k, v, plan)
	assert torch.equal(out[:at - past], want[:at - past]) and torch.equal(out[new], want[new])
	assert torch.isfinite(want).all() and not torch.isfinite(out[at - past:new]).all(-1).all()


@pytest.mark.parametrize('dtype', ['fp16', 'bf16', 'fp32'])
@pytest.mark.parametrize('past,new,at,clean', [(0, 20, 19, 0), (0, 16, 15, 0), (0, 40, 37, 0), (0, 300, 290, 256)])
def test_hidden_values_that_are_not_finite(past, new, at, clean, dtype):
	"""A value at position `at` makes the rows that see it infinite or NaN.  Rows of tiles whose last row does not see it, and other requests, are as
	they were; rows between may be NaN.  clean: rows of full tiles of the kernel for chunks (fp32: the tiles have 16 rows)."""
	s = Step([past, 33], [new, 1], 2, 2, 64, 16, dtype)
	k, v = s.k.to(DEV), s.v.to(DEV)
	q = s.parts(s.qkv.to(DEV))[0]
	plan = make_plan(s, k)
	want = G.paged_attention(q, k, v, plan)
	v[s.table[0][at // 16], :, at % 16] = math.inf
	out = G.paged_attention(q, k, v, plan)
	if dtype == 'fp32' or new <= 16:
		clean = at // 16 * 16
	assert torch.equal(out[:clean], want[:clean]) and torch.equal(out[new], want[new]) and torch.isfinite(want).all()
	assert not torch.isfinite(out[at - past:new]).any()


@pytest.mark.parametrize('dtype', ['fp16', 'bf16', 'fp32'])
@pytest.mark.parametrize('past,new,columns', [([0], [40], 1), ([0, 5], [20, 1], 1), ([3000, 0], [40, 3100], 190), ([0], [300], 2)])
def test_rows_that_see_nothing(past, new, columns, dtype):
	"""A table too narrow for the tokens: the status says so, and rows that no key is left for are zero; in whole jobs and in cut ones."""
	s = Step(past, new, 2, 2, 64, 16, dtype)
	s.table = [row[:columns] for row in s.table]
	lens = [min(p + n, 16 * columns) for p, n in zip(past, new)]
	assert any(L < n for L, n in zip(lens, new))
	k, v = s.k.to(DEV), s.v.to(DEV)
	plan = make_plan(s, k)
	assert status() == 8 and plan.lens.tolist() == lens
	out = G.paged_attention(s.parts(s.qkv.to(DEV))[0], k, v, plan).cpu()
	start = [0]
	for n in new:
		start.append(start[-1] + n)
	want, absolute, score = O.attention(s.parts()[0], s.k, s.v, s.table, start, lens)
	for a, L, n in zip(start, lens, new):
		assert (out[a:a + max(n - L, 0)] == 0).all()
	assert ((out.double() - want).abs() <= bound(want, absolute, score, 64, max(lens), s.dtype)).all()
