"""Work lists of the paged attention at sizes where the plan forms them in another way: more entries than it keeps in shared memory, more
blocks of keys than it counts; the order in which the partial results of cut jobs are added up."""
import pytest
import torch

import gptq_triton_b200 as G
from test_gpu_paged import DEV, healthy, status      # noqa: F401 (healthy: status is zero behind every test)

pytestmark = pytest.mark.gpu
PAGE = 1 << 24


@pytest.mark.parametrize('requests,columns', [(16, 64), (32, 64), (1024, 4), (4096, 2), (8192, 64)])
def test_more_blocks_than_the_lists_count(requests, columns):
	"""Tables whose columns all name one page of 2^24 rows: 2^30 blocks of 16 keys and more.  The status says so, whatever the sum is, and nothing
	is computed."""
	cache = torch.zeros((1, 1, PAGE, 8), dtype=torch.float16, device=DEV)
	past = torch.full((requests,), columns * PAGE - 1, dtype=torch.int32, device=DEV)
	table = torch.zeros((requests, columns), dtype=torch.int32, device=DEV)
	plan = G.paged_plan(past, torch.ones_like(past), table, cache, requests, 1, max_new=1)
	assert status() == 8
	assert plan.lens.tolist() == [columns * PAGE] * requests and plan.slots.tolist() == [PAGE - 1] * requests
	out = torch.full((requests, 1, 8), 7.0, dtype=torch.float16, device=DEV)
	G.paged_attention(out.clone(), cache, cache, plan, out=out)
	assert (out == 7).all()


def test_pages_of_many_long_requests_are_counted():
	"""New tokens that need more pages than an int counts: the pool has none left, and the place behind the pages taken is its end."""
	cache = torch.zeros((4, 1, 1, 8), dtype=torch.float16, device=DEV)
	new = torch.full((8,), 1 << 29, dtype=torch.int32, device=DEV)
	table = torch.full((8, 4), -1, dtype=torch.int32, device=DEV)
	pool = torch.arange(4, dtype=torch.int32, device=DEV)
	plan = G.paged_plan(torch.zeros_like(new), new, table, cache, 4, 1, pool=pool, head=torch.zeros(1, dtype=torch.int32, device=DEV))
	assert status() == 8
	assert plan.head.tolist() == [4] and plan.row_start.tolist() == [0] + [4] * 8 and table[0].tolist() == [0, 1, 2, 3] and (table[1:] == -1).all()


@pytest.mark.parametrize('first', [0.3, -0.45])
def test_partial_results_are_added_in_one_order(first):
	"""Two partial results of one row, keys 0 .. 15 and 16 .. 47, exact in themselves: equal scores within each (weights of one), values that are whole
	numbers.  Heads of 64 are folded by two halves of a warp, heads of 72 by one lane after the other; both add the first to the second."""
	L = 48
	g = torch.Generator().manual_seed(3)
	values = torch.randint(-999, 1000, (L, 64), generator=g).float()
	outs = []
	for dim in (64, 72):
		k, v, q = torch.zeros(3, 1, 16, dim), torch.zeros(3, 1, 16, dim), torch.zeros(1, 1, dim)
		k[0, 0, :, 0] = first
		q[0, 0, 0] = 1.0
		v[..., :64] = values.view(3, 1, 16, 64)
		i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)
		k, v, q = k.to(DEV), v.to(DEV), q.to(DEV)
		plan = G.paged_plan(i32([L - 1]), i32([1]), i32([[0, 1, 2]]), k, 1, 1, max_new=1)
		outs.append(G.paged_attention(q, k, v, plan, scale=1.0)[0, 0, :64].cpu())
	w = torch.tensor([first] * 16 + [0.0] * 32, dtype=torch.float64).softmax(0)
	assert ((outs[0].double() - w @ values.double()).abs() <= 2e-6 * (w @ values.double().abs())).all()
	assert torch.equal(outs[0], outs[1])
