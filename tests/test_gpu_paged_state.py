"""What engines on one model share and what not: rotary tables, streams with their workspaces, captured steps; status words that a
step meets."""
import weakref

import pytest
import torch

import gptq_triton_b200 as G
from gptq_triton_b200 import _lib, _paged
from test_gpu_decode import build_pair

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def model():
	return build_pair(4)[1]


@pytest.mark.parametrize('batch', [1, 3])
def test_a_captured_step_holds_the_tables_that_it_reads(model, batch):
	"""Tables of the layers that grow later: the old ones live as long as the step that was captured with them."""
	engine = G.DecodeEngine(model, batch=batch, max_seq=40)
	prompt = torch.randint(0, 512, (batch, 9), generator=torch.Generator().manual_seed(1)).cuda()
	want = engine.generate(prompt, 6)
	refs = [weakref.ref(t) for layer in model.model.layers for t in layer.self_attn._tables]
	dev = prompt.device
	for layer in model.model.layers:
		layer.self_attn.tables(dev, 2 * layer.self_attn._tables[0].shape[0])
	assert all(r() is not None for r in refs)
	assert torch.equal(engine.generate(prompt, 6), want)
	engine.close()
	assert all(r() is None for r in refs)          # ... and no longer


def count_streams(monkeypatch):
	made = []
	real = torch.cuda.Stream

	class Counted(real):
		def __new__(cls, *a, **kw):
			if 'stream_id' not in kw:          # (not the wrappers of a stream that exists)
				made.append(1)
			return real.__new__(real, *a, **kw)
	monkeypatch.setattr(torch.cuda, 'Stream', Counted)
	return made


def serve(engine, count, steps=3):
	"""Requests that come one by one, so that 1 .. count run."""
	numbers = []
	for i in range(count):
		numbers.append(engine.add([1 + i, 2, 3], steps + 2 * (count - i)))
		engine.step()          # its prompt
		engine.step()          # single tokens of all that run
	while engine.busy:
		engine.step()
	return [engine.results.pop(n) for n in numbers]


def test_one_stream_for_all_captured_steps(model, monkeypatch):
	engine = G.PagedEngine(model, pages=400, requests=12, max_seq=80)
	made = count_streams(monkeypatch)
	serve(engine, 12)
	assert len(made) <= 1
	engine.close()


def test_captured_steps_share_their_workspace_with_nobody(model):
	"""The workspace of the projections in a captured step is the engine's: no stream has it, that of the capture least of all, whose number somebody
	else may be given.  Its status word is asked for, and it goes with the engine."""
	first, second = (G.PagedEngine(model, pages=100, requests=2, max_seq=80) for _ in range(2))
	want = serve(first, 2)
	known = dict(_lib._workspaces)
	assert serve(second, 2) == want and _lib._workspaces.keys() == known.keys()
	mine = [e._workspace.buffer for e in (first, second)]
	assert all(m.numel() > 0 and m is not ws for m in mine for ws in [*_lib._workspaces.values(), *_lib._retired]) and mine[0] is not mine[1]
	_lib.status_word(mine[1]).fill_(3)
	try:
		assert _lib.kernel_status() == 3
		assert serve(first, 2) == want
		with pytest.raises(_lib.GptqB200Error, match='3'):
			serve(second, 2)
	finally:
		_lib.clear_kernel_status()
	side = torch.cuda.Stream()
	with torch.cuda.stream(first._stream):          # the same stream for other work: it has a workspace of its own
		assert serve(G.PagedEngine(model, pages=100, requests=2, max_seq=80, use_graph=False), 2) == want
	side.wait_stream(torch.cuda.current_stream())
	with torch.cuda.stream(side):
		assert serve(first, 2) == want
	side.synchronize()
	assert first._workspace.buffer is mine[0]
	seen = weakref.ref(mine[0])
	first.close()
	del mine, first
	assert seen() is None


def test_few_captured_steps_with_one_pool(model):
	engine = G.PagedEngine(model, pages=2000, requests=40, max_seq=120)
	with_graph = serve(engine, 40)
	graphs = [g for g, _ in engine._graphs.values()]
	assert len(graphs) <= 20 and len({g.pool() for g in graphs}) == 1
	engine.close()
	assert not engine._graphs
	assert serve(engine, 3) == serve(G.PagedEngine(model, pages=100, requests=3, max_seq=120, use_graph=False), 3)          # (captured again)
	assert serve(G.PagedEngine(model, pages=2000, requests=40, max_seq=120, use_graph=False), 40) == with_graph


def test_a_step_that_meets_a_status_raises(model):
	engine = G.PagedEngine(model, pages=40, requests=2, max_seq=80)
	a = engine.add([1, 2, 3], 6)
	engine.step()
	engine.step()
	b = engine.add([4], 3)
	word = _paged._control[0][_paged.CONTROL_BYTES - 4:].view(torch.int32)
	word.fill_(8)
	try:
		with pytest.raises(_lib.GptqB200Error, match='8'):
			engine.step()
		assert not engine.busy and sorted(engine.free) == list(range(40)) and engine.reserved == 0 and not engine.results
		with pytest.raises(_lib.GptqB200Error, match='8'):
			engine.generate([[1, 2], [3], [4, 5, 6]], 4)
		assert not engine.busy and sorted(engine.free) == list(range(40)) and engine.reserved == 0 and not engine.results
	finally:
		_lib.clear_kernel_status()
	c = engine.add([1, 2, 3], 6)
	while engine.busy:
		engine.step()
	assert len(engine.results.pop(c)) == 6 and a < b < c
