"""Host side of PagedEngine: its tables, who gets which part of a step.  No kernel is launched: the steps of the device are stand-ins."""
import pytest
import torch

import gptq_triton_b200 as G
from gptq_triton_b200.llama import LlamaConfig


@pytest.fixture(scope='module')
def model():
	cfg = LlamaConfig(hidden_size=256, intermediate_size=256, num_hidden_layers=2, num_attention_heads=2, vocab_size=64, max_position_embeddings=64)
	m = G.synthetic_quantized_llama(cfg, groupsize=128, seed=0, device='cpu', fuse=False)
	G.make_quant_attn(m)
	return m


def test_the_layers_keep_their_tables(model):
	"""A captured step of another engine reads the tables of the layers at their addresses: an engine with more positions makes its own."""
	attn = model.model.layers[0].self_attn
	before = attn.tables(torch.device('cpu'), 64)
	engine = G.PagedEngine(model, pages=8, max_seq=500)
	after = attn._tables
	assert after[0] is before[0] and after[1] is before[1] and before[0].shape[0] == 64
	assert engine.cos.shape == engine.sin.shape == (500, 128)
	assert torch.equal(engine.cos[:64], before[0]) and torch.equal(engine.sin[:64], before[1])


def fake(engine, fed):
	"""Steps that generate token 1 for everyone; fed: (request, tokens) of every step."""
	def run(active):
		fed.append([(r.number, n) for r, n in active])
		return [1] * len(active)
	engine._mixed = engine._decode = run


def test_portions_go_to_the_request_that_came_first(model):
	"""A prompt is not held up by prompts that came later, whatever slots they sit in."""
	engine = G.PagedEngine(model, pages=100, page_size=8, requests=2, max_seq=64, portion=10)
	fed = []
	fake(engine, fed)
	a, b = engine.add([0] * 10, 1), engine.add([0] * 30, 1)
	later = []
	for _ in range(4):          # short prompts keep coming to the slot before that of b
		later.append(engine.add([0] * 10, 1))
		engine.step()
	assert fed[0] == [(a, 10)] and fed[1:4] == [[(b, 10)]] * 3
	assert engine.results[b] == [1]
	while engine.busy:
		engine.step()
	assert all(engine.results[n] == [1] for n in [a, b, *later])
	assert sorted(engine.free) == list(range(100)) and engine.reserved == 0


def test_rows_of_a_step_stay_in_the_order_of_the_slots(model):
	engine = G.PagedEngine(model, pages=100, page_size=8, requests=3, max_seq=64, portion=12)
	fed = []
	fake(engine, fed)
	a, b, c = engine.add([0] * 4, 2), engine.add([0] * 9, 3), engine.add([0] * 9, 1)
	engine.step()
	assert fed == [[(a, 4), (b, 8)]]          # (b is one token short, c waits)
	engine.step()
	d = engine.add([0] * 9, 1)
	engine.step()          # a and c have ended, d takes the slot of a: its rows come before that of b
	assert fed[1:] == [[(a, 1), (b, 1), (c, 9)], [(d, 9), (b, 1)]]
	while engine.busy:
		engine.step()
	for step in fed:
		assert len({n for n, _ in step}) == len(step) and all(k > 0 for _, k in step)
	assert [len(engine.results[n]) for n in (a, b, c, d)] == [2, 3, 1, 1]
