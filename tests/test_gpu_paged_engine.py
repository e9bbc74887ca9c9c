"""Requests of different lengths through the engine with pages: the same greedy tokens as the dequantise-then-matmul twin of the model
gives for each request alone."""
import json

import pytest
import torch

from test_gpu_decode import build_pair, reference_greedy

pytestmark = pytest.mark.gpu
LENGTHS, STEPS = [40, 1, 17, 65, 5], 12


@pytest.fixture(scope='module')
def case():
	"""A model and prompts whose greedy choices are clear in every step (random weights give flat logits)."""
	for seed in range(40):
		cfg, model, dense = build_pair(seed)
		g = torch.Generator().manual_seed(seed)
		prompts, want, clear = [], [], True
		for n in LENGTHS:
			for _ in range(12):
				p = torch.randint(0, cfg.vocab_size, (1, n), generator=g)
				toks, margins = reference_greedy(dense, p.cuda(), STEPS)
				if min(margins) > 0.02:
					break
			else:
				clear = False
				break
			prompts.append(p[0].tolist())
			want.append(toks[0].tolist())
		if clear:
			return cfg, model, prompts, want
	raise AssertionError('no seed with clear choices')


@pytest.mark.parametrize('use_graph', [False, True])
@pytest.mark.parametrize('page_size,requests,portion', [(16, 8, 2048), (8, 2, 7), (64, 3, 33), (5, 5, 16)])
def test_tokens(case, use_graph, page_size, requests, portion):
	import gptq_triton_b200 as G
	cfg, model, prompts, want = case
	pages = sum(-(-(n + STEPS) // page_size) for n in sorted(LENGTHS)[-requests:]) + 1
	engine = G.PagedEngine(model, pages=pages, page_size=page_size, requests=requests, max_seq=80, portion=portion, use_graph=use_graph)
	assert engine.generate(prompts, STEPS) == want
	assert sorted(engine.free) == list(range(pages)) and engine.reserved == 0 and not engine.busy
	assert engine.generate(prompts[::-1], STEPS) == want[::-1]          # pages in another order
	engine.close()


def test_requests_come_and_go(case):
	"""Requests that are added while others decode, a stop token, a single token to generate."""
	import gptq_triton_b200 as G
	cfg, model, prompts, want = case
	engine = G.PagedEngine(model, pages=40, requests=3, max_seq=80, portion=20)
	stop = want[2][4]
	seen = {}

	def step():
		for number, token in engine.step():
			seen.setdefault(number, []).append(token)
	a = engine.add(prompts[0], STEPS)
	step()
	step()
	b = engine.add(prompts[2], STEPS, stop=stop)
	step()
	c = engine.add(prompts[3], 1)
	while engine.busy:
		step()
	assert engine.results[a] == want[0] and engine.results[c] == want[3][:1]
	assert engine.results[b] == want[2][:want[2].index(stop) + 1] == seen[b]
	from gptq_triton_b200 import _lib
	assert _lib.kernel_status() == 0


@torch.no_grad()
def test_cached_rows():
	"""Keys and values that the steps leave in the pages, against those of the twin for each request alone: positions, portions, pages."""
	import gptq_triton_b200 as G
	cfg, model, dense = build_pair(5)
	g = torch.Generator().manual_seed(1)
	prompts = [torch.randint(0, cfg.vocab_size, (n,), generator=g).tolist() for n in LENGTHS]
	engine = G.PagedEngine(model, pages=64, page_size=8, max_seq=90, portion=23)
	for p in prompts:
		engine.add(p, STEPS)
	for _ in range(11):          # prompts in portions, then single tokens
		engine.step()
	for r in engine.slots[:len(prompts)]:
		ids = (r.prompt + r.out)[:r.fed]
		assert len(r.out) > 2
		_, past = dense(torch.tensor([ids]).cuda(), use_cache=True)
		j = torch.arange(r.fed, device='cuda')
		where = torch.tensor(r.pages, device='cuda')[j // 8]
		assert engine.table[r.slot, :len(r.pages)].tolist() == r.pages
		for i in range(cfg.num_hidden_layers):
			for cache, want in ((engine.kcache[i], past[i][0][0]), (engine.vcache[i], past[i][1][0])):
				got = cache[where, :, j % 8].transpose(0, 1)
				assert (got.float() - want.float()).abs().max() <= 2e-2 * want.float().abs().max()          # (fp16 activations through a few layers)


def test_refusals(case):
	import gptq_triton_b200 as G
	cfg, model, prompts, _ = case
	engine = G.PagedEngine(model, pages=4, max_seq=80)
	for prompt, steps in (([], 3), ([1], 0), ([cfg.vocab_size], 1), ([-1], 1), ([1] * 81, 1), ([1] * 65, 2)):
		with pytest.raises(ValueError):
			engine.add(prompt, steps)
	with pytest.raises(ValueError):
		G.PagedEngine(model, pages=0)
	assert engine.step() == [] and not engine.busy


def test_command_line(case, tmp_path, capsys):
	"""`generate` with prompts of different lengths."""
	import gptq_triton_b200 as G
	from gptq_triton_b200 import __main__, loader
	from gptq_triton_b200.llama import LlamaConfig
	cfg = LlamaConfig(hidden_size=512, intermediate_size=1408, num_hidden_layers=2, num_attention_heads=4, vocab_size=512, max_position_embeddings=256)
	model = G.synthetic_quantized_llama(cfg, groupsize=128, seed=3, device='cpu', fuse=False)
	loader.save_quant(model, tmp_path, 128)
	assert __main__.main(['generate', '--model', str(tmp_path), '--prompt-ids', '1,2,3;7;9,10', '--steps', '5']) == 0
	rows = [json.loads(line) for line in capsys.readouterr().out.strip().splitlines()]
	assert [len(r) for r in rows] == [5, 5, 5]
	engine = G.PagedEngine(G.load_model(str(tmp_path)), pages=8, max_seq=20)
	assert engine.generate([[1, 2, 3], [7], [9, 10]], 5) == rows


def test_a_refused_prompt_leaves_nothing_queued(case):
	import gptq_triton_b200 as G
	cfg, model, prompts, want = case
	engine = G.PagedEngine(model, pages=64, max_seq=80)
	with pytest.raises(ValueError):
		engine.generate([prompts[0], [-1]], STEPS)
	assert not engine.busy and engine.generate([prompts[1]], STEPS) == [want[1]]
