"""What engines on one model share and what not."""
import weakref

import pytest
import torch

import gptq_triton_b200 as G
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
