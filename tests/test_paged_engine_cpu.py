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
