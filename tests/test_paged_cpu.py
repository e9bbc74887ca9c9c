"""Host side of the cache in pages: the library's symbols and refusals, the Python layer's checks.  No kernel is launched."""
import ctypes
import re
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parent.parent


@pytest.fixture(scope='module')
def lib():
	from gptq_triton_b200 import _paged, build
	build.build(only=['gptq'])
	return _paged.lib()


def test_header_binding_and_library_agree(lib):
	from gptq_triton_b200 import _paged
	text = re.sub(r'/\*.*?\*/', '', (ROOT / 'include' / 'paged_b200.h').read_text(), flags=re.S)
	names = sorted(set(re.findall(r'\b(paged_[a-z0-9_]+)\s*\(', text)))
	assert names == sorted(_paged.exported_symbols()) and len(names) == 7
	for n in names:
		assert hasattr(lib, n)
	assert lib.paged_version() >= 100


def _plan(**kw):
	from gptq_triton_b200 import _paged
	a = _paged.Plan()
	v = dict(requests=2, rows=4, table_width=3, page=16, pages=8, pool_size=0, table_ld=3, past=64, fresh=64, table=64, pool=None, head=None, next_head=None, row_start=64, lens=64, positions=64, slots=64,
			 heads=4, kv_heads=2, dim=64, max_fresh=4, work=64, status=64)
	v.update(kw)
	for n, x in v.items():
		setattr(a, n, x)
	return a


@pytest.mark.parametrize('kw', [dict(requests=-1), dict(requests=8193), dict(rows=-1), dict(page=0), dict(pages=-1), dict(table_width=0), dict(table_ld=2), dict(heads=3), dict(kv_heads=0), dict(past=None), dict(fresh=None),
								dict(table=None), dict(lens=None), dict(positions=None), dict(slots=None), dict(row_start=None), dict(work=None), dict(status=None), dict(pool=64), dict(pool=64, head=64, next_head=64),
								dict(max_fresh=-1)], ids=str)
def test_plan_refuses(lib, kw):
	assert lib.paged_plan(ctypes.byref(_plan(**kw)), 2, None) == -1
	assert lib.paged_plan(ctypes.byref(_plan()), 3, None) == -1 and lib.paged_plan(None, 2, None) == -1


def _append(**kw):
	from gptq_triton_b200 import _paged
	a = _paged.Append()
	v = dict(rows=4, heads=4, kv_heads=2, dim=64, rot=64, max_pos=9, page=16, pages=8, q=64, k=64, v=64, cos_t=64, sin_t=64, positions=64, slots=64, q_out=64, k_cache=64, v_cache=64, status=64)
	v.update(kw)
	for n, x in v.items():
		setattr(a, n, x)
	return a


@pytest.mark.parametrize('kw', [dict(rows=-1), dict(heads=5), dict(dim=0), dict(rot=66), dict(rot=3), dict(rot=-2), dict(max_pos=0), dict(page=0), dict(q=None), dict(k=None), dict(v=None), dict(cos_t=None), dict(sin_t=None),
								dict(positions=None), dict(slots=None), dict(q_out=None), dict(k_cache=None), dict(v_cache=None), dict(status=None)], ids=str)
def test_append_refuses(lib, kw):
	assert lib.paged_append(ctypes.byref(_append(**kw)), 0, None) == -1
	assert lib.paged_append(ctypes.byref(_append(rows=0)), 0, None) == 0          # nothing to do


def _attention(**kw):
	from gptq_triton_b200 import _paged
	a = _paged.Attention()
	v = dict(requests=2, rows=4, heads=4, kv_heads=2, dim=64, page=16, pages=8, table_width=3, max_fresh=4, table_ld=3, scale=0.125, q=64, q_row=256, q_head=64, k_cache=64, v_cache=64, k_page=2048, k_kv=1024, v_page=2048,
			 v_kv=1024, table=64, row_start=64, lens=64, work=64, out=64, scratch=64, scratch_bytes=0, status=64)
	v.update(kw)
	for n, x in v.items():
		setattr(a, n, x)
	return a


@pytest.mark.parametrize('kw,code', [(dict(requests=-1), -1), (dict(rows=-1), -1), (dict(heads=3), -1), (dict(page=0), -1), (dict(scale=0.0), -1), (dict(scale=-1.0), -1), (dict(scale=float('inf')), -1), (dict(scale=float('nan')), -1),
									 (dict(q=None), -1), (dict(k_cache=None), -1), (dict(v_cache=None), -1), (dict(table=None), -1), (dict(row_start=None), -1), (dict(lens=None), -1), (dict(work=None), -1), (dict(out=None), -1),
									 (dict(status=None), -1), (dict(dim=63), -2), (dict(dim=264), -2), (dict(q=66), -4), (dict(k_cache=72), -4), (dict(q_row=257), -4), (dict(k_page=2049), -4), (dict(v_kv=1028), -4)], ids=str)
def test_attention_refuses(lib, kw, code):
	assert lib.paged_attention(ctypes.byref(_attention(**kw)), 2, None) == code
	assert lib.paged_attention(ctypes.byref(_attention(rows=0)), 2, None) == 0


def test_sizing_needs_no_device(lib):
	assert lib.paged_work_ints(0, 0, 1, 1) > 0 and lib.paged_work_ints(8192, 1 << 20, 64, 8) < 1 << 24
	assert lib.paged_work_ints(1, 1, 3, 2) == -1


def test_cpu_tensors_are_refused(lib):
	from gptq_triton_b200 import _lib, paged_plan
	i = torch.zeros(1, dtype=torch.int32)
	with pytest.raises(_lib.GptqB200Error, match='CUDA'):
		paged_plan(i, i, i.view(1, 1), torch.zeros(1, 1, 16, 64, dtype=torch.float16), 1, 1)


def test_pages_longer_than_positions_count_are_refused(lib):
	"""Positions are counted up to 2^30; past + page must stay an int."""
	from gptq_triton_b200 import _paged
	page = _paged.MAX_PAGE + 1
	assert lib.paged_plan(ctypes.byref(_plan(page=page)), 2, None) == -1
	assert lib.paged_append(ctypes.byref(_append(page=page)), 0, None) == -1
	assert lib.paged_attention(ctypes.byref(_attention(page=page)), 2, None) == -1
	assert lib.paged_attention_scratch(ctypes.byref(_attention(page=page)), 2) == -1
	assert lib.paged_attention_scratch(ctypes.byref(_attention(page=page - 1)), 2) > 0
