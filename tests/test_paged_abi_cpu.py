"""Refusals and status bits of the C ABI of the paged cache.  No kernel is launched."""
import ctypes
import itertools
import re
from pathlib import Path

import pytest

from test_paged_cpu import _append, _attention, _plan, lib      # noqa: F401


@pytest.mark.parametrize('sizes', [dict(rows=1 << 30, heads=1, kv_heads=1), dict(rows=2 ** 31 - 1, heads=1, kv_heads=1), dict(rows=1 << 20, heads=4096, kv_heads=1)], ids=str)
def test_sizes_that_no_plan_has(lib, sizes):          # noqa: F811
	"""rows + 1, and rows times the query heads of a key head, are counted in ints."""
	assert lib.paged_work_ints(1, *sizes.values()) == -1
	assert lib.paged_plan(ctypes.byref(_plan(**sizes)), 2, None) == -1
	assert lib.paged_attention(ctypes.byref(_attention(**sizes)), 2, None) == -1


def test_attention_refuses_a_negative_number_of_new_tokens(lib):          # noqa: F811
	assert lib.paged_attention(ctypes.byref(_attention(max_fresh=-1)), 2, None) == -1


def test_status_bits():
	"""The operators set bits beside one another, in a word whose other values are codes: no two of them may add up to another's code."""
	root = Path(__file__).resolve().parent.parent
	bits = {n: int(v) for n, v in re.findall(r'#define (PAGED_(?:BAD_INDEX|NO_ROOM|TIMED_OUT)) (\d+)', (root / 'include' / 'paged_b200.h').read_text())}
	assert len(bits) == 3
	assert {sum(c) for n in (1, 2, 3) for c in itertools.combinations(bits.values(), n)} & set(range(1, 8)) == {bits['PAGED_BAD_INDEX']} == {4}          # (4 is that code)
	for f in (root / 'gptq_triton_b200' / 'csrc' / 'paged').glob('*.cu'):
		for what in re.findall(r'atomicOr\(p\.status, ([^)]*)\)', f.read_text()):
			assert what in (*bits, 'bad'), (f.name, what)


@pytest.mark.parametrize('kw', [dict(k_page=0), dict(v_page=1023), dict(k_kv=0), dict(v_kv=1023)], ids=str)
def test_append_refuses_pages_that_lie_on_one_another(lib, kw):          # noqa: F811
	strides = dict(q_row=256, q_head=64, k_row=128, k_head=64, v_row=128, v_head=64, k_page=2048, k_kv=1024, v_page=2048, v_kv=1024)
	assert lib.paged_append(ctypes.byref(_append(**{**strides, **kw})), 2, None) == -1
	assert lib.paged_append(ctypes.byref(_append(**{**strides, **kw, 'rows': 0})), 2, None) == 0
