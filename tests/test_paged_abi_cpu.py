"""Refusals and status bits of the C ABI of the paged cache.  No kernel is launched."""
import ctypes
import itertools
import re
from pathlib import Path

import pytest

from test_paged_cpu import _attention, _plan, lib      # noqa: F401


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
