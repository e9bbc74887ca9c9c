"""ctypes binding of the paged-cache entry points of libgptq_b200.so (declared in include/paged_b200.h).  Like the other bindings it has
no fallback: a missing library or a failing kernel raises."""
from __future__ import annotations

import ctypes
import threading
from ctypes import c_float, c_int, c_int64, c_size_t, c_void_p
from typing import Dict, Optional

import torch

from ._lib import LIB_PATH, GptqB200Error, ptr, register_status_buffer, require_cuda, stream_ptr      # noqa: F401

CONTROL_BYTES = 16384
MAX_REQUESTS = 8192
MAX_DIM = 256
MAX_PAGE = 1 << 24
DTYPE_CODE = {torch.bfloat16: 0, torch.float32: 1, torch.float16: 2}

_P, _I = c_void_p, c_int


class Plan(ctypes.Structure):
	_fields_ = [(n, _I) for n in ('requests', 'rows', 'table_width', 'page', 'pages', 'pool_size')] + [('table_ld', c_int64)] + [
		(n, _P) for n in ('past', 'fresh', 'table', 'pool', 'head', 'next_head', 'row_start', 'lens', 'positions', 'slots')] + [
		(n, _I) for n in ('heads', 'kv_heads', 'dim', 'max_fresh')] + [('work', _P), ('status', _P)]


class Append(ctypes.Structure):
	_fields_ = [(n, _I) for n in ('rows', 'heads', 'kv_heads', 'dim', 'rot', 'max_pos', 'page', 'pages')] + [(n, _P) for n in ('q', 'k', 'v')] + [
		(n, c_int64) for n in ('q_row', 'q_head', 'k_row', 'k_head', 'v_row', 'v_head')] + [
		(n, _P) for n in ('cos_t', 'sin_t', 'positions', 'slots', 'q_out', 'k_cache', 'v_cache')] + [
		(n, c_int64) for n in ('k_page', 'k_kv', 'v_page', 'v_kv')] + [('status', _P)]


class Attention(ctypes.Structure):
	_fields_ = [(n, _I) for n in ('requests', 'rows', 'heads', 'kv_heads', 'dim', 'page', 'pages', 'table_width', 'max_fresh')] + [
		('table_ld', c_int64), ('scale', c_float), ('q', _P), ('q_row', c_int64), ('q_head', c_int64), ('k_cache', _P), ('v_cache', _P)] + [
		(n, c_int64) for n in ('k_page', 'k_kv', 'v_page', 'v_kv')] + [(n, _P) for n in ('table', 'row_start', 'lens', 'work', 'out', 'scratch')] + [
		('scratch_bytes', c_size_t), ('status', _P)]


_SIGNATURES = {
	'paged_version': (c_int, []),
	'paged_last_cuda_error': (c_int, []),
	'paged_work_ints': (c_int64, [_I, _I, _I, _I]),
	'paged_plan': (c_int, [_P, _I, _P]),
	'paged_append': (c_int, [_P, _I, _P]),
	'paged_attention_scratch': (c_int64, [_P, _I]),
	'paged_attention': (c_int, [_P, _I, _P]),
}

_lib: Optional[ctypes.CDLL] = None
_control: Dict[int, torch.Tensor] = {}
_status: Dict[int, int] = {}
_lock = threading.Lock()


def exported_symbols():
	"""Names that include/paged_b200.h declares."""
	return list(_SIGNATURES)


def lib() -> ctypes.CDLL:
	global _lib
	if _lib is None:
		if not LIB_PATH.exists():
			raise ImportError(f'{LIB_PATH} is missing: build it with `python -m gptq_triton_b200.build` (needs nvcc with sm_100a support). '
							  'There is no CPU or Triton fallback.')
		l = ctypes.CDLL(str(LIB_PATH))
		for name, (res, args) in _SIGNATURES.items():
			fn = getattr(l, name)
			fn.restype, fn.argtypes = res, args
		_lib = l
	return _lib


class _Ctypes:
	"""In the place of the extension module: serves nothing, so every call goes through ctypes."""
	paged_plan = paged_append = paged_attention = staticmethod(lambda *a: None)


_native = None


def native():
	"""The operators in native code (csrc/host/calls.cpp); each returns None when the call is not the plain case."""
	global _native
	if _native is None:
		from . import _lib as base
		module, l = base.host(), lib()
		if hasattr(module, 'paged_bind'):
			module.paged_bind(*(ctypes.cast(getattr(l, name), c_void_p).value for name in ('paged_plan', 'paged_append', 'paged_attention', 'paged_attention_scratch', 'paged_work_ints')))
			_native = module
		else:
			_native = _Ctypes
	return _native


_MESSAGES = {-1: 'invalid argument', -2: 'shape violates a divisibility rule', -3: 'scratch missing or too small', -4: 'pointer or stride misaligned', -5: 'CUDA error', -6: 'not supported'}


def check(code: int, what: str):
	if code != 0:
		extra = f' (cudaError {lib().paged_last_cuda_error()})' if code == -5 else ''
		raise (ValueError if code in (-1, -2, -4) else GptqB200Error)(f'{what}: {_MESSAGES.get(code, "unknown error code")}{extra}')


def status_ptr(index: int) -> int:
	"""Address of the status word of the paged operators on device `index` (part of _lib.kernel_status())."""
	known = _status.get(index)
	if known is not None:
		return known
	with _lock:
		if index not in _status:
			if torch.cuda.is_current_stream_capturing():
				raise GptqB200Error('the first paged operator on a device must run outside of a graph capture: it sets up the status word')
			device = torch.device('cuda', index)
			buf = torch.zeros(CONTROL_BYTES, dtype=torch.uint8, device=device)
			torch.cuda.current_stream(device).synchronize()          # (any stream may use it from now on)
			register_status_buffer(buf)
			_control[index] = buf
			_status[index] = buf.data_ptr() + CONTROL_BYTES - 4
	return _status[index]
