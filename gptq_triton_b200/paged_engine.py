"""Serving of LLaMA models from a cache in pages: requests of different lengths side by side, prompts in portions beside decode steps,
pages given back when a request ends.

	engine = PagedEngine(model, pages=4096)
	a = engine.add([1, 2, 3], steps=20)          # a request: prompt, tokens to generate
	while engine.busy:
		for request, token in engine.step():      # one step of all requests that run
			...
	tokens = engine.results.pop(a)               # all tokens of a request that has ended; they stay until somebody takes them
or engine.generate(prompts, steps).  Decoding is greedy.
"""
from __future__ import annotations

from dataclasses import dataclass, field
from typing import Dict, List, Optional, Sequence, Tuple

import torch

from . import _lib, _paged
from .fused_attention import QuantLlamaAttention, rope_tables
from .fused_attention import rmsnorm as rmsnorm_kernel
from .paged import paged_append, paged_attention, paged_plan


@dataclass
class _Request:
	number: int
	prompt: List[int]
	steps: int
	stop: Optional[int]
	slot: int = -1
	fed: int = 0                                          # tokens in the cache
	out: List[int] = field(default_factory=list)
	pages: List[int] = field(default_factory=list)

	@property
	def pending(self) -> int:
		"""Tokens that are known and not yet in the cache."""
		return len(self.prompt) + len(self.out) - self.fed


class PagedEngine:
	"""pages: of page_size tokens each, shared by all requests (prompts are fastest in pages of 8, 16, 32, 64 or a multiple of 128).  requests: how many
	may run at once.  max_seq: longest request, its generated tokens included (rotary tables, columns of the block table).  portion: prompt
	tokens per step; longer prompts take several steps, in which the others go on decoding."""

	def __init__(self, model, pages: int, page_size: int = 16, requests: int = 16, max_seq: Optional[int] = None, portion: int = 2048, use_graph: bool = True):
		if getattr(model, 'tp_world', 1) != 1:
			raise ValueError('PagedEngine serves models that are not sharded')
		for layer in model.model.layers:
			if not isinstance(layer.self_attn, QuantLlamaAttention):
				raise ValueError('PagedEngine: run make_quant_attn first')
		if pages < 1 or page_size < 1 or not 1 <= requests <= _paged.MAX_REQUESTS or portion < 1:
			raise ValueError(f'PagedEngine: {pages} pages of {page_size}, {requests} requests, portions of {portion}')
		self.model, self.cfg = model, model.config
		self.device = model.lm_head.weight.device
		self.page_size, self.portion, self.use_graph = page_size, portion, use_graph
		self.max_seq = max_seq or self.cfg.max_position_embeddings
		attn = model.model.layers[0].self_attn
		self.heads, self.dim = attn.num_heads, attn.head_dim
		shape = (pages, self.heads, page_size, self.dim)
		zeros = lambda *s, dtype=torch.float16: torch.zeros(s, dtype=dtype, device=self.device)
		self.kcache = [zeros(*shape) for _ in model.model.layers]
		self.vcache = [zeros(*shape) for _ in model.model.layers]
		self.cos, self.sin = rope_tables(self.dim, self.max_seq, attn.rope_theta, device=self.device)          # (those of the layers belong to other engines' captured steps)
		self.table = zeros(requests, -(-self.max_seq // page_size), dtype=torch.int32)
		# what a step reads: cached and new tokens per slot, tokens of the rows, free pages in the order in which they are taken
		self.past, self.new = zeros(requests, dtype=torch.int32), zeros(requests, dtype=torch.int32)
		self.tok = zeros(requests, dtype=torch.int64)
		self.pool, self.head = zeros(pages, dtype=torch.int32), zeros(1, dtype=torch.int32)
		self.free: List[int] = list(range(pages))
		self.reserved = 0                                    # pages that running requests may still take
		self.slots: List[Optional[_Request]] = [None] * requests
		self.waiting: List[_Request] = []
		self.results: Dict[int, List[int]] = {}
		self._numbers = 0
		self.told = zeros(requests + 2, dtype=torch.int32)   # what a step answers: see _tell
		self._graphs: Dict[int, Tuple[torch.cuda.CUDAGraph, torch.Tensor]] = {}
		# of all captures: their stream, the workspace of their projections, their memory (none needs its own while another runs)
		self._stream = self._workspace = self._pool = None
		self._decoding = None                                # the requests that the device buffers are set up for

	# -- requests ------------------------------------------------------------------------------------
	def _needs(self, tokens: int) -> int:
		return -(-tokens // self.page_size)

	def add(self, prompt: Sequence[int], steps: int, stop: Optional[int] = None) -> int:
		"""Queues a request for `steps` tokens behind `prompt` (fewer when `stop` comes up); returns its number."""
		prompt = [int(t) for t in prompt]
		total = len(prompt) + steps - 1                      # (the last token is not fed)
		if not prompt or steps < 1:
			raise ValueError('a request has a prompt of one token at least and generates one token at least')
		if min(prompt) < 0 or max(prompt) >= self.cfg.vocab_size:
			raise ValueError(f'tokens lie in 0 .. {self.cfg.vocab_size - 1}')
		if total > self.max_seq:
			raise ValueError(f'{total} positions, the engine was built for max_seq = {self.max_seq}')
		if self._needs(total) > self.kcache[0].shape[0]:
			raise ValueError(f'{self._needs(total)} pages, the engine has {self.kcache[0].shape[0]}')
		self._numbers += 1
		self.waiting.append(_Request(self._numbers, prompt, int(steps), stop))
		return self._numbers

	@property
	def busy(self) -> bool:
		return bool(self.waiting) or any(r is not None for r in self.slots)

	def _admit(self):
		"""Requests start in the order in which they came, when a slot and the pages of their whole length are free."""
		for slot, r in enumerate(self.slots):
			if r is None and self.waiting:
				need = self._needs(len(self.waiting[0].prompt) + self.waiting[0].steps - 1)
				if need > len(self.free) - self.reserved:
					return
				r = self.waiting.pop(0)
				r.slot, self.slots[slot] = slot, r
				self.reserved += need

	def _finish(self, r: _Request):
		self.free += r.pages
		self.reserved -= self._needs(len(r.prompt) + r.steps - 1) - len(r.pages)
		self.slots[r.slot] = None
		self.results[r.number] = r.out

	def _forget(self, numbers: Sequence[int]):
		self.waiting = [r for r in self.waiting if r.number not in numbers]
		for r in self.slots:
			if r is not None and r.number in numbers:
				self._finish(r)
		self._decoding = None
		for n in numbers:
			self.results.pop(n, None)

	# -- a step --------------------------------------------------------------------------------------
	@torch.no_grad()
	def step(self) -> List[Tuple[int, int]]:
		"""One step: every running request feeds its next token or a portion of its prompt.  Returns (request, token) for those that have
		generated one.  Raises when a kernel has reported a status (see _lib.kernel_status): that step gives no tokens, and the
		requests that took part in it end without results."""
		self._admit()
		running = [r for r in self.slots if r is not None]
		if not running:
			return []
		left, feed = self.portion, {}
		for r in sorted(running, key=lambda r: r.number):    # single tokens always go on; portions share what a step may take, the first request first
			n = r.pending
			if n > 1:
				n = min(n, left)
				left -= n
			feed[r.number] = n
		active = [(r, feed[r.number]) for r in running if feed[r.number]]          # (rows in the order of the slots)
		decode = all(r.pending == 1 for r in running)
		try:
			tokens = self._decode(active) if decode else self._mixed(active)
		except _lib.GptqB200Error:
			self._forget([r.number for r, _ in active])
			raise
		for r, n in active:
			taken = self._needs(r.fed + n) - len(r.pages)
			r.pages += self.free[:taken]
			del self.free[:taken]
			self.reserved -= taken
			r.fed += n
		done = []
		for (r, n), t in zip(active, tokens):
			if r.fed < len(r.prompt):
				continue                                      # a portion inside the prompt
			r.out.append(int(t))
			done.append((r.number, int(t)))
			if len(r.out) == r.steps or t == r.stop:
				self._finish(r)
				self._decoding = None
		return done

	def _tell(self, tokens: torch.Tensor) -> torch.Tensor:
		"""Tokens, and behind them the status words of the layers and of the paged operators: int32 [rows + words]."""
		index = self.device.index
		words = [_lib.status_word(buf) for buf in (_lib._workspaces.get((index, _lib.stream_ptr(self.device))), _paged._control.get(index)) if buf is not None]
		return torch.cat([tokens.to(torch.int32), *words], out=self.told[:len(tokens) + len(words)])

	def _read(self, told: torch.Tensor, rows: int) -> List[int]:
		values = told.tolist()                                # (waits for the device)
		status = 0
		for v in values[rows:]:
			status |= v
		if status != 0:
			raise _lib.GptqB200Error(f'a kernel reported status {status} (see _lib.kernel_status)')
		return values[:rows]

	def _upload(self, active, last: int):
		"""Lengths of the slots 0 .. last - 1 and the pages that the step takes."""
		past, new = [0] * last, [0] * last
		for r, n in active:
			past[r.slot], new[r.slot] = r.fed, n
		ints = torch.tensor(past + new + self.free, dtype=torch.int32).pin_memory().to(self.device, non_blocking=True)
		self.past[:last], self.new[:last] = ints[:last], ints[last:2 * last]
		self.pool[:len(self.free)] = ints[2 * last:]
		self.head.zero_()

	def _plan(self, last: int, rows: int, max_new: int):
		return paged_plan(self.past[:last], self.new[:last], self.table[:last], self.kcache[0], rows, self.heads, pool=self.pool, head=self.head, max_new=max_new)

	def _layers(self, tokens: torch.Tensor, plan) -> torch.Tensor:
		m, H, D = self.model.model, self.heads, self.dim
		h = m.embed_tokens(tokens)
		rows = h.shape[0]
		for i, layer in enumerate(m.layers):
			attn = layer.self_attn
			qkv = attn.qkv_proj(rmsnorm_kernel(h, layer.input_layernorm.weight, layer.input_layernorm.variance_epsilon)).view(rows, 3, H, D)
			q = paged_append(qkv[:, 0], qkv[:, 1], qkv[:, 2], self.kcache[i], self.vcache[i], plan, self.cos, self.sin)
			o = paged_attention(q, self.kcache[i], self.vcache[i], plan)
			h = attn.o_proj(o.view(rows, H * D), residual=h)
			x = rmsnorm_kernel(h, layer.post_attention_layernorm.weight, layer.post_attention_layernorm.variance_epsilon)
			h = layer.mlp(x, residual=h) if hasattr(layer.mlp, 'intermediate') else h + layer.mlp(x)
		return h

	def _greedy(self, h: torch.Tensor) -> torch.Tensor:
		norm = self.model.model.norm
		return self.model.lm_head(rmsnorm_kernel(h.contiguous(), norm.weight, norm.variance_epsilon)).argmax(-1)

	def _mixed(self, active) -> List[int]:
		"""A step with portions of prompts."""
		last = max(r.slot for r, _ in active) + 1
		self._upload(active, last)
		self._decoding = None
		ids, ends = [], []
		for r, n in active:                                  # (in the order of their slots, as the rows are)
			known = r.prompt + r.out
			ids += known[r.fed:r.fed + n]
			ends.append(len(ids) - 1)
		both = torch.tensor(ids + ends, dtype=torch.int64).pin_memory().to(self.device, non_blocking=True)
		h = self._layers(both[:len(ids)], self._plan(last, len(ids), max(n for _, n in active)))
		return self._read(self._tell(self._greedy(h.index_select(0, both[len(ids):]))), len(active))

	def _decode_body(self, last: int) -> torch.Tensor:
		plan = self._plan(last, last, 1)
		self.past[:last] += self.new[:last]
		tok = self._greedy(self._layers(self.tok[:last], plan))
		self.tok[:last].copy_(tok)
		self.head.copy_(plan.head)                           # (behind the plan's own reading of it)
		return self._tell(tok)

	def _slots_served(self, last: int) -> int:
		"""Slots (rows) of a decode step for `last` of them: a few sizes, so that few steps are captured.  Every one up to 8, then four per power of
		two; the slots behind have no new tokens."""
		step = (1 << (last - 1).bit_length()) // 8 if last > 8 else 1
		return min(-(-last // step) * step, len(self.slots))

	def _decode(self, active) -> List[int]:
		"""A step of single tokens; as long as the same requests run, the device buffers carry on by themselves."""
		last = self._slots_served(max(r.slot for r, _ in active) + 1)
		running = [r.number for r, _ in active]
		if self._decoding != running:
			self._upload(active, last)
			known = [(r.prompt + r.out)[r.fed] for r, _ in active]
			self.tok[:len(active)] = torch.tensor(known, dtype=torch.int64).pin_memory().to(self.device, non_blocking=True)
			self._decoding = running
		if not self.use_graph:
			return self._read(self._decode_body(last), last)[:len(active)]
		if last not in self._graphs:
			self._graphs[last] = self._capture(last)
		graph, told = self._graphs[last]
		graph.replay()
		return self._read(told, last)[:len(active)]

	def _capture(self, last: int) -> Tuple[torch.cuda.CUDAGraph, torch.Tensor]:
		# The trial run writes pages and cache rows that the first real step writes again.
		if self._stream is None:
			self._stream, self._workspace, self._pool = torch.cuda.Stream(self.device), _lib.OwnWorkspace(self.device), torch.cuda.graph_pool_handle()
		here, s = torch.cuda.current_stream(self.device), self._stream
		state = (self.past, self.tok, self.head)
		saved = [t.clone() for t in state]
		s.wait_stream(here)
		g = torch.cuda.CUDAGraph()
		with torch.cuda.stream(s), self._workspace:
			self._decode_body(last)
			for t, old in zip(state, saved):
				t.copy_(old)
			s.synchronize()
			with torch.cuda.graph(g, stream=s, pool=self._pool):          # (one at a time is replayed, and what a step leaves lies outside)
				told = self._decode_body(last)
		here.wait_stream(s)
		return g, told

	# -- convenience ---------------------------------------------------------------------------------
	@torch.no_grad()
	def generate(self, prompts: Sequence[Sequence[int]], steps: int, stop: Optional[int] = None) -> List[List[int]]:
		"""Greedy generation for prompts of any lengths: the generated tokens of each."""
		numbers = []
		try:
			for p in prompts:
				numbers.append(self.add(p, steps, stop))
			while self.busy:
				self.step()
			status = _lib.kernel_status(self.device)
			if status != 0:
				raise _lib.GptqB200Error(f'a kernel reported status {status} (see _lib.kernel_status)')
		except Exception:                                     # a prompt is refused, or a step has failed: none of them stays
			self._forget(numbers)
			raise
		return [self.results.pop(n) for n in numbers]

	def close(self):
		"""Releases the captured graphs and their memory."""
		self._graphs.clear()
		self._stream = self._workspace = self._pool = None
