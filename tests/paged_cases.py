"""Inputs of the paged-cache tests: requests of given lengths, their pages dealt out at random, everything that no request owns filled
with NaN."""
import random

import torch

DTYPES = {'fp16': torch.float16, 'bf16': torch.bfloat16, 'fp32': torch.float32}


def ceil(n, page):
	return -(-n // page)


class Step:
	"""past, new: lists.  Caches [pages, kv_heads, page, dim] on the CPU; a few keys of every request stand out (weights of all sizes)."""

	def __init__(self, past, new, heads, kv_heads, dim, page, dtype, seed=0, pad=0, filled=True, spare=3, fill=float('nan'), together=False):
		g, rng = torch.Generator().manual_seed(seed), random.Random(seed)
		self.past, self.new, self.heads, self.kv_heads, self.dim, self.page = list(past), list(new), heads, kv_heads, dim, page
		self.dtype = DTYPES[dtype]
		self.rows = sum(new) + pad
		full = [ceil(p + n, page) for p, n in zip(past, new)]
		self.pages, self.width = sum(full) + spare, max(full + [1]) + 1
		ids = list(range(self.pages))
		rng.shuffle(ids)
		self.table, at = [], 0
		for n in full:
			self.table.append(ids[at:at + n] + [-1] * (self.width - n))
			at += n
		shape = (self.pages, kv_heads, page, dim)
		both = torch.full((2, *shape) if not together else (self.pages, 2, kv_heads, page, dim), fill).to(self.dtype)
		self.k, self.v = (both[0], both[1]) if not together else (both[:, 0], both[:, 1])          # together: strides between pages
		for r in range(len(past)):
			L = past[r] + (new[r] if filled else 0)
			j = torch.arange(L)
			where = torch.tensor(self.table[r], dtype=torch.long)[j // page] if L else j
			k = torch.randn(L, kv_heads, dim, generator=g)
			if L:
				k *= torch.where(torch.rand(L, 1, 1, generator=g) < 0.1, 3.0, 1.0)
			self.k[where, :, j % page] = k.to(self.dtype)
			self.v[where, :, j % page] = torch.randn(L, kv_heads, dim, generator=g).to(self.dtype)
		self.qkv = torch.randn(self.rows, (heads + 2 * kv_heads) * dim, generator=g).to(self.dtype)

	def parts(self, qkv=None):
		"""Queries, keys and values as columns of the rows of a fused projection."""
		t, H, G, D = self.qkv if qkv is None else qkv, self.heads, self.kv_heads, self.dim
		return t[:, :H * D].unflatten(1, (H, D)), t[:, H * D:(H + G) * D].unflatten(1, (G, D)), t[:, (H + G) * D:].unflatten(1, (G, D))

	def ints(self, v, device='cuda'):
		return torch.tensor(v, dtype=torch.int32, device=device)


def bound(exact, absolute, score, dim, keys, dtype, p_bits=True):
	"""How far a kernel may be from `exact` per element.  A = `absolute` = sum p |v|, B = `score` = max scale sum |q k|.
	Output: half a step of the type, u |out|.  Weights that are multiplied in the type (p_bits): half a step each, u A.  Scores: a sum of
	dim products in fp32 is off by at most (dim + 16) 2^-24 B (scale and base included), which a weight and the sum of weights take on as
	a factor each; the exponential 2^-20 of a weight.  Sums over the keys in fp32: (keys + 64) 2^-24 of A, and of the sum of weights."""
	u = torch.finfo(dtype).eps / 2
	weight = 2 * ((dim + 16) * 2.0 ** -24 * score + 2.0 ** -20 + (keys + 64) * 2.0 ** -24)
	# (products with an output already off by `weight` and u A; a subnormal step of fp16 results)
	tiny = 2.0 ** -25 if dtype == torch.float16 else 1e-30
	return 1.01 * (u * exact.abs() + absolute * ((u if p_bits and dtype != torch.float32 else 0.0) + weight)) + tiny
