"""64-bit restatement of the paged-cache operators, written from their definitions (CPU, torch and plain Python)."""
import math

import torch


def plan(past, new, table, page, rows, pool=None, head=0):
	"""past, new: lists; table: list of lists (changed in place).  Returns row_start, lens, positions, slots, the place in the pool behind the
	pages taken."""
	ceil = lambda n: -(-n // page)
	start, pos, slots = [0], [], []
	for r, (p, n) in enumerate(zip(past, new)):
		if pool is not None:
			for c in range(ceil(p), ceil(p + n)):
				table[r][c] = pool[head]
				head += 1
		for i in range(p, p + n):
			pos.append(i)
			slots.append(table[r][i // page] * page + i % page)
		start.append(start[-1] + n)
	pad = rows - len(pos)
	return start, [p + n for p, n in zip(past, new)], pos + [0] * pad, slots + [-1] * pad, head


def rotate(x, cos, sin):
	"""x [rows, heads, dim] by the table rows cos, sin [rows, rot]; the entries behind rot stay."""
	x, cos, sin = x.double(), cos.double()[:, None], sin.double()[:, None]
	rot = cos.shape[-1]
	half = rot // 2
	a, b = x[..., :half], x[..., half:rot]
	return torch.cat([a * cos[..., :half] - b * sin[..., :half], b * cos[..., half:] + a * sin[..., half:], x[..., rot:]], -1)


def attention(q, k_cache, v_cache, table, row_start, lens, scale=None):
	"""out [rows in use, heads, dim], and per element what errors of a kernel are measured by: A = sum p |v|, per row B = the largest
	scale * sum |q k|."""
	rows, (_, heads, dim), (_, kv_heads, page, _) = row_start[-1], q.shape, k_cache.shape
	scale = 1 / math.sqrt(dim) if scale is None else scale
	out, absolute, score = torch.zeros(rows, heads, dim, dtype=torch.float64), torch.zeros(rows, heads, dim, dtype=torch.float64), torch.zeros(rows, heads, 1, dtype=torch.float64)
	for r, L in enumerate(lens):
		a, b = row_start[r], row_start[r + 1]
		if a == b:
			continue
		pos = torch.arange(L - (b - a), L)
		j = torch.arange(L)
		where = torch.tensor([table[r][c] for c in range(-(-L // page))], dtype=torch.long)[j // page] if L else j
		seen = j[None] <= pos[:, None]
		for g in range(kv_heads):
			k, v = k_cache[where, g, j % page].double(), v_cache[where, g, j % page].double()
			for h in range(g * heads // kv_heads, (g + 1) * heads // kv_heads):
				x = q[a:b, h].double()
				s = (x @ k.T * scale).masked_fill(~seen, -math.inf)
				p = torch.softmax(s, -1).masked_fill(~seen, 0.0)
				out[a:b, h], absolute[a:b, h] = p @ v, p @ v.abs()
				score[a:b, h, 0] = ((x.abs() @ k.abs().T) * scale).masked_fill(~seen, 0.0).amax(-1) if L else 0.0
				none = pos < 0
				out[a:b, h][none], absolute[a:b, h][none] = 0.0, 0.0
	return out, absolute, score
