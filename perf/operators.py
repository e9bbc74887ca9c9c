"""Timed cases of serving from a cache in pages: block tables and slot maps from request lengths, rotation of queries and keys with
the store of the new rows, and attention of the new tokens of every request over its pages.

Head counts and sizes are those of the 7B and 65B architectures and of layers with shared key heads; lengths run from one token
behind nothing to a chunk behind tens of thousands.  Pages are dealt out at random, as they are in a pool that has been in use.
"""
import math
import random

import torch

own = False

DEV = 'cuda'
DTYPE = {'fp16': torch.float16, 'bf16': torch.bfloat16, 'fp32': torch.float32}


def listed():
	return [
		# the plan of a decode step of a small server: the smallest call
		{'name': 'plan_24', 'op': 'plan', 'dtype': 'fp16', 'heads': 32, 'kv_heads': 32, 'dim': 128, 'page': 16, 'requests': 24, 'past_lo': 1, 'past_hi': 2000, 'chunk_lo': 1, 'chunk_hi': 1,
		 'singles': 1.0, 'waiting': 0.0, 'pad': 0, 'lengths': 1},
		# the plan of a large server's step: single tokens, portions of prompts, requests that wait, rows left over
		{'name': 'plan_1500', 'op': 'plan', 'dtype': 'bf16', 'heads': 32, 'kv_heads': 8, 'dim': 64, 'page': 32, 'requests': 1500, 'past_lo': 0, 'past_hi': 3000, 'chunk_lo': 2, 'chunk_hi': 400,
		 'singles': 0.7, 'waiting': 0.1, 'pad': 77, 'lengths': 2},
		# new rows of a decode step of a 7B layer
		{'name': 'append_7', 'op': 'append', 'dtype': 'fp16', 'heads': 32, 'kv_heads': 32, 'dim': 128, 'page': 16, 'requests': 7, 'past_lo': 1, 'past_hi': 2000, 'chunk_lo': 1, 'chunk_hi': 1,
		 'singles': 1.0, 'waiting': 0.0, 'pad': 0, 'lengths': 3},
		# new rows of three prompts, 64 heads over 8 key heads
		{'name': 'append_prompts', 'op': 'append', 'dtype': 'bf16', 'heads': 64, 'kv_heads': 8, 'dim': 128, 'page': 64, 'requests': 3, 'past_lo': 0, 'past_hi': 500, 'chunk_lo': 1200, 'chunk_hi': 1900,
		 'singles': 0.0, 'waiting': 0.0, 'pad': 5, 'lengths': 4},
		# one token of one request to a 7B model behind the headline context: latency counts
		{'name': 'decode_1', 'op': 'attention', 'dtype': 'fp16', 'heads': 32, 'kv_heads': 32, 'dim': 128, 'page': 16, 'requests': 1, 'past_lo': 2100, 'past_hi': 2100, 'chunk_lo': 1, 'chunk_hi': 1,
		 'singles': 1.0, 'waiting': 0.0, 'pad': 0, 'lengths': 5},
		# a decode step of many requests of very different lengths, 8 query heads per key head
		{'name': 'decode_48', 'op': 'attention', 'dtype': 'bf16', 'heads': 64, 'kv_heads': 8, 'dim': 128, 'page': 64, 'requests': 48, 'past_lo': 1, 'past_hi': 12000, 'chunk_lo': 1, 'chunk_hi': 1,
		 'singles': 1.0, 'waiting': 0.0, 'pad': 0, 'lengths': 6},
		# a decode step in 32 bits, narrow heads
		{'name': 'decode_fp32', 'op': 'attention', 'dtype': 'fp32', 'heads': 12, 'kv_heads': 4, 'dim': 64, 'page': 16, 'requests': 9, 'past_lo': 300, 'past_hi': 4000, 'chunk_lo': 2, 'chunk_hi': 3,
		 'singles': 0.6, 'waiting': 0.0, 'pad': 0, 'lengths': 7},
		# five drafted tokens of each of sixteen requests
		{'name': 'draft_16', 'op': 'attention', 'dtype': 'fp16', 'heads': 32, 'kv_heads': 8, 'dim': 64, 'page': 32, 'requests': 16, 'past_lo': 300, 'past_hi': 5000, 'chunk_lo': 5, 'chunk_hi': 5,
		 'singles': 0.0, 'waiting': 0.0, 'pad': 0, 'lengths': 8},
		# the prompt of one request to a 7B model, one short of the whole context
		{'name': 'prompt_2047', 'op': 'attention', 'dtype': 'fp16', 'heads': 32, 'kv_heads': 32, 'dim': 128, 'page': 16, 'requests': 1, 'past_lo': 0, 'past_hi': 0, 'chunk_lo': 2047, 'chunk_hi': 2047,
		 'singles': 0.0, 'waiting': 0.0, 'pad': 0, 'lengths': 9},
		# prompts of very different lengths in one batch
		{'name': 'prompts_12', 'op': 'attention', 'dtype': 'bf16', 'heads': 32, 'kv_heads': 8, 'dim': 128, 'page': 128, 'requests': 12, 'past_lo': 0, 'past_hi': 0, 'chunk_lo': 90, 'chunk_hi': 3000,
		 'singles': 0.0, 'waiting': 0.0, 'pad': 0, 'lengths': 10},
		# a portion of a long document behind what has been read of it
		{'name': 'chunk_512', 'op': 'attention', 'dtype': 'bf16', 'heads': 64, 'kv_heads': 8, 'dim': 128, 'page': 64, 'requests': 1, 'past_lo': 30001, 'past_hi': 30001, 'chunk_lo': 512, 'chunk_hi': 512,
		 'singles': 0.0, 'waiting': 0.0, 'pad': 0, 'lengths': 11},
		# a server's step: mostly single tokens, some portions of prompts among them
		{'name': 'mixed_40', 'op': 'attention', 'dtype': 'fp16', 'heads': 32, 'kv_heads': 32, 'dim': 128, 'page': 16, 'requests': 40, 'past_lo': 0, 'past_hi': 2000, 'chunk_lo': 100, 'chunk_hi': 512,
		 'singles': 0.85, 'waiting': 0.0, 'pad': 3, 'lengths': 12},
	]


def _log(rng, lo, hi):
	return int(round(math.exp(rng.uniform(math.log(lo + 1), math.log(hi + 1))))) - 1


def draw(rng):
	heads, kv_heads = rng.choice([(32, 32), (32, 32), (40, 40), (64, 64), (32, 8), (64, 8), (40, 8), (28, 4), (12, 4), (16, 1)])
	case = {'dtype': rng.choice(['fp16', 'fp16', 'bf16', 'bf16']), 'heads': heads, 'kv_heads': kv_heads, 'dim': rng.choice([128, 128, 128, 64, 96]), 'page': rng.choice([16, 16, 32, 64, 128]),
			'waiting': 0.0, 'pad': rng.choice([0, 0, rng.randint(1, 50)]), 'lengths': rng.randint(100, 1 << 30)}
	kind = rng.choice(['plan', 'append', 'decode', 'decode', 'prompt', 'chunk', 'mixed', 'draft'])
	case['op'] = kind if kind in ('plan', 'append') else 'attention'
	if kind == 'plan':
		case.update(requests=_log(rng, 1, 1500), past_lo=0, past_hi=_log(rng, 1, 3000), chunk_lo=2, chunk_hi=_log(rng, 3, 400), singles=rng.choice([1.0, 0.7, 0.1]), waiting=rng.choice([0.0, 0.1]))
	elif kind == 'append':
		hi = _log(rng, 1, 1900)
		case.update(requests=_log(rng, 1, max(1, 5000 // hi)) if hi > 40 else _log(rng, 1, 128), past_lo=0, past_hi=_log(rng, 1, 1000), chunk_lo=max(1, hi // 2), chunk_hi=hi, singles=rng.choice([1.0, 0.0]))
	elif kind == 'decode':
		hi = _log(rng, 16, 12000)
		case.update(requests=_log(rng, 1, max(1, min(256, 128 * 8 * 2000 // (hi * kv_heads)))), past_lo=rng.choice([0, hi // 2]), past_hi=hi, chunk_lo=1, chunk_hi=1, singles=1.0)
		if rng.random() < 0.15:
			case['dtype'] = 'fp32'
	elif kind == 'draft':
		n = rng.randint(2, 9)
		case.update(requests=_log(rng, 1, 32), past_lo=20, past_hi=_log(rng, 100, 4000), chunk_lo=n, chunk_hi=n, singles=0.0)
	elif kind == 'prompt':
		hi = _log(rng, 60, 3000)
		case.update(requests=_log(rng, 1, max(1, 6000 // hi)), past_lo=0, past_hi=0, chunk_lo=max(1, hi // rng.choice([1, 2, 20])), chunk_hi=hi, singles=0.0)
	elif kind == 'chunk':
		case.update(requests=rng.choice([1, 1, 2]), past_lo=500, past_hi=_log(rng, 1000, 14000), chunk_lo=20, chunk_hi=_log(rng, 30, 512), singles=0.0)
	else:
		case.update(requests=_log(rng, 4, 48), past_lo=0, past_hi=_log(rng, 100, 2000), chunk_lo=20, chunk_hi=_log(rng, 30, 512), singles=0.85)
	return case


# ---- lengths and inputs ----------------------------------------------------------------------------------------------------
def lengths(case):
	"""(tokens in the cache, new tokens) of every request: they belong to the case, inputs to the seed."""
	rng = random.Random(case['lengths'])
	out = []
	for _ in range(case['requests']):
		past = _log(rng, case['past_lo'], case['past_hi'])
		new = 1 if rng.random() < case['singles'] else _log(rng, case['chunk_lo'], case['chunk_hi'])
		out.append((past, 0 if rng.random() < case['waiting'] else new))
	return out


def _pages(n, page):
	return (n + page - 1) // page


def _inputs(case, seed):
	gen = torch.Generator(device=DEV).manual_seed(seed)
	rng = random.Random(seed)
	lens = lengths(case)
	page, H, G, D, dt = case['page'], case['heads'], case['kv_heads'], case['dim'], DTYPE[case['dtype']]
	rows = sum(n for _, n in lens) + case['pad']
	old = [_pages(p, page) for p, _ in lens]
	full = [_pages(p + n, page) for p, n in lens]
	total, width = sum(full) + 7, max(max(full), 1) + 2
	ids = list(range(total))
	rng.shuffle(ids)
	have = old if case['op'] == 'plan' else full          # the plan deals out the rest
	table, at = torch.full((len(lens), width), -1, dtype=torch.int32), 0
	for r, n in enumerate(have):
		table[r, :n] = torch.tensor(ids[at:at + n], dtype=torch.int32)
		at += n
	s = {'case': case, 'lens': lens, 'rows': rows, 'valid': rows - case['pad'], 'table': table.to(DEV), 'full': full,
		 'past': torch.tensor([p for p, _ in lens], dtype=torch.int32, device=DEV), 'new': torch.tensor([n for _, n in lens], dtype=torch.int32, device=DEV)}
	if case['op'] == 'plan':
		s['pool'] = torch.tensor(ids[:2] + ids[at:], dtype=torch.int32, device=DEV)          # two of them are taken already
		s['head'] = torch.tensor([2], dtype=torch.int32, device=DEV)
		s['k'] = torch.empty((total, G, page, D), dtype=dt, device=DEV)          # (its sizes count here)
		return s
	randn = lambda *shape: torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32).to(dt)
	s['k'], s['v'] = randn(total, G, page, D), randn(total, G, page, D)
	if case['op'] == 'append':
		qkv = randn(rows, (H + 2 * G) * D)          # the rows of a fused projection
		s['q'], s['k_new'], s['v_new'] = qkv[:, :H * D].view(rows, H, D), qkv[:, H * D:(H + G) * D].view(rows, G, D), qkv[:, (H + G) * D:].view(rows, G, D)
		top = max(p + n for p, n in lens)
		angle = torch.outer(torch.arange(top, dtype=torch.float64, device=DEV), 10000.0 ** (-torch.arange(0, D, 2, dtype=torch.float64, device=DEV) / D))
		s['cos'], s['sin'] = torch.cat([angle, angle], 1).cos().to(dt), torch.cat([angle, angle], 1).sin().to(dt)
	else:
		s['q'] = randn(rows, H, D)
	pos = [p + i for p, n in lens for i in range(n)] + [0] * case['pad']
	tab = table.tolist()
	slot = [tab[r][(p + i) // page] * page + (p + i) % page for r, (p, n) in enumerate(lens) for i in range(n)] + [-1] * case['pad']
	s['pos'], s['slots'] = torch.tensor(pos, device=DEV), torch.tensor(slot, device=DEV)
	return s


def prepare(case, seed):
	s = _inputs(case, seed)
	if own and case['op'] != 'plan':
		from gptq_triton_b200 import paged_plan
		s['plan'] = paged_plan(s['past'], s['new'], s['table'], s['k'], s['rows'], case['heads'], max_new=max(n for _, n in s['lens']))
	return s


# ---- plain forms -----------------------------------------------------------------------------------------------------------
def _plain_plan(s):
	past, new, page = s['past'], s['new'], s['case']['page']
	start = torch.cat([torch.zeros_like(new[:1]), torch.cumsum(new, 0, dtype=torch.int32)])
	lens = past + new
	old, full = (past + page - 1) // page, (lens + page - 1) // page
	take = full - old
	off = torch.cumsum(take, 0, dtype=torch.int32) - take
	col = torch.arange(s['table'].shape[1], dtype=torch.int32, device=DEV)[None]
	fresh = (col >= old[:, None]) & (col < full[:, None])
	source = (s['head'] + off[:, None] + col - old[:, None]).clamp(0, s['pool'].numel() - 1)
	table = torch.where(fresh, s['pool'][source.long()], s['table'])
	row = torch.arange(s['rows'], dtype=torch.int32, device=DEV)
	req = torch.searchsorted(start[1:].contiguous(), row, right=True).clamp(max=new.numel() - 1)
	used = row < start[-1]
	pos = torch.where(used, past[req] + row - start[req], 0)
	slots = torch.where(used, table[req, (pos // page).long()].long() * page + pos % page, -1)
	return [table, start, lens, pos, slots, s['head'] + take.sum(0, keepdim=True, dtype=torch.int32)]


def _turn(x, cos, sin):
	half = x.shape[-1] // 2
	return x * cos + torch.cat([-x[..., half:], x[..., :half]], -1) * sin


def _plain_append(s):
	page, n = s['case']['page'], s['valid']
	cos, sin = s['cos'][s['pos']].float()[:, None], s['sin'][s['pos']].float()[:, None]
	q = _turn(s['q'].float(), cos, sin).to(s['q'].dtype)
	k = _turn(s['k_new'][:n].float(), cos[:n], sin[:n]).to(q.dtype)
	where, at = s['slots'][:n] // page, s['slots'][:n] % page
	s['k'][where, :, at] = k
	s['v'][where, :, at] = s['v_new'][:n]
	return [q, s['k'], s['v']]


def _plain_attention(s):
	case = s['case']
	H, G, D, page = case['heads'], case['kv_heads'], case['dim'], case['page']
	out, at = torch.zeros_like(s['q']), 0
	for r, (past, n) in enumerate(s['lens']):
		if n:
			S = past + n
			ids = s['table'][r, :_pages(S, page)].long()
			hidden = torch.arange(S, device=DEV)[None] > torch.arange(past, S, device=DEV)[:, None]
			per = max(1, min(G, (1 << 28) // (n * S * (H // G))))          # key heads at a time
			for g in range(0, G, per):
				e = min(G, g + per)
				k, v = (t[ids, g:e].transpose(0, 1).reshape(e - g, -1, D)[:, :S].float() for t in (s['k'], s['v']))
				q = s['q'][at:at + n, g * (H // G):e * (H // G)].float().reshape(n, e - g, H // G, D).permute(1, 2, 0, 3)
				x = (q @ k[:, None].transpose(-1, -2)) * (1.0 / math.sqrt(D))
				x = x.masked_fill(hidden, float('-inf'))
				x = torch.exp(x - x.amax(-1, keepdim=True))
				o = (x @ v[:, None]) / x.sum(-1, keepdim=True)
				out[at:at + n, g * (H // G):e * (H // G)] = o.permute(2, 0, 1, 3).reshape(n, -1, D).to(out.dtype)
		at += n
	return [out[:s['valid']]]


def run(s):
	op = s['case']['op']
	if not own:
		return _plain_plan(s) if op == 'plan' else _plain_append(s) if op == 'append' else _plain_attention(s)
	from gptq_triton_b200 import paged_append, paged_attention, paged_plan
	if op == 'plan':
		p = paged_plan(s['past'], s['new'], s['table'], s['k'], s['rows'], s['case']['heads'], pool=s['pool'], head=s['head'], max_new=s['case']['chunk_hi'])
		return [p.table, p.row_start, p.lens, p.positions, p.slots, p.head]
	if op == 'append':
		return [paged_append(s['q'], s['k_new'], s['v_new'], s['k'], s['v'], s['plan'], s['cos'], s['sin']), s['k'], s['v']]
	return [paged_attention(s['q'], s['k'], s['v'], s['plan'])[:s['valid']]]


# ---- 64 bits ---------------------------------------------------------------------------------------------------------------
def exact(case, seed):
	s = _inputs(case, seed)
	H, G, D, page, lens = case['heads'], case['kv_heads'], case['dim'], case['page'], s['lens']
	if case['op'] == 'plan':
		table, pool, head = s['table'].tolist(), s['pool'].tolist(), int(s['head'])
		start, pos, slots = [0], [], []
		for r, (past, n) in enumerate(lens):
			for c in range(_pages(past, page), _pages(past + n, page)):
				table[r][c] = pool[head]
				head += 1
			start.append(start[-1] + n)
			for p in range(past, past + n):
				pos.append(p)
				slots.append(table[r][p // page] * page + p % page)
		i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
		return [i32(table), i32(start), i32([p + n for p, n in lens]), i32(pos + [0] * case['pad']), torch.tensor(slots + [-1] * case['pad'], device=DEV), i32([head])]
	if case['op'] == 'append':
		def rotated(x):
			x, c, d = x.double(), s['cos'].double()[s['pos']].unsqueeze(1), s['sin'].double()[s['pos']].unsqueeze(1)
			a, b = x.split(D // 2, -1)
			return torch.cat([a * c[..., :D // 2] - b * d[..., :D // 2], b * c[..., D // 2:] + a * d[..., D // 2:]], -1)
		flat = lambda t: t.double().transpose(1, 2).reshape(-1, G, D)          # rows by slot
		back = lambda t: t.reshape(-1, page, G, D).transpose(1, 2)
		k, v, n = flat(s['k']), flat(s['v']), s['valid']
		k.index_copy_(0, s['slots'][:n], rotated(s['k_new'])[:n])
		v.index_copy_(0, s['slots'][:n], s['v_new'].double()[:n])
		return [rotated(s['q']), back(k), back(v)]
	out, first = torch.zeros((s['valid'], H, D), dtype=torch.float64, device=DEV), 0
	for r, (past, n) in enumerate(lens):
		if n == 0:
			continue
		j = torch.arange(past + n, device=DEV)
		where, inside = s['table'][r].long()[j // page], j % page
		lower = j[None, :] <= torch.arange(past, past + n, device=DEV)[:, None]
		for h in range(H):
			g = h * G // H
			score = torch.mm(s['q'][first:first + n, h].double(), s['k'][where, g, inside].double().t()) / math.sqrt(D)
			p = torch.where(lower, torch.exp(score - torch.where(lower, score, -math.inf).max(1, keepdim=True).values), 0.0)
			out[first:first + n, h] = torch.mm(p, s['v'][where, g, inside].double()) / p.sum(1, keepdim=True)
		first += n
	return [out]


# ---- what a pass cannot do without -----------------------------------------------------------------------------------------
def work(case):
	lens = lengths(case)
	H, G, D, page = case['heads'], case['kv_heads'], case['dim'], case['page']
	size, rows, R = (4 if case['dtype'] == 'fp32' else 2), sum(n for _, n in lens), len(lens)
	taken = sum(_pages(p + n, page) - _pages(p, page) for p, n in lens)
	if case['op'] == 'plan':
		return {'bytes': 16 * R + 8 * taken + 12 * (rows + case['pad']), 'flops': 2 * (R + rows)}
	if case['op'] == 'append':
		top = len({p + i for p, n in lens for i in range(n)})
		return {'bytes': size * D * (2 * rows * (H + 2 * G) + 2 * top) + 12 * rows, 'flops': 3 * rows * (H + G) * D}
	seen = sum(p + n for p, n in lens if n)
	pairs = sum(n * p + n * (n + 1) // 2 for p, n in lens)
	return {'bytes': size * D * (2 * rows * H + 2 * seen * G) + 4 * sum(_pages(p + n, page) for p, n in lens if n), 'flops': 4 * D * H * pairs}
