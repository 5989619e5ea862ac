"""The paged key-value cache's operators, as cases to be measured: append, attend (one new token per sequence) and evict.

Each case is one call as a serving loop makes it. `own` selects the library's kernels (tacotron_amd.kv_cache.KvCache) or
their plain form in elementary torch operations."""
import math

import numpy as np
import torch

own = False

DTYPES = {'float32': torch.float32, 'bfloat16': torch.bfloat16, 'float16': torch.float16}
SIZES = {'float32': 4, 'bfloat16': 2, 'float16': 2}


# ---------------------------------------------------------------------------------------
# cases
def _attend(name, B, cap, hq, hkv, d, page, dtype, mass, ragged):
    return {'name': name, 'op': 'attend', 'B': B, 'cap': cap, 'hq': hq, 'hkv': hkv, 'd': d, 'page': page, 'dtype': dtype,
            'mass': mass, 'ragged': ragged}


def _append(name, B, cap, T, hq, hkv, d, page, dtype, ragged):
    return {'name': name, 'op': 'append', 'B': B, 'cap': cap, 'T': T, 'hq': hq, 'hkv': hkv, 'd': d, 'page': page,
            'dtype': dtype, 'ragged': ragged}


def _evict(name, B, cap, budget, recent, hkv, d, page, dtype, ragged):
    return {'name': name, 'op': 'evict', 'B': B, 'cap': cap, 'budget': budget, 'recent': recent, 'hkv': hkv, 'd': d,
            'page': page, 'dtype': dtype, 'ragged': ragged}


def listed():
    return [
        # the encoder memories of a batch of 32 utterances of up to 150 characters, one head of depth 256, fp32
        _attend('attend-memory-f32', 32, 160, 1, 1, 256, 16, 'float32', True, True),
        # one sequence of some thousand tokens alone on the card: latency
        _attend('attend-one-bf16', 1, 8190, 32, 8, 128, 16, 'bfloat16', True, False),
        # an ordinary serving batch, lengths from a quarter of the table to all of it, one row empty
        _attend('attend-batch-bf16', 64, 4096, 32, 8, 128, 16, 'bfloat16', True, True),
        # two very long sequences, eight query heads to a key head, weights not collected
        _attend('attend-long-f16', 2, 131072, 16, 2, 64, 64, 'float16', False, False),
        # a full pool: 32 long sequences
        _attend('attend-pool-bf16', 32, 32768, 32, 8, 128, 32, 'bfloat16', True, True),
        # one new token for each of 64 sequences, out of a fused projection
        _append('append-step-bf16', 64, 2048, 1, 32, 8, 128, 16, 'bfloat16', False),
        # the memories of 32 utterances written once
        _append('append-memory-f32', 32, 160, 150, 0, 1, 256, 16, 'float32', True),
        # prompts of thousands of tokens
        _append('append-prompt-bf16', 8, 8192, 4097, 32, 8, 128, 16, 'bfloat16', True),
        # steady state: every sequence is one token over its budget
        _evict('evict-step-bf16', 32, 2064, 2048, 256, 8, 128, 16, 'bfloat16', False),
        # alignments' worth of memory dropped from ragged fp32 sequences, odd budget
        _evict('evict-ragged-f32', 16, 8192, 3001, 64, 2, 64, 32, 'float32', True),
        # long prompts cut to an eighth
        _evict('evict-long-bf16', 4, 65536, 8192, 512, 8, 128, 16, 'bfloat16', False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(['attend', 'attend', 'append', 'evict'])
    dtype = rng.choice(['float32', 'bfloat16', 'bfloat16', 'float16'])
    d, page = rng.choice([64, 128, 256]), rng.choice([8, 16, 32, 64, 128])
    hkv, group = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 2, 3, 4, 5, 8, 16])
    B, cap = _log(rng, 1, 96), _log(rng, 24, 65536)
    rows = (1 << 29) // (hkv * d * SIZES[dtype])    # half a GiB of keys at most
    cap = max(24, min(cap, rows // B))
    ragged = B > 1 and rng.random() < 0.7
    if op == 'attend':
        c = _attend('', B, cap, hkv * group, hkv, d, page, dtype, rng.random() < 0.6, ragged)
    elif op == 'append':
        T = min(_log(rng, 1, 4000), cap)
        c = _append('', B, cap, T, hkv * group, hkv, d, page, dtype, ragged)
    else:
        budget = min(cap - 1, _log(rng, 8, cap))
        c = _evict('', B, cap, budget, rng.randrange(0, budget // 2 + 1), hkv, d, page, dtype, ragged)
    del c['name']
    return c


def _lengths(c):
    """Tokens per sequence (before the seed shuffles them): all the table's, or from a quarter of it up, one row empty."""
    if c['op'] == 'append':
        starts = [c['cap'] - c['T']] * c['B']
        return [s * (i + 1) // c['B'] for i, s in enumerate(starts)] if c['ragged'] else starts
    full = c['cap'] if c['op'] == 'attend' or c['cap'] - c['budget'] > 16 else c['budget'] + 1
    if not c['ragged']:
        return [full] * c['B']
    lens = [full // 4 + (full - full // 4) * i // max(c['B'] - 1, 1) for i in range(c['B'])]
    if c['B'] >= 8:
        lens[1] = 0
    return lens


def _counts(c):
    """New tokens per sequence of an append: all T, or from half of T up."""
    return [c['T'] - (c['T'] // 2) * i // c['B'] for i in range(c['B'])] if c['ragged'] else [c['T']] * c['B']


def work(case):
    c, e = case, SIZES[case['dtype']]
    if c['op'] == 'attend':
        n = sum(_lengths(c))
        side = 8 * n * c['hkv'] if c['mass'] else 0
        return {'bytes': 2 * e * n * c['hkv'] * c['d'] + side + 2 * e * c['B'] * c['hq'] * c['d'],
                'flops': 4 * n * c['hq'] * c['d']}
    if c['op'] == 'append':
        n = sum(_counts(c))
        return {'bytes': n * c['hkv'] * (4 * e * c['d'] + 8), 'flops': 0}
    # rows that move: those kept from beyond the budget, when every unprotected token is as likely to be kept
    total = 0.0
    for L in _lengths(c):
        n = min(L, c['budget'])
        r = min(c['recent'], n)
        moved = (L - n) * n / L if L > n else 0
        total += 8 * L + 8 * c['cap'] + (4 * e * c['d'] * moved if r < n else 0)
    return {'bytes': total * c['hkv'], 'flops': 0}


# ---------------------------------------------------------------------------------------
# inputs
def _pages(c):
    return -(-c['cap'] // c['page'])


def prepare(case, seed):
    c, dev, dtype = case, torch.device('cuda'), DTYPES[case['dtype']]
    g = torch.Generator(device=dev).manual_seed(int(seed))
    B, hkv, d, page, mp = c['B'], c['hkv'], c['d'], c['page'], _pages(c)
    cap = mp * page
    lens = _lengths(c)
    order = torch.randperm(B, generator=g, device=dev)
    lengths = torch.tensor(lens, dtype=torch.int32, device=dev)[order].contiguous()
    # a pool in use: pages in no order, the last one spare; table entries behind a sequence name the spare page, which
    # holds what nobody wrote
    k_pages = torch.randn(B * mp + 1, hkv, page, d, generator=g, device=dev, dtype=dtype)
    v_pages = torch.randn(B * mp + 1, hkv, page, d, generator=g, device=dev, dtype=dtype)
    k_pages[-1] = float('nan')
    v_pages[-1] = float('nan')
    table = torch.randperm(B * mp, generator=g, device=dev).view(B, mp).to(torch.int32)
    s = {'case': c, 'k_pages': k_pages, 'v_pages': v_pages}
    top = lengths
    if c['op'] == 'append':
        counts = torch.tensor(_counts(c), dtype=torch.int32, device=dev)[order].contiguous()
        top = lengths + counts
        # rows come out of one projection, queries beside them
        qkv = torch.randn(B, c['T'], c['hq'] + 2 * hkv, d, generator=g, device=dev, dtype=dtype)
        s['k'], s['v'] = qkv[:, :, c['hq']:c['hq'] + hkv], qkv[:, :, c['hq'] + hkv:]
        s['starts'], s['counts'] = lengths, counts
        s['first'] = lengths + torch.randint(0, 1000, (B,), generator=g, device=dev, dtype=torch.int32)
    used = -(-top.to(torch.int64) // page)
    s['table'] = torch.where(torch.arange(mp, device=dev)[None] < used[:, None], table, B * mp).to(torch.int32)
    s['lengths'] = lengths
    live = torch.arange(cap, device=dev)[None, None] < lengths[:, None, None]
    # attention gathered over many steps: a few tokens hold most of it, tokens that were just appended hold none
    mass = torch.rand(B, hkv, cap, generator=g, device=dev).clamp_(1e-6).log_().mul_(-1).square_()
    fresh = torch.arange(cap, device=dev)[None, None] >= lengths[:, None, None] - 4
    s['mass'] = torch.where(live & ~fresh, mass, torch.zeros((), device=dev))
    if c['op'] != 'attend':
        # tokens stand in no order once an eviction has filled gaps
        pos = torch.rand(B, hkv, cap, generator=g, device=dev).masked_fill_(~live, 2.0).argsort(-1).argsort(-1)
        s['positions'] = torch.where(live, pos, -1).to(torch.int32)
    if c['op'] == 'attend':
        s['q'] = torch.randn(B, c['hq'] + 2 * hkv, d, generator=g, device=dev, dtype=dtype)[:, :c['hq']]
        s['scale'] = 1.5 / math.sqrt(d)
    return s


# ---------------------------------------------------------------------------------------
# the plain form
def _gather(pages, table):
    """[B, hkv, cap, d] in 32 bits: the pages of each sequence one after the other."""
    B, mp = table.shape
    P, hkv, page, d = pages.shape
    return pages[table.long()].permute(0, 2, 1, 3, 4).reshape(B, hkv, mp * page, d).float()


def _plain_attend(s):
    c = s['case']
    B, hkv, d = c['B'], c['hkv'], c['d']
    cap = s['mass'].shape[2]
    live = (torch.arange(cap, device=s['q'].device)[None] < s['lengths'][:, None])[:, None, None, :]
    q = s['q'].float().reshape(B, hkv, -1, d)
    S = torch.matmul(_gather(s['k_pages'], s['table']), q.transpose(-1, -2).contiguous()).transpose(-1, -2) * s['scale']
    S = torch.where(live, S, float('-inf'))
    m = S.amax(-1, keepdim=True)
    m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
    p = torch.exp(S - m)
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    v = torch.where(live.transpose(-1, -2), _gather(s['v_pages'], s['table']), torch.zeros((), device=p.device))
    out = torch.matmul(p, v).reshape(B, c['hq'], d).to(s['q'].dtype)
    lse = (m + torch.log(total)).reshape(B, c['hq'])
    if c['mass']:
        s['mass'] += p.sum(2)
        return out, lse, s['mass']
    return out, lse


def _rows(table, slots, hkv, page):
    """Row of the flattened pool [pages * hkv * page, d] that holds slot slots[b, h, i]."""
    B = table.shape[0]
    ids = torch.gather(table.long()[:, None].expand(B, hkv, -1), 2, slots // page)
    return (ids * hkv + torch.arange(hkv, device=slots.device)[None, :, None]) * page + slots % page


def _plain_append(s):
    c = s['case']
    B, hkv, d, page, T = c['B'], c['hkv'], c['d'], c['page'], c['T']
    t = torch.arange(T, device=s['k'].device)[None]
    b, i = torch.nonzero(t < s['counts'][:, None], as_tuple=True)
    slot = s['starts'].long()[b] + i
    page_id = s['table'].long()[b, slot // page]
    s['k_pages'][page_id, :, slot % page] = s['k'][b, i]
    s['v_pages'][page_id, :, slot % page] = s['v'][b, i]
    s['mass'][b, :, slot] = 0.0
    s['positions'][b, :, slot] = (s['first'].long()[b] + i).to(torch.int32)[:, None]
    return s['k_pages'], s['v_pages'], s['starts'] + s['counts'], s['mass'], s['positions']


def _plain_evict(s):
    c = s['case']
    B, hkv, d, page, budget = c['B'], c['hkv'], c['d'], c['page'], c['budget']
    mass, pos, L = s['mass'], s['positions'], s['lengths'].long()[:, None, None]
    cap = mass.shape[2]
    slot = torch.arange(cap, device=mass.device)[None, None].expand(B, hkv, cap)
    live = slot < L
    newest = torch.where(live, pos, -1).amax(-1, keepdim=True)
    key = torch.where(live & (pos > newest - c['recent']), float('inf'), mass)
    key = torch.where(live, key, float('-inf'))
    best = torch.argsort(key, dim=-1, descending=True, stable=True)[:, :, :budget]
    kept = torch.zeros_like(live).scatter_(2, best, True) & live
    n = L.clamp(max=budget)
    late = kept & (slot >= n)
    hole = ~kept & (slot < n)
    taken = torch.argsort(late.to(torch.uint8), dim=-1, descending=True, stable=True)
    rank = (hole.cumsum(-1) - 1).clamp_(min=0)
    src = torch.where(hole, torch.gather(taken, 2, rank), slot)
    new_mass = torch.where(slot < n, torch.gather(mass, 2, src), torch.zeros((), device=mass.device))
    new_pos = torch.where(slot < n, torch.gather(pos, 2, src), -1).to(torch.int32)
    # only slots below the budget are written; where nothing moves a row is written over itself
    to, fro = _rows(s['table'], slot[:, :, :budget], hkv, page), _rows(s['table'], src[:, :, :budget], hkv, page)
    k, v = s['k_pages'].view(-1, d), s['v_pages'].view(-1, d)
    k[to.reshape(-1)] = k[fro.reshape(-1)]
    v[to.reshape(-1)] = v[fro.reshape(-1)]
    return s['k_pages'], s['v_pages'], n.reshape(B).to(torch.int32), new_mass, new_pos


def run(state):
    s, c = state, state['case']
    if not own:
        return {'attend': _plain_attend, 'append': _plain_append, 'evict': _plain_evict}[c['op']](s)
    if 'cache' not in s:    # the pool's handle, which a serving loop keeps
        from tacotron_amd.kv_cache import KvCache
        s['cache'] = KvCache(s['k_pages'], s['v_pages'])
    cache = s['cache']
    if c['op'] == 'attend':
        if not c['mass']:
            return cache.attend(s['q'], s['table'], s['lengths'], scale=s['scale'])
        out, lse = cache.attend(s['q'], s['table'], s['lengths'], scale=s['scale'], mass=s['mass'])
        return out, lse, s['mass']
    if c['op'] == 'append':
        lengths = cache.append(s['k'], s['v'], s['table'], s['starts'], counts=s['counts'], first=s['first'],
                               mass=s['mass'], positions=s['positions'])
        return s['k_pages'], s['v_pages'], lengths, s['mass'], s['positions']
    lengths, mass, positions = cache.evict(s['table'], s['lengths'], s['mass'], s['positions'], c['budget'], c['recent'])
    return s['k_pages'], s['v_pages'], lengths, mass, positions


# ---------------------------------------------------------------------------------------
# the definition in 64 bits, sequence by sequence
def _exact_attend(s):
    c = s['case']
    B, hq, hkv, d, page = c['B'], c['hq'], c['hkv'], c['d'], c['page']
    dev = s['q'].device
    out = torch.zeros(B, hq, d, dtype=torch.float64, device=dev)
    lse = torch.full((B, hq), float('-inf'), dtype=torch.float64, device=dev)
    mass = s['mass'].double()
    for b, L in enumerate(s['lengths'].tolist()):
        if not L:
            continue
        ids = s['table'][b, :-(-L // page)].long()
        for h in range(hkv):
            heads = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
            k = s['k_pages'][ids, h].reshape(-1, d)[:L].double()
            v = s['v_pages'][ids, h].reshape(-1, d)[:L].double()
            score = (s['q'][b, heads].double() @ k.t()) * s['scale']
            lse[b, heads] = torch.logsumexp(score, 1)
            weight = torch.exp(score - lse[b, heads, None])
            out[b, heads] = weight @ v
            mass[b, h, :L] += weight.sum(0)
    return (out, lse, mass) if c['mass'] else (out, lse)


def _exact_append(s):
    c = s['case']
    page = c['page']
    k, v, mass, pos = s['k_pages'].double(), s['v_pages'].double(), s['mass'].double(), s['positions'].long()
    ends = []
    table = s['table'].cpu().numpy()
    for b, (start, count, first) in enumerate(zip(s['starts'].tolist(), s['counts'].tolist(), s['first'].tolist())):
        ends.append(start + count)
        mass[b, :, start:start + count] = 0
        pos[b, :, start:start + count] = torch.arange(first, first + count, device=pos.device)
        at = start
        while at < start + count:    # page by page
            stop = min((at // page + 1) * page, start + count)
            for pool, new in ((k, s['k']), (v, s['v'])):
                pool[int(table[b, at // page]), :, at % page:at % page + stop - at] = new[b, at - start:stop - start].double().transpose(0, 1)
            at = stop
    return k, v, torch.tensor(ends, dtype=torch.int32), mass, pos.to(torch.int32)


def _exact_evict(s):
    c = s['case']
    page, cap = c['page'], s['mass'].shape[2]
    k, v = s['k_pages'].double(), s['v_pages'].double()
    mass, pos, table = s['mass'].double().cpu().numpy(), s['positions'].cpu().numpy(), s['table'].cpu().numpy()
    new_mass, new_pos, lengths = np.zeros_like(mass), np.full_like(pos, -1), []
    for b, L in enumerate(s['lengths'].tolist()):
        n = min(L, c['budget'])
        lengths.append(n)
        for h in range(c['hkv']):
            m, p = mass[b, h, :L], pos[b, h, :L]
            new = p > p.max() - c['recent'] if L else np.zeros(0, bool)
            keep = np.sort(np.lexsort((np.arange(L), -m, ~new))[:n])
            low, late = keep[keep < n], keep[keep >= n]
            gaps = np.setdiff1d(np.arange(n), low)
            src = np.arange(n)
            src[gaps] = late
            new_mass[b, h, :n], new_pos[b, h, :n] = m[src], p[src]
            if len(gaps):
                to, fro = (torch.from_numpy(x).to(k.device) for x in (gaps, late))
                ids = torch.from_numpy(table[b].astype(np.int64)).to(k.device)
                for pool in (k, v):
                    pool[ids[to // page], h, to % page] = pool[ids[fro // page], h, fro % page]
    return k, v, torch.tensor(lengths, dtype=torch.int32), torch.from_numpy(new_mass), torch.from_numpy(new_pos)


def exact(case, seed):
    s = prepare(case, seed)
    return {'attend': _exact_attend, 'append': _exact_append, 'evict': _exact_evict}[case['op']](s)
