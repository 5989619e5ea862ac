"""The paged key-value cache on the GPU (tacotron_amd.kv_cache) against the 64-bit reference of tests/kv_reference.py, which
also derives the tolerances; moves, ties, lengths and untouched memory are compared bit for bit."""
import math

import numpy as np
import pytest

from tests import kv_reference as R

pytestmark = pytest.mark.gpu

TYPES = ['float32', 'bfloat16', 'float16']


def _make(seed, lens, hkv, d, page, dtype, spare=3, slots=None, layout='heads'):
    """A cache whose pages stand in no order, NaN in every slot and page that no sequence owns, and in the table -1 behind
    a sequence's pages. Returns (cache, table, lengths)."""
    import torch
    from tacotron_amd.kv_cache import KvCache
    g = torch.Generator().manual_seed(seed)
    dtype = getattr(torch, dtype)
    mp = max(1, -(-(slots or max(lens)) // page))
    used = [-(-n // page) for n in lens]
    P = sum(used) + spare
    order = torch.randperm(P, generator=g).tolist()
    table = torch.full((len(lens), mp), -1, dtype=torch.int32)
    k = torch.full((P, hkv, page, d), float('nan'))
    v = k.clone()
    for b, n in enumerate(lens):
        for j in range(used[b]):
            i = order.pop()
            table[b, j] = i
            m = min(page, n - j * page)
            k[i, :, :m] = torch.randn(hkv, m, d, generator=g)
            v[i, :, :m] = torch.randn(hkv, m, d, generator=g)
    k, v = k.to(dtype).cuda(), v.to(dtype).cuda()
    if layout == 'tokens':           # [P, page, hkv, d] in memory
        k, v = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v))
    return KvCache(k, v), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()


def _q(seed, B, hq, d, dtype, size=1.0):
    import torch
    return (size * torch.randn(B, hq, d, generator=torch.Generator().manual_seed(seed))).to(getattr(torch, dtype)).cuda()


def _close(got, want, tol, what):
    got = got.double().cpu().numpy() if hasattr(got, 'cpu') else got
    with np.errstate(invalid='ignore'):              # (-inf where both have it)
        same = (got == want) | (np.abs(got - want) <= tol)
    assert same.all(), '%s: off by %g where %g is allowed' % (what, np.abs(got - want)[~same].max(), np.asarray(tol)[~same].min())


def _check_attend(cache, table, lengths, q, scale=None, with_mass=True, mass0=0.0):
    import torch
    B, slots = table.shape[0], table.shape[1] * cache.page_size
    mass = torch.full((B, cache.kv_heads, slots + 5), mass0, device='cuda') if with_mass else None
    out, lse = cache.attend(q, table, lengths, scale=scale, mass=mass)
    lens = lengths.tolist()
    want, tol, wl, tl, weights, wt = R.attend(q, cache.k_pages, cache.v_pages, table, lens,
                                              1 / math.sqrt(cache.head_dim) if scale is None else scale)
    _close(out, want, tol, 'out')
    _close(lse, wl, tl, 'lse')
    if with_mass:
        m = mass.double().cpu().numpy()
        for b, L in enumerate(lens):
            _close(m[b, :, :L], mass0 + weights[b], wt[b] + 4 * R.U * (mass0 + weights[b]), 'mass')
            assert (m[b, :, L:] == mass0).all()
    cache.status()
    return out, lse, mass


# ---------------------------------------------------------------------------------------
# attend
RAGGED = [0, 1, 7, 8, 9, 31, 32, 33, 63, 64, 65, 127, 128, 129, 130, 300, 0, 515]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('d', [64, 128, 256])
@pytest.mark.parametrize('hkv,group', [(1, 1), (2, 3), (3, 8), (1, 16), (2, 17), (1, 32), (1, 33), (1, 40)])
def test_attend_ragged(dtype, d, hkv, group):
    page = {1: 8, 2: 16, 3: 64}[hkv]
    cache, table, lengths = _make(d + group, RAGGED, hkv, d, page, dtype)
    _check_attend(cache, table, lengths, _q(group, len(RAGGED), hkv * group, d, dtype))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('d', [64, 128, 256])
@pytest.mark.parametrize('hkv,group', [(1, 1), (5, 1), (2, 2), (3, 7), (1, 16), (1, 17)])
@pytest.mark.parametrize('slots', [64, 160, 256, 512])
def test_attend_short_memories(dtype, d, hkv, group, slots):
    """Tables of few slots, whose rows one workgroup can hold: every length about the sizes it deals out."""
    lens = sorted({n for k in (0, 8, 16, 32, 64, 96, 100, 128, 150, 256, 500, 512) for n in (k - 1, k, k + 1) if 0 <= n <= slots})
    cache, table, lengths = _make(d + slots, lens, hkv, d, 32 if slots % 32 == 0 and d > 64 else 8, dtype, slots=slots)
    _check_attend(cache, table, lengths, _q(group, len(lens), hkv * group, d, dtype, size=2.0), with_mass=slots != 160, mass0=1.5 if slots == 64 else 0.0)


@pytest.mark.parametrize('d,batch', [(64, 250), (64, 270), (128, 60), (128, 70)])
def test_attend_many_short_memories(d, batch):
    lens = [(7 * b) % 41 for b in range(batch)]
    cache, table, lengths = _make(d + batch, lens, 8, d, 8, 'bfloat16')
    _check_attend(cache, table, lengths, _q(batch, batch, 16, d, 'bfloat16'))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('page', [8, 16, 32, 64, 128, 256])
def test_attend_page_sizes(dtype, page):
    lens = [page, page - 1, page + 1, 3 * page + 5, 1, 2 * page]
    cache, table, lengths = _make(page, lens, 2, 128, page, dtype)
    _check_attend(cache, table, lengths, _q(page, len(lens), 8, 128, dtype), with_mass=page != 32, mass0=2.5)


@pytest.mark.parametrize('dtype,lens,hkv,group,d', [('bfloat16', [20011], 2, 4, 128), ('float16', [9973, 3, 12345], 1, 8, 64),
                                                     ('float32', [7001, 0, 256], 1, 2, 256), ('bfloat16', [70001], 1, 1, 64)])
def test_attend_split_over_a_long_axis(dtype, lens, hkv, group, d):
    cache, table, lengths = _make(5, lens, hkv, d, 16, dtype)
    _check_attend(cache, table, lengths, _q(6, len(lens), hkv * group, d, dtype, size=2.0))


def test_attend_many_short_rows():
    """More sequences than a wave has lanes, and more than there are workgroups."""
    rng = np.random.default_rng(3)
    lens = rng.integers(0, 40, 1500).tolist()
    cache, table, lengths = _make(7, lens, 1, 64, 8, 'bfloat16')
    _check_attend(cache, table, lengths, _q(8, len(lens), 2, 64, 'bfloat16'))


def test_attend_one_long_row_among_empty_ones():
    for at in (0, 70, 129):
        lens = [0] * 130
        lens[at] = 6007
        cache, table, lengths = _make(at, lens, 2, 64, 32, 'float16')
        _check_attend(cache, table, lengths, _q(9, 130, 4, 64, 'float16'))


@pytest.mark.parametrize('dtype', TYPES)
def test_attend_sharp_and_flat(dtype):
    """One token that takes everything, wherever it stands; and no preference at all."""
    import torch
    lens = [700, 700, 700]
    cache, table, lengths = _make(11, lens, 1, 64, 16, dtype)
    q = _q(12, 3, 4, 64, dtype)
    for b, at in ((0, 0), (1, 699)):
        page = int(table[b, at // 16])
        cache.k_pages[page, 0, at % 16] = 40 * q[b, 1]
    q[2] = 0
    _check_attend(cache, table, lengths, q)
    _check_attend(cache, table, lengths, q, scale=-0.3)
    _check_attend(cache, table, lengths, q, scale=0.0)


@pytest.mark.parametrize('dtype', TYPES)
def test_attend_many_small_weights_next_to_a_large_one(dtype):
    """30000 weights of e^-12 beside one of 1: together they are 0.18 of it, alone each is below fp16's smallest step."""
    lens = [30001]
    cache, table, lengths = _make(13, lens, 1, 64, 64, dtype)
    q = _q(14, 1, 1, 64, dtype)
    q[:] = 0
    q[..., 0] = 1.0
    cache.k_pages[..., 0] = 0
    cache.k_pages[int(table[0, 0]), 0, 3, 0] = 12.0
    cache.v_pages[..., 1] = 1.0
    cache.v_pages[int(table[0, 0]), 0, 3, 1] = -1.0
    _check_attend(cache, table, lengths, q, scale=1.0)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('group,slots', [(3, 150), (1, 150), (3, 3000), (1, 3000)])
def test_attend_infinite_scores(dtype, group, slots):
    """Tokens whose score is -inf weigh nothing; a row of them is a row without tokens."""
    import torch
    lens = [150, 150, 40]
    cache, table, lengths = _make(15, lens, 1, 64, 16, dtype, slots=slots)
    q = _q(16, 3, group, 64, dtype)
    q[..., 0] = 1.0
    for b in (0, 2):
        for t in range(lens[b]):
            if b == 2 or t % 3:
                cache.k_pages[int(table[b, t // 16]), 0, t % 16, 0] = -math.inf
    mass = torch.zeros(3, 1, table.shape[1] * 16, device='cuda')
    out, lse = cache.attend(q, table, lengths, mass=mass)
    assert (out[2] == 0).all() and (lse[2] == -math.inf).all() and (mass[2] == 0).all()
    keep = list(range(0, 150, 3))
    k, v = (torch.from_numpy(R.rows_of(x, table, 0, 0, 150)[keep]) for x in (cache.k_pages, cache.v_pages))
    s = q[0].double().cpu() @ k.t() / 8
    p = torch.softmax(s, 1)
    assert (out[0].double().cpu() - p @ v).abs().max() < 2 ** -7 and (lse[0].double().cpu() - torch.logsumexp(s, 1)).abs().max() < 1e-4
    got = mass[0, 0].double().cpu()
    assert (got[keep] - p.sum(0)).abs().max() < 1e-4 and got.sum() - got[keep].sum() == 0
    assert torch.isfinite(out).all()
    cache.status()


@pytest.mark.parametrize('group,slots', [(2, 200), (1, 200), (2, 3000)])
def test_attend_nan_stays_in_its_row(group, slots):
    import torch
    lens = [200, 200]
    cache, table, lengths = _make(17, lens, 2, 64, 16, 'bfloat16', slots=slots)
    q = _q(18, 2, 2 * group, 64, 'bfloat16')
    clean, _ = cache.attend(q, table, lengths)
    cache.v_pages[int(table[1, 4]), 1, 3, 5] = math.nan
    out, lse = cache.attend(q, table, lengths)
    hit = torch.zeros_like(out, dtype=torch.bool)
    hit[1, group:, 5] = True
    assert torch.equal(torch.isnan(out), hit) and torch.equal(out[~hit], clean[~hit])
    cache.k_pages[int(table[0, 2]), 0, 1, 7] = math.nan
    out, lse = cache.attend(q, table, lengths)
    assert torch.isnan(out[0, :group]).all() and torch.isnan(lse[0, :group]).all() and not torch.isnan(out[0, group:]).any()


@pytest.mark.parametrize('group,slots', [(2, 100), (1, 100), (2, 3000)])
def test_attend_bad_pages_and_lengths_are_masked(group, slots):
    import torch
    from tacotron_amd.engine import TacoError
    lens = [100, 40, 64, 33]
    cache, table, lengths = _make(19, lens, 2, 64, 16, 'float32', slots=slots)
    q = _q(20, 4, 2 * group, 64, 'float32')
    good, good_lse = cache.attend(q, table, lengths)
    bad = table.clone()
    bad[0, 2], bad[0, 5] = cache.num_pages, -7
    mass = torch.zeros(4, 2, table.shape[1] * 16, device='cuda')
    out, lse = cache.attend(q, bad, lengths, mass=mass)
    with pytest.raises(TacoError, match='page id'):
        cache.status()
    cache.status()                                   # read once
    rows = [t for t in range(100) if t // 16 not in (2, 5)]
    for h in range(2):
        k, v = (torch.from_numpy(R.rows_of(x, table, 0, h, 100)[rows]) for x in (cache.k_pages, cache.v_pages))
        mine = slice(group * h, group * h + group)
        p = torch.softmax(q[0, mine].double().cpu() @ k.t() / 8, 1)
        assert (out[0, mine].double().cpu() - p @ v).abs().max() < 1e-5
        assert (mass[0, h, rows].double().cpu() - p.sum(0)).abs().max() < 1e-5
    assert (mass[0, :, 32:48] == 0).all() and torch.equal(out[1:], good[1:]) and torch.equal(lse[1:], good_lse[1:])
    # every page of a row bad: a row without tokens
    bad[0] = -1
    out, lse = cache.attend(q, bad, lengths)
    assert (out[0] == 0).all() and (lse[0] == -math.inf).all()
    with pytest.raises(TacoError, match='page id'):
        cache.status()
    # lengths outside the table: clamped
    n = lengths.clone()
    n[1], n[2] = -5, 64
    out, lse = cache.attend(q, table[:, :4], n)      # (row 0 asks for 100 slots of 64)
    with pytest.raises(TacoError, match='length'):
        cache.status()
    n[0], n[1] = 64, 0
    want, want_lse = cache.attend(q, table[:, :4], n)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    cache.status()


def test_attend_strides_and_alignment():
    """Queries out of a fused projection or at an odd address, tables that are part of a wider one, a token-major pool."""
    import torch
    lens = [77, 130, 5]
    for dtype in TYPES:
        cache, table, lengths = _make(21, lens, 2, 128, 16, dtype, layout='tokens')
        plain, table2, _ = _make(21, lens, 2, 128, 16, dtype)
        assert torch.equal(table, table2) and not cache.k_pages.is_contiguous()
        q = _q(22, 3, 6, 128, dtype)
        want = plain.attend(q, table, lengths)
        fused = torch.randn(3, 10, 128, device='cuda').to(q.dtype)
        fused[:, 2:8] = q
        odd = torch.empty(q.numel() + 1, dtype=q.dtype, device='cuda')[1:].view(q.shape).copy_(q)
        turned = q.transpose(0, 1).contiguous().transpose(0, 1)
        strided = torch.stack([q, q], -1)[..., 0]
        wide = torch.full((3, 40), -1, dtype=torch.int32, device='cuda')
        wide[:, 3:3 + table.shape[1]] = table
        part = wide[:, 3:3 + table.shape[1]]
        for qq in (q, fused[:, 2:8], odd, turned, strided):
            for tt in (table, part):
                for got, exp in zip(cache.attend(qq, tt, lengths), want):
                    assert torch.equal(got, exp)
        _check_attend(cache, part, lengths, q)


def test_attend_pages_shared_by_sequences():
    import torch
    cache, table, _ = _make(23, [90], 2, 64, 16, 'bfloat16')
    table = table.expand(5, -1)                       # (stride 0: copied)
    lengths = torch.tensor([90, 17, 0, 64, 90], dtype=torch.int32, device='cuda')
    _check_attend(cache, table, lengths, _q(24, 5, 4, 64, 'bfloat16'))


def test_attend_same_call_same_bits():
    import torch
    lens = [3000, 1, 0, 257, 1999]
    cache, table, lengths = _make(25, lens, 2, 128, 16, 'bfloat16')
    q = _q(26, 5, 8, 128, 'bfloat16')
    first = _check_attend(cache, table, lengths, q)
    for _ in range(3):
        mass = torch.zeros_like(first[2])
        out, lse = cache.attend(q, table, lengths, mass=mass)
        assert torch.equal(out, first[0]) and torch.equal(lse, first[1]) and torch.equal(mass, first[2])


def test_offsets_past_32_bits():
    """A pool of more than 2^32 bytes and 2^31 elements: pages at its far end, read, written and evicted."""
    import torch
    from tacotron_amd.kv_cache import KvCache
    page, d = 256, 128
    P = (1 << 31) // (page * d) + 64
    cache = KvCache.empty(P, page, 1, d, torch.bfloat16)
    ids = [P - 1, 0, P - 3, P // 2 + 5]
    table = torch.tensor([ids], dtype=torch.int32, device='cuda')
    rows = torch.randn(1, 1000, 1, d, device='cuda').bfloat16()
    vals = torch.randn(1, 1000, 1, d, device='cuda').bfloat16()
    side = (torch.zeros(1, 1, 1024, device='cuda'), torch.zeros(1, 1, 1024, dtype=torch.int32, device='cuda'))
    zero = torch.zeros(1, dtype=torch.int32, device='cuda')
    lengths = cache.append(rows, vals, table, zero, mass=side[0], positions=side[1])
    flat = torch.cat([cache.k_pages[i, 0] for i in ids])
    assert lengths.tolist() == [1000] and torch.equal(flat[:1000], rows[0, :, 0])
    _check_attend(cache, table, lengths, _q(27, 1, 4, d, 'bfloat16'))
    side[0][:] = torch.rand(1, 1, 1024, device='cuda')
    want = R.evict(flat.float().cpu().numpy()[None, None], torch.cat([cache.v_pages[i, 0] for i in ids]).float().cpu().numpy()[None, None],
                   side[0].cpu().numpy(), side[1].cpu().numpy(), [1000], 300, 20)
    n, m, p = cache.evict(table, lengths, side[0], side[1], 300, 20)
    assert n.tolist() == [300] and np.array_equal(p.cpu().numpy(), want[3])
    assert np.array_equal(torch.cat([cache.k_pages[i, 0] for i in ids])[:300].float().cpu().numpy(), want[0][0, 0, :300])
    cache.status()


# ---------------------------------------------------------------------------------------
# append
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('d,hkv,page,T', [(64, 1, 8, 1), (128, 3, 16, 37), (256, 2, 32, 5), (64, 8, 256, 300)])
def test_append(dtype, d, hkv, page, T):
    import torch
    starts = [0, 1, page - 1, page, 5 * page + 3, 2]
    counts = [T, max(T - 1, 0), T, 0, T, min(T, 2)]
    cache, table, _ = _make(31, [s + T for s in starts], hkv, d, page, dtype)
    slots = table.shape[1] * page
    g = torch.Generator().manual_seed(5)
    fused = torch.randn(6, T, 2 * hkv + 3, d, generator=g).to(cache.dtype).cuda()
    k, v = fused[:, :, 3:3 + hkv], fused[:, :, 3 + hkv:]
    mass = torch.rand(6, hkv, slots + 3, generator=g).cuda()
    pos = torch.randint(0, 99, (6, hkv, slots + 3), generator=g, dtype=torch.int32).cuda()
    first = torch.tensor([1000 * i for i in range(6)], dtype=torch.int32, device='cuda')
    want_k, want_v, want_m, want_p = (x.clone() for x in (cache.k_pages, cache.v_pages, mass, pos))
    for b in range(6):
        for t in range(counts[b]):
            s = starts[b] + t
            want_k[table[b, s // page], :, s % page] = k[b, t]
            want_v[table[b, s // page], :, s % page] = v[b, t]
            want_m[b, :, s] = 0
            want_p[b, :, s] = 1000 * b + t
    dev = lambda x: torch.tensor(x, dtype=torch.int32, device='cuda')  # noqa: E731
    n = cache.append(k, v, table, dev(starts), counts=dev(counts), first=first, mass=mass, positions=pos)
    bits = lambda x: x.view(torch.int32 if x.element_size() == 4 else torch.int16)  # noqa: E731
    assert torch.equal(bits(cache.k_pages), bits(want_k)) and torch.equal(bits(cache.v_pages), bits(want_v))
    assert torch.equal(mass, want_m) and torch.equal(pos, want_p)
    assert n.tolist() == [s + c for s, c in zip(starts, counts)]
    # without counts, firsts and side tables: all T, rows in another order, at an odd address
    k2 = torch.empty(k.numel() + 1, dtype=k.dtype, device='cuda')[1:].view(k.shape).copy_(k)
    v2 = v.transpose(0, 2).contiguous().transpose(0, 2)
    n = cache.append(k2, v2, table, dev(starts))
    for b in range(6):
        for t in range(T):
            s = starts[b] + t
            want_k[table[b, s // page], :, s % page] = k[b, t]
            want_v[table[b, s // page], :, s % page] = v[b, t]
    assert torch.equal(bits(cache.k_pages), bits(want_k)) and torch.equal(bits(cache.v_pages), bits(want_v))
    assert n.tolist() == [s + T for s in starts]
    pos.fill_(-9)
    cache.append(k, v, table, dev(starts), positions=pos)      # positions alone: they start at the slots
    assert pos[4, 0, starts[4]:starts[4] + T].tolist() == list(range(starts[4], starts[4] + T)) and (pos == -9).sum() == pos.numel() - 6 * hkv * T
    cache.status()


def test_append_beyond_the_table_is_dropped():
    import torch
    from tacotron_amd.engine import TacoError
    cache, table, _ = _make(33, [64, 64, 64, 64], 1, 64, 16, 'float32')
    table[3, 1] = cache.num_pages
    before = cache.k_pages.clone()
    rows = torch.ones(4, 20, 1, 64, device='cuda')
    mass = torch.full((4, 1, 64), 7.0, device='cuda')
    n = cache.append(rows, rows, table, torch.tensor([60, 70, -3, 10], dtype=torch.int32, device='cuda'),
                     counts=torch.tensor([20, 20, 2, 21], dtype=torch.int32, device='cuda'), mass=mass)
    # row 0: four fit; row 1 starts beyond; row 2 starts at 0; row 3: a count over T is T, and page 1 is bad
    assert n.tolist() == [64, 64, 2, 30]
    with pytest.raises(TacoError, match='page id.*length'):
        cache.status()
    after = cache.k_pages
    want = before.clone()
    want[table[0, 3], :, 12:] = 1
    want[table[2, 0], :, :2] = 1
    want[table[3, 0], :, 10:] = 1
    assert torch.equal(torch.nan_to_num(after, 5.0), torch.nan_to_num(want, 5.0))
    assert (mass[0, 0, 60:] == 0).all() and (mass[1] == 7).all() and (mass[0, 0, :60] == 7).all()


# ---------------------------------------------------------------------------------------
# evict
def _flat(cache, pages, table, b, h, n):
    import torch
    page = cache.page_size
    ids = table[b, :-(-n // page)].long()
    return pages[ids, h].reshape(-1, cache.head_dim)[:n]


def _check_evict(cache, table, lengths, mass, pos, budget, recent, inplace):
    import torch
    lens = lengths.tolist()
    slots = table.shape[1] * cache.page_size
    B, hkv, d = len(lens), cache.kv_heads, cache.head_dim
    rows = {x: np.zeros((B, hkv, slots, d), np.float32) for x in 'kv'}
    for b, n in enumerate(lens):
        for h in range(hkv):
            for x, pages in (('k', cache.k_pages), ('v', cache.v_pages)):
                rows[x][b, h, :n] = _flat(cache, pages, table, b, h, n).float().cpu().numpy()
    wk, wv, wm, wp, wn = R.evict(rows['k'], rows['v'], mass.cpu().numpy(), pos.cpu().numpy(), lens, budget, recent)
    before = cache.k_pages.clone()
    out = (lengths, mass, pos) if inplace else None
    keep_in = (lengths.clone(), mass.clone(), pos.clone())
    n, m, p = cache.evict(table, lengths, mass, pos, budget, recent, out=out)
    assert np.array_equal(n.cpu().numpy(), wn)
    assert np.array_equal(m.cpu().numpy(), wm, equal_nan=True) and np.array_equal(p.cpu().numpy(), wp)
    if inplace:
        assert n is lengths and m is mass and p is pos
    else:
        for a, b in zip((lengths, mass, pos), keep_in):
            assert np.array_equal(a.cpu().numpy(), b.cpu().numpy(), equal_nan=True)
    moved = torch.zeros(cache.num_pages, dtype=torch.bool)
    for b in range(B):
        for h in range(hkv):
            assert np.array_equal(_flat(cache, cache.k_pages, table, b, h, int(wn[b])).float().cpu().numpy(), wk[b, h, :wn[b]])
            assert np.array_equal(_flat(cache, cache.v_pages, table, b, h, int(wn[b])).float().cpu().numpy(), wv[b, h, :wn[b]])
        moved[table[b, :-(-int(wn[b]) // cache.page_size)].long().cpu()] = True
    other = ~moved.cuda()
    assert torch.equal(torch.nan_to_num(before[other].float(), 5.0), torch.nan_to_num(cache.k_pages[other].float(), 5.0))
    cache.status()


@pytest.mark.parametrize('inplace', [False, True])
@pytest.mark.parametrize('dtype,d,hkv,page,budget,recent', [
    ('float32', 64, 1, 8, 1, 0), ('float32', 256, 2, 16, 64, 64), ('bfloat16', 128, 3, 16, 100, 7),
    ('float16', 64, 2, 32, 513, 0), ('bfloat16', 256, 1, 128, 1000, 999), ('float32', 128, 2, 8, 5000, 10)])
@pytest.mark.parametrize('masses', ['random', 'ties', 'odd'])
def test_evict(inplace, dtype, d, hkv, page, budget, recent, masses):
    import torch
    lens = [0, 1, budget - 1, budget, budget + 1, 2 * budget + 3, 1500, 2049, 700]
    cache, table, lengths = _make(41, lens, hkv, d, page, dtype)
    slots = table.shape[1] * page + 2
    g = torch.Generator().manual_seed(budget)
    mass = torch.rand(len(lens), hkv, slots, generator=g) ** 4
    if masses == 'ties':
        mass = torch.floor(mass * 4)
    if masses == 'odd':
        pick = torch.rand(mass.shape, generator=g)
        mass[pick < 0.1] = 0.0
        mass[(pick > 0.1) & (pick < 0.15)] = -0.0
        mass[(pick > 0.2) & (pick < 0.22)] = float('nan')
        mass[(pick > 0.3) & (pick < 0.35)] = float('inf')
        mass[(pick > 0.4) & (pick < 0.5)] *= -1
        mass[(pick > 0.5) & (pick < 0.6)] *= 1e-42
    # NaN is the greatest, an infinity the next: the reference orders them by hand
    pos = torch.stack([torch.stack([torch.randperm(slots, generator=g) * 3 for _ in range(hkv)]) for _ in lens]).to(torch.int32)
    _check_evict(cache, table, lengths, mass.cuda(), pos.cuda(), budget, recent, inplace)


@pytest.mark.parametrize('inplace', [False, True])
@pytest.mark.parametrize('masses', ['random', 'ties', 'odd', 'equal', 'last'])
@pytest.mark.parametrize('dtype,d,hkv,page,budget,recent', [
    ('float32', 64, 1, 8, 1, 0), ('float32', 64, 1, 8, 1, 1), ('float32', 256, 2, 16, 63, 5), ('bfloat16', 128, 3, 16, 64, 64),
    ('float16', 64, 2, 8, 1023, 0), ('bfloat16', 256, 1, 32, 1024, 100), ('bfloat16', 64, 2, 16, 4095, 4095),
    ('float32', 64, 1, 16, 4096, 1), ('float16', 128, 1, 256, 16383, 300)])
def test_evict_one_over(inplace, masses, dtype, d, hkv, page, budget, recent):
    """Rows one token over the budget beside others; a table that ends with the token, and one that does not."""
    import torch
    for lens in ([budget + 1], [budget + 1, budget, 0, budget + 1], [budget + 1, min(2 * budget + 3, 16384), budget + 1]):
        cache, table, lengths = _make(budget, lens, hkv, d, page, dtype)
        slots = table.shape[1] * page
        g = torch.Generator().manual_seed(budget + len(lens))
        mass = torch.rand(len(lens), hkv, slots, generator=g) ** 3
        pos = torch.stack([torch.stack([torch.randperm(slots, generator=g) for _ in range(hkv)]) for _ in lens]).to(torch.int32)
        if masses == 'ties':
            mass = torch.floor(mass * 3)
        if masses == 'equal':
            mass[:] = 0.25
        if masses == 'last':                 # the token that goes is the one in the last slot
            mass[:, :, budget] = 0.0
            pos[:, :, budget] = -1
        if masses == 'odd':
            pick = torch.rand(mass.shape, generator=g)
            mass[pick < 0.3] = float('nan')
            mass[(pick > 0.3) & (pick < 0.6)] = float('inf')
            mass[(pick > 0.6) & (pick < 0.65)] = -float('inf')
            mass[pick > 0.9] = -0.0
            pos //= 2
        _check_evict(cache, table, lengths, mass.cuda(), pos.cuda(), budget, recent, inplace)


@pytest.mark.parametrize('gone', [70, 150, 200])
def test_evict_one_over_bad_page(gone):
    """A bad page under the row that moves, or under the gap: nothing is written there, side tables stay consistent."""
    import torch
    from tacotron_amd.engine import TacoError
    for hurt in (70, 200):
        cache, table, lengths = _make(51, [201], 2, 64, 16, 'bfloat16')
        mass = torch.ones(1, 2, 208, device='cuda')
        mass[0, :, gone] = 0.0
        pos = torch.arange(208, dtype=torch.int32, device='cuda').expand(1, 2, 208).contiguous()
        bad = table.clone()
        bad[0, hurt // 16] = cache.num_pages
        before, rows = cache.k_pages.clone(), _flat(cache, cache.v_pages, table, 0, 1, 201).clone()
        n, m, p = cache.evict(bad, lengths, mass, pos, 200, 0)
        if gone != 200 and hurt in (gone, 200):
            with pytest.raises(TacoError, match='page id'):
                cache.status()
            assert torch.equal(torch.nan_to_num(before.float(), 5.0), torch.nan_to_num(cache.k_pages.float(), 5.0))
        else:
            cache.status()
            if gone != 200:
                rows[gone] = rows[200]
            assert torch.equal(_flat(cache, cache.v_pages, table, 0, 1, 200), rows[:200])
        want = list(range(200))
        if gone != 200:
            want[gone] = 200
        assert n.tolist() == [200] and p[0, 1, :200].tolist() == want
        assert (p[..., 200:] == -1).all() and (m[..., 200:] == 0).all() and (m[..., :200] == 1).all()


@pytest.mark.parametrize('inplace', [False, True])
def test_evict_long(inplace):
    import torch
    lens = [70003, 8193]
    cache, table, lengths = _make(43, lens, 2, 64, 64, 'bfloat16')
    slots = table.shape[1] * 64
    g = torch.Generator().manual_seed(1)
    mass = -torch.log(torch.rand(2, 2, slots, generator=g).clamp(1e-6)).cuda()
    mass[1] = 0.0
    pos = torch.arange(slots, dtype=torch.int32, device='cuda').expand(2, 2, slots).contiguous()
    _check_evict(cache, table, lengths, mass, pos, 8192, 100, inplace)


@pytest.mark.parametrize('inplace', [False, True])
def test_evict_shared_by_workgroups(inplace):
    """Tables past what one workgroup holds: rows under the budget and empty ones among long ones, every kind of mass, a
    budget in the middle of a stretch, more stretches than a wave has lanes."""
    import torch
    lens = [70003, 100, 0, 40000, 39999, 8192, 16385]
    cache, table, lengths = _make(47, lens, 2, 64, 128, 'float16')
    slots = table.shape[1] * 128 + 3
    g = torch.Generator().manual_seed(2)
    mass = torch.rand(len(lens), 2, slots, generator=g) ** 3
    pick = torch.rand(mass.shape, generator=g)
    mass[pick < 0.05] = 0.0
    mass[(pick > 0.1) & (pick < 0.15)] = float('nan')
    mass[(pick > 0.2) & (pick < 0.25)] = float('inf')
    mass[(pick > 0.3) & (pick < 0.5)] = 0.125
    mass[(pick > 0.6) & (pick < 0.7)] *= -1
    pos = torch.stack([torch.stack([torch.randperm(slots, generator=g) for _ in range(2)]) for _ in lens]).to(torch.int32)
    _check_evict(cache, table, lengths, mass.cuda(), pos.cuda(), 39999, 5000, inplace)


def test_evict_more_stretches_than_lanes():
    import torch
    lens = [600001]
    cache, table, lengths = _make(49, lens, 1, 64, 256, 'bfloat16')
    slots = table.shape[1] * 256
    g = torch.Generator().manual_seed(3)
    pos = torch.arange(slots, dtype=torch.int32).view(1, 1, slots).cuda()
    _check_evict(cache, table, lengths, torch.rand(1, 1, slots, generator=g).cuda(), pos, 100000, 64, False)
    cache, table, lengths = _make(49, lens, 1, 64, 256, 'bfloat16')
    mass = torch.floor(torch.rand(1, 1, slots, generator=g) * 3).cuda()
    _check_evict(cache, table, lengths, mass, pos, 300000, 0, False)


def test_evict_bad_pages_move_nothing_there():
    import torch
    from tacotron_amd.engine import TacoError
    cache, table, lengths = _make(45, [200], 1, 64, 16, 'float32')
    mass = torch.zeros(1, 1, 208, device='cuda')
    mass[0, 0, 100:150] = 1.0
    pos = torch.arange(208, dtype=torch.int32, device='cuda').view(1, 1, 208)
    bad = table.clone()
    bad[0, 8] = -1                    # slots 128..143
    before = cache.k_pages.clone()
    n, m, p = cache.evict(bad, lengths, mass, pos, 50, 0)
    with pytest.raises(TacoError, match='page id'):
        cache.status()
    assert n.tolist() == [50] and p[0, 0, :50].tolist() == list(range(100, 150))
    for i in range(50):
        page, row = int(table[0, i // 16]), i % 16
        src = 100 + i
        want = before[page, 0, row] if src // 16 == 8 else before[int(table[0, src // 16]), 0, src % 16]
        assert torch.equal(cache.k_pages[page, 0, row], want)
    over = torch.tensor([999], dtype=torch.int32, device='cuda')
    cache.evict(table, over, mass, pos, 50, 0)
    with pytest.raises(TacoError, match='length'):
        cache.status()


# ---------------------------------------------------------------------------------------
# refusals of the Python face that need tensors on the GPU
def test_refusals():
    import torch
    from tacotron_amd.engine import TacoError
    cache, table, lengths = _make(51, [40, 20], 2, 64, 16, 'float32')
    q = _q(1, 2, 4, 64, 'float32')
    rows = torch.zeros(2, 3, 2, 64, device='cuda')
    slots = table.shape[1] * 16
    mass, pos = torch.zeros(2, 2, slots, device='cuda'), torch.zeros(2, 2, slots, dtype=torch.int32, device='cuda')
    for call, text in [
            (lambda: cache.attend(q[:, :3], table, lengths), 'q_heads'), (lambda: cache.attend(q[:, :, :32], table, lengths), 'q must'),
            (lambda: cache.attend(q.half(), table, lengths), 'float32'), (lambda: cache.attend(q.cpu(), table, lengths), 'cuda'),
            (lambda: cache.attend(q[:0], table, lengths), 'q must'), (lambda: cache.attend(q, table.long(), lengths), 'page_table'),
            (lambda: cache.attend(q, table[:1], lengths), 'page_table'), (lambda: cache.attend(q, table, lengths.long()), 'lengths'),
            (lambda: cache.attend(q, table, lengths[:1]), 'lengths'), (lambda: cache.attend(q, table, lengths, mass=mass[:, :, :-1]), 'mass'),
            (lambda: cache.attend(q, table, lengths, mass=mass.double()), 'mass'), (lambda: cache.attend(q, table, lengths, scale=math.nan), 'scale'),
            (lambda: cache.append(rows, rows[:, :2], table, lengths), 'same shape'), (lambda: cache.append(rows[:, :, :1], rows[:, :, :1], table, lengths), 'must be'),
            (lambda: cache.append(rows.half(), rows.half(), table, lengths), 'float32'), (lambda: cache.append(rows, rows, table, lengths, counts=lengths[:1]), 'counts'),
            (lambda: cache.append(rows, rows, table, lengths, mass=mass, positions=torch.zeros(2, 2, slots + 1, dtype=torch.int32, device='cuda')), 'same shape'),
            (lambda: cache.append(rows[:, :0], rows[:, :0], table, lengths), 'must be'),
            (lambda: cache.evict(table, lengths, mass, pos, 0), 'budget'), (lambda: cache.evict(table, lengths, mass, pos, 4, 5), 'recent'),
            (lambda: cache.evict(table, lengths, mass, pos.float(), 4), 'positions'), (lambda: cache.evict(table, lengths, mass, pos, 4, out=(lengths, mass)), 'out'),
            (lambda: cache.evict(table, lengths, mass, pos, 4, out=(lengths, mass, pos.transpose(0, 1))), 'out')]:
        with pytest.raises(TacoError, match=text):
            call()
    cache.status()


# ---------------------------------------------------------------------------------------
# together, as they are used
def test_a_decode_with_a_budget():
    """A prompt, then tokens one by one: append, attend (weights collected), evict. Every step's attention against the
    64-bit one over the rows the cache should hold; the eviction's choice from the masses the cache collected."""
    import torch
    B, hkv, group, d, page, budget, recent = 3, 2, 4, 128, 16, 40, 8
    prompt = [37, 5, 61]
    for dtype in ('bfloat16', 'float32'):
        from tacotron_amd.kv_cache import KvCache
        mp = 5
        cache = KvCache.empty(B * mp, page, hkv, d, getattr(torch, dtype))
        g = torch.Generator().manual_seed(3)
        table = torch.randperm(B * mp, generator=g).view(B, mp).to(torch.int32).cuda()
        mass, pos = torch.zeros(B, hkv, mp * page, device='cuda'), torch.full((B, hkv, mp * page), -1, dtype=torch.int32, device='cuda')
        new = lambda T: [torch.randn(B, T, hkv, d, generator=g).to(cache.dtype).cuda() for _ in range(2)]  # noqa: E731
        k, v = new(max(prompt))
        history = [[(k[b, t], v[b, t]) for t in range(prompt[b])] for b in range(B)]
        lengths = cache.append(k, v, table, torch.zeros(B, dtype=torch.int32, device='cuda'),
                               counts=torch.tensor(prompt, dtype=torch.int32, device='cuda'), mass=mass, positions=pos)
        seen = lengths.clone()
        for step in range(30):
            k, v = new(1)
            for b in range(B):
                history[b].append((k[b, 0], v[b, 0]))
            lengths = cache.append(k, v, table, lengths, first=seen, mass=mass, positions=pos)
            seen += 1
            _, _, got = _check_attend(cache, table, lengths, _q(100 + step, B, hkv * group, d, dtype))
            mass += got[:, :, :mp * page]
            old = (mass.cpu().numpy(), pos.cpu().numpy(), lengths.tolist())
            lengths, mass, pos = cache.evict(table, lengths, mass, pos, budget, recent)
            assert lengths.tolist() == [min(n, budget) for n in old[2]]
            for b, n in enumerate(lengths.tolist()):
                for h in range(hkv):
                    L = old[2][b]
                    keep = R.survivors(old[0][b, h, :L], old[1][b, h, :L], n, recent)
                    assert sorted(old[1][b, h, keep].tolist()) == sorted(pos[b, h, :n].tolist())
                    assert set(range(max(0, int(seen[b]) - recent), int(seen[b]))) <= set(pos[b, h, :n].tolist())
                    for pages, which in ((cache.k_pages, 0), (cache.v_pages, 1)):
                        want = torch.stack([history[b][t][which][h] for t in pos[b, h, :n].tolist()])
                        assert torch.equal(_flat(cache, pages, table, b, h, n), want)
        cache.status()


def test_captured_steps_follow_their_tensors():
    """A step (append, attend, evict in place) captured once and replayed: lengths, tables and masses are read when the
    graph runs. The same steps run eagerly on a twin give the same bits; eager work and synchronisations between."""
    import torch
    B, hkv, group, d, page, budget = 4, 2, 2, 64, 16, 33
    twins = []
    for _ in range(2):
        cache, table, lengths = _make(61, [40, 12, 0, 33], hkv, d, page, 'bfloat16', slots=64)
        own = torch.randperm(B * 4, generator=torch.Generator().manual_seed(1)).view(B, 4).to(torch.int32).cuda()
        from tacotron_amd.kv_cache import KvCache
        k, v = (torch.zeros(B * 4, hkv, page, d, dtype=torch.bfloat16, device='cuda') for _ in range(2))
        for b in range(B):
            for j in range(4):
                if table[b, j] >= 0:
                    k[own[b, j]], v[own[b, j]] = cache.k_pages[table[b, j]], cache.v_pages[table[b, j]]
        twins.append(dict(cache=KvCache(k, v), table=own, lengths=lengths, mass=torch.zeros(B, hkv, 64, device='cuda'),
                          pos=torch.arange(64, dtype=torch.int32, device='cuda').expand(B, hkv, 64).contiguous(),
                          seen=torch.full((B,), 100, dtype=torch.int32, device='cuda'),
                          q=_q(1, B, hkv * group, d, 'bfloat16'), rows=torch.zeros(2, B, 1, hkv, d, dtype=torch.bfloat16, device='cuda')))

    def step(s):
        n = s['cache'].append(s['rows'][0], s['rows'][1], s['table'], s['lengths'], first=s['seen'], mass=s['mass'], positions=s['pos'])
        s['seen'].add_(1)
        out, lse = s['cache'].attend(s['q'], s['table'], n, mass=s['mass'])
        _, _, _ = s['cache'].evict(s['table'], n, s['mass'], s['pos'], budget, 4, out=(s['lengths'], s['mass'], s['pos']))
        return out, lse

    graph = torch.cuda.CUDAGraph()
    stream = torch.cuda.Stream()
    keep = {n: twins[0][n].clone() for n in ('lengths', 'mass', 'pos', 'seen')}
    pages = [x.clone() for x in (twins[0]['cache'].k_pages, twins[0]['cache'].v_pages)]
    with torch.cuda.stream(stream):
        step(twins[0])
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out, lse = step(twins[0])
    for n, x in keep.items():
        twins[0][n].copy_(x)
    for a, b in zip((twins[0]['cache'].k_pages, twins[0]['cache'].v_pages), pages):
        a.copy_(b)
    for i in range(12):
        for s in twins:
            s['q'].copy_(_q(200 + i, B, hkv * group, d, 'bfloat16'))
            s['rows'].copy_(torch.randn(2, B, 1, hkv, d, generator=torch.Generator().manual_seed(i)).bfloat16())
            if i == 5:
                s['lengths'][2] = 0
        graph.replay()
        want = step(twins[1])
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1]), i
        for n in ('lengths', 'mass', 'pos', 'seen'):
            assert torch.equal(twins[0][n], twins[1][n]), (i, n)
        for a, b in zip(*((s['cache'].k_pages, s['cache'].v_pages) for s in twins)):
            same = torch.equal(a.view(torch.int16), b.view(torch.int16))      # (bits: unused slots hold NaN)
            assert same, i
    for s in twins:
        s['cache'].status()


def test_calls_on_several_streams():
    """Two streams, each with its own batch over one pool, at the same time: the bits of one after the other."""
    import torch
    lens = [900, 31, 2500]
    cache, table, lengths = _make(71, lens, 2, 128, 16, 'float16')
    qs = [_q(72 + i, 3, 8, 128, 'float16') for i in range(2)]
    want = []
    for q in qs:
        mass = torch.zeros(3, 2, table.shape[1] * 16, device='cuda')
        want.append((*cache.attend(q, table, lengths, mass=mass), mass))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                mass = torch.zeros(3, 2, table.shape[1] * 16, device='cuda')
                got[i].append((*cache.attend(qs[i], table, lengths, mass=mass), mass))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            for a, b in zip(r, want[i]):
                assert torch.equal(a, b)


def test_other_streams_and_captured_graphs_share_nothing():
    """Two captured attends of different sizes, replayed in turn and beside an eager one on another stream."""
    import torch
    cases = []
    for i, lens in enumerate(([700, 31, 2500], [64, 9000])):
        cache, table, lengths = _make(73 + i, lens, 2, 64, 16, 'bfloat16')
        q = _q(75 + i, len(lens), 6, 64, 'bfloat16')
        mass = torch.zeros(len(lens), 2, table.shape[1] * 16, device='cuda')
        want = (*cache.attend(q, table, lengths, mass=mass), mass)
        graph, out = torch.cuda.CUDAGraph(), torch.zeros_like(mass)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            out.zero_()
            got = (*cache.attend(q, table, lengths, mass=out), out)
        cases.append((cache, table, lengths, q, want, graph, got))
    side = torch.cuda.Stream()
    for turn in range(6):
        order = cases if turn % 2 else cases[::-1]
        for c in order:
            c[5].replay()
        with torch.cuda.stream(side):
            eager = cases[turn % 2]
            out, lse = eager[0].attend(eager[3], eager[1], eager[2])
        torch.cuda.synchronize()
        assert torch.equal(out, eager[4][0]) and torch.equal(lse, eager[4][1])
        for c in cases:
            for a, b in zip(c[6], c[4]):
                assert torch.equal(a, b), turn
        torch.zeros(1 << 20, device='cuda').add_(1)


def test_encoder_memory(engine, hp):
    """The memory of a batch of utterances (TacoEngine.encode), written once and attended as a decoder would."""
    import torch
    from tacotron_amd.kv_cache import KvCache
    from tests.util import synth_ids
    ids, lens = synth_ids(np.random.default_rng(2), 5, 70)
    enc = engine.encode(ids, lens)
    B, T, d = enc.shape
    page = 16
    mp = -(-T // page)
    cache = KvCache.empty(B * mp, page, 1, d)
    cache.k_pages.fill_(math.nan)
    cache.v_pages.fill_(math.nan)
    table = torch.arange(B * mp, dtype=torch.int32, device='cuda').view(B, mp)
    counts = torch.as_tensor(lens, dtype=torch.int32, device='cuda')
    rows = enc[:, :, None]
    n = cache.append(rows, rows, table, torch.zeros_like(counts), counts=counts)
    assert torch.equal(n, counts)
    _check_attend(cache, table, n, _q(3, B, 1, d, 'float32'))
