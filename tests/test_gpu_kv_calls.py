"""Calls of the key-value cache beside each other on the GPU: evictions on several streams and in captured graphs, and what the
cache object itself keeps."""
import pytest

from tests.test_gpu_kv_cache import TYPES, _make, _q

pytestmark = pytest.mark.gpu


def _same(a, b):
    import torch
    return torch.equal(a.view(torch.int32 if a.element_size() == 4 else torch.int16), b.view(torch.int32 if b.element_size() == 4 else torch.int16))


class Evictions:
    """One pool, `n` sequences of pages of their own, each cut down by a call of its own."""

    def __init__(self, n, slots, budget, hkv=1, page=8):
        import torch
        lens = [slots - i % 3 for i in range(n)]
        self.cache, self.table, self.lengths = _make(slots, lens, hkv, 64, page, 'bfloat16', slots=slots)
        g = torch.Generator().manual_seed(budget)
        shape = (n, hkv, self.table.shape[1] * page)
        self.mass = torch.rand(shape, generator=g).cuda()
        self.pos = torch.arange(shape[2], dtype=torch.int32).expand(shape).contiguous().cuda()
        self.pages = [x.clone() for x in (self.cache.k_pages, self.cache.v_pages)]
        self.n, self.budget = n, budget

    def restore(self):
        for x, y in zip((self.cache.k_pages, self.cache.v_pages), self.pages):
            x.copy_(y)

    def call(self, i):
        s = slice(i, i + 1)
        return self.cache.evict(self.table[s], self.lengths[s], self.mass[s], self.pos[s], self.budget, min(3, self.budget - 1))

    def outcome(self, results):
        return [x.clone() for r in results for x in r] + [self.cache.k_pages.clone(), self.cache.v_pages.clone()]


SIZES = [(64, 1), (200, 2), (2064, 700), (20000, 5000)]      # 16 bytes of workspace; moved in one launch; in two; by chunks


@pytest.mark.parametrize('slots,budget', SIZES)
def test_evictions_on_two_streams(slots, budget):
    import torch
    e = Evictions(12, slots, budget)
    want = e.outcome([e.call(i) for i in range(e.n)])
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(4):
        e.restore()
        torch.cuda.synchronize()
        results = [None] * e.n
        for i in range(e.n):
            with torch.cuda.stream(streams[i % 2]):
                results[i] = e.call(i)
        torch.cuda.synchronize()
        assert all(_same(a, b) for a, b in zip(e.outcome(results), want))
    e.cache.status()


@pytest.mark.parametrize('slots,budget', SIZES)
def test_captured_evictions_beside_eager_ones(slots, budget):
    """Two graphs of three evictions each, replayed on streams of their own while the rest run eagerly on a third."""
    import torch
    e = Evictions(9, slots, budget)
    want = e.outcome([e.call(i) for i in range(e.n)])
    graphs, results = [], [None] * e.n
    torch.cuda.synchronize()
    for g in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[g]):
            for i in range(3 * g, 3 * g + 3):
                results[i] = e.call(i)
    streams = [torch.cuda.Stream() for _ in range(3)]
    for turn in range(4):
        e.restore()
        torch.cuda.synchronize()
        for g in ((0, 1) if turn % 2 else (1, 0)):
            with torch.cuda.stream(streams[g]):
                graphs[g].replay()
        with torch.cuda.stream(streams[2]):
            for i in range(6, 9):
                results[i] = e.call(i)
        torch.cuda.synchronize()
        assert all(_same(a, b) for a, b in zip(e.outcome(results), want)), turn
        torch.zeros(1 << 20, device='cuda').add_(1)
    e.cache.status()


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('d,hkv,group,lens', [
    (64, 2, 3, [40, 0, 64, 1]), (128, 1, 16, [100, 7]), (256, 3, 17, [33, 150, 2]), (64, 1, 40, [9000, 0, 5]), (128, 2, 4, [20000])])
def test_attend_over_its_queries(dtype, d, hkv, group, lens):
    """The C entry with contiguous queries as the output too: the bits of a call with a buffer of its own."""
    import torch
    from tacotron_amd import _lib
    cache, table, lengths = _make(d + group, lens, hkv, d, 16, dtype)
    B, hq, mp, lib = len(lens), hkv * group, table.shape[1], _lib.load_library()
    q = _q(group, B, hq, d, dtype)
    want, want_lse = cache.attend(q, table, lengths)
    lse = torch.empty_like(want_lse)
    ws = torch.empty(lib.taco_kv_attend_workspace_bytes(cache._ref, B, hq, mp, 0), dtype=torch.uint8, device='cuda')
    assert lib.taco_kv_attend(cache._ref, table.data_ptr(), mp, B, mp, lengths.data_ptr(), q.data_ptr(), hq * d, d, hq, d ** -0.5, q.data_ptr(),
                              lse.data_ptr(), None, 0, ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream) == 0
    assert _same(q, want) and _same(lse, want_lse)


def _one_bad_page():
    """A call that meets a page id outside the pool, and a cache to make it with."""
    import torch
    cache, table, lengths = _make(5, [40], 1, 64, 16, 'float32')
    bad = table.clone()
    bad[0, 1] = cache.num_pages
    q = _q(1, 1, 2, 64, 'float32')
    torch.cuda.synchronize()
    return cache, bad, lengths, q


def test_status_keeps_what_is_met_while_it_is_read(monkeypatch):
    """A call of another stream between the reading of the word and its clearing."""
    import torch
    from tacotron_amd.engine import TacoError
    cache, bad, lengths, q = _one_bad_page()
    side, read = torch.cuda.Stream(), torch.Tensor.item

    def item(t):
        x = read(t)
        monkeypatch.undo()
        with torch.cuda.stream(side):
            cache.attend(q, bad, lengths)
        torch.cuda.synchronize()
        return x
    cache.attend(q, bad, lengths)
    monkeypatch.setattr(torch.Tensor, 'item', item)
    for _ in range(2):
        with pytest.raises(TacoError, match='page id'):
            cache.status()
    cache.status()


def test_status_of_a_cache_made_on_a_busy_stream():
    """What a call of another stream meets before the stream of the cache's making has come so far."""
    import torch
    from tacotron_amd.engine import TacoError
    from tacotron_amd.kv_cache import KvCache
    made, bad, lengths, q = _one_bad_page()
    with torch.cuda.stream(torch.cuda.Stream()):
        torch.cuda._sleep(50_000_000)
        cache = KvCache(made.k_pages, made.v_pages)
    cache.attend(q, bad, lengths)
    with pytest.raises(TacoError, match='page id'):
        cache.status()
    cache.status()


def test_a_cache_that_goes_while_a_call_runs():
    """Neither the status word nor the pool is given to another tensor before the calls of every stream are over."""
    import torch
    from tacotron_amd.kv_cache import KvCache
    table = torch.zeros(1, 3, dtype=torch.int32, device='cuda')
    lengths = torch.full((1,), 40, dtype=torch.int32, device='cuda')
    q = _q(1, 1, 2, 64, 'float32')
    side = torch.cuda.Stream()
    cache = KvCache.empty(1024, 16, 1, 64)
    held = {x.data_ptr() for x in (cache._status, cache.k_pages, cache.v_pages)}
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(400_000_000)
        out, lse = cache.attend(q, table, lengths)
    del cache
    others = [torch.empty(n, dtype=torch.int32, device='cuda') for n in [8] * 200 + [1 << 20] * 4]
    assert not side.query() and not held & {x.data_ptr() for x in others}
    torch.cuda.synchronize()


def test_a_call_for_no_device_leaves_no_error_behind():
    """What is refused for its device is not reported again by the next call, nor by the library's next launch."""
    import ctypes

    import torch
    from tacotron_amd import _lib
    cache, table, lengths = _make(6, [40], 1, 64, 16, 'float32')
    q = _q(1, 1, 2, 64, 'float32')
    want, _ = cache.attend(q, table, lengths)
    pool = type(cache._pool).from_buffer_copy(cache._pool)
    pool.device = torch.cuda.device_count()
    bits = torch.zeros(1, dtype=torch.int32, device='cuda')
    torch.cuda.synchronize()
    assert cache.lib.taco_kv_take_status(ctypes.byref(pool), bits.data_ptr(), None) < 0 and 'not available' in _lib.last_error()
    got, _ = cache.attend(q, table, lengths)
    assert torch.equal(got, want)
    assert cache.lib.taco_kv_take_status(ctypes.byref(pool), bits.data_ptr(), None) < 0
    assert (bits + 1).item() == 1


def test_gradients_are_refused_by_the_calls():
    import torch
    from tacotron_amd.engine import TacoError
    cache, table, lengths = _make(7, [40, 3], 1, 64, 16, 'float32')
    q, rows = _q(1, 2, 2, 64, 'float32').requires_grad_(), torch.zeros(2, 1, 1, 64, device='cuda')
    slots = table.shape[1] * 16
    mass, pos = torch.zeros(2, 1, slots, device='cuda', requires_grad=True), torch.zeros(2, 1, slots, dtype=torch.int32, device='cuda')
    for call in (lambda: cache.attend(q, table, lengths), lambda: cache.attend(q.detach(), table, lengths, mass=mass),
                 lambda: cache.append(rows + q[:, None, :1], rows, table, lengths), lambda: cache.append(rows, rows + q[:, None, :1], table, lengths),
                 lambda: cache.evict(table, lengths, mass, pos, 2), lambda: type(cache)(cache.k_pages.clone().requires_grad_(), cache.v_pages)):
        with pytest.raises(TacoError, match='gradient'):
            call()
        with torch.no_grad():
            call()
    cache.status()


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('d', [64, 128, 256])
@pytest.mark.parametrize('slots', [16, 3000])
def test_attend_weights_keep_their_bits(dtype, d, slots):
    """Three tokens of a sequence weigh w, 1 and 1, with values 1, -a and -b, where a + b is w to as many bits as two numbers of
    the type hold: what is left, (w - a - b) / (2 + w), is there only if the weight's other bits reach the product.

    Tolerance, in U = 2^-24 (half a step of fp32): the score is one product, exact, below 1 in units of ln 2; its factor and itself are
    rounded (2 U, 1.4 in w), the exponential is off by a step (2 U), a sum of three products of at most 1 by up to 4 U, and a
    weight in 16-bit pieces by half a step of the last: U / 2 (three of bf16), 4 U (two of fp16). Then the rounding to the type."""
    import numpy as np
    import torch
    rng, U = np.random.default_rng(d), 2.0 ** -24
    t = getattr(torch, dtype)
    as_t = lambda x: torch.tensor(np.asarray(x)).to(t).double().numpy()  # noqa: E731
    k, q = as_t(-rng.uniform(0.2, 0.9, 4000)), as_t(rng.uniform(0.2, 0.75, 4000))
    w = np.exp(k * q)
    a = as_t(w)
    b = as_t(w - a)
    left = w - a - b
    if dtype == 'bfloat16':
        pick = np.flatnonzero(np.abs(left) > 2.0 ** -18.5)
        k, q, w, a, b, left = (x[pick] for x in (k, q, w, a, b, left))
    k, q, w, a, b, left = (x[:64] for x in (k, q, w, a, b, left))
    n = len(k)
    assert n == 64
    cache, table, lengths = _make(d, [3] * n, 1, d, 16, dtype, slots=slots)
    rows = torch.zeros(2, n, 3, d, dtype=torch.float64)
    rows[0, :, 0, 0] = torch.tensor(k)
    rows[1, :, :, 5] = torch.tensor(np.stack([np.ones(n), -a, -b], 1))
    for x, pages in zip(rows, (cache.k_pages, cache.v_pages)):
        pages[table[:, 0].long(), 0, :3] = x.to(t).cuda()
    qs = torch.zeros(n, 1, d, dtype=torch.float64)
    qs[:, 0, 0] = torch.tensor(q)
    out, _ = cache.attend(qs.to(t).cuda(), table, lengths, scale=1.0)
    got, want = out[:, 0, 5].double().cpu().numpy(), left / (2 + w)
    tol = ((1.4 + 2) * U * w + 4 * U + {'float32': 0, 'bfloat16': 0.5, 'float16': 4}[dtype] * U * w) / (2 + w)
    tol += np.abs(want) * (torch.finfo(t).eps / 2 + 4 * U) + torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2
    assert (np.abs(got - want) <= tol).all(), (np.abs(got - want) / tol).max()
    assert (out[:, 0, :5] == 0).all() and (out[:, 0, 6:] == 0).all()


@pytest.mark.parametrize('inplace', [False, True])
@pytest.mark.parametrize('recent', [0, 7])
def test_evict_one_over_in_a_table_shared_by_workgroups(inplace, recent):
    """A token over the budget where a head is more than one workgroup holds; masses all different, and all the same."""
    import torch
    from tests.test_gpu_kv_cache import _check_evict
    for same in (False, True):
        lens = [20001, 300, 0, 20000, 20001]
        cache, table, lengths = _make(81, lens, 2, 64, 32, 'float16')
        g = torch.Generator().manual_seed(4)
        shape = (len(lens), 2, table.shape[1] * 32)
        mass = torch.full(shape, 0.5) if same else torch.rand(shape, generator=g)
        pos = torch.stack([torch.randperm(shape[2], generator=g) for _ in range(shape[0] * 2)]).view(shape).to(torch.int32)
        _check_evict(cache, table, lengths, mass.cuda(), pos.cuda(), 20000, recent, inplace)


def test_two_threads_on_one_cache():
    """Appends, attentions and evictions of two threads, each on a stream of its own, over one pool: the bits of one after the other."""
    import threading

    import torch
    lens = [[600, 31, 2], [90, 64, 1200]]
    cache, table, lengths = _make(91, lens[0] + lens[1], 2, 64, 16, 'bfloat16', slots=1216)
    own = [(table[3 * i:3 * i + 3], lengths[3 * i:3 * i + 3]) for i in range(2)]
    pages = [x.clone() for x in (cache.k_pages, cache.v_pages)]
    qs = [[_q(100 * i + j, 3, 4, 64, 'bfloat16') for j in range(6)] for i in range(2)]
    sides = torch.rand(3, 2, 1216, generator=torch.Generator().manual_seed(5)).cuda()

    def work(i, out):
        tab, n = own[i]
        n, mass = n.clone(), sides.clone()
        pos = torch.arange(1216, dtype=torch.int32, device='cuda').expand(3, 2, 1216).contiguous()
        for j in range(6):
            o, lse = cache.attend(qs[i][j], tab, n, mass=mass)
            n, mass, pos = cache.evict(tab, n, mass, pos, 500 - 60 * j, 4)
            n = cache.append(qs[i][j][:, None, :2], qs[i][j][:, None, 2:], tab, n - 1, first=pos.amax((1, 2)) + 1, mass=mass, positions=pos)
            out += [o, lse, n, mass.clone(), pos.clone()]

    want = [[], []]
    for i in range(2):
        work(i, want[i])
    torch.cuda.synchronize()
    final = [x.clone() for x in (cache.k_pages, cache.v_pages)]
    for _ in range(3):
        for x, y in zip((cache.k_pages, cache.v_pages), pages):
            x.copy_(y)
        torch.cuda.synchronize()
        got, threads = [[], []], []
        for i in range(2):
            def run(i=i):
                with torch.cuda.stream(torch.cuda.Stream()):
                    work(i, got[i])
            threads.append(threading.Thread(target=run))
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        torch.cuda.synchronize()
        for i in range(2):
            assert len(got[i]) == 30 and all(_same(a, b) for a, b in zip(got[i], want[i]))
        assert all(_same(a, b) for a, b in zip((cache.k_pages, cache.v_pages), final))
    cache.status()


def test_a_pool_of_another_stream_that_goes_while_a_call_runs():
    """A pool made on one stream, its cache made and called on another: neither is given away before that call is over."""
    import torch
    from tacotron_amd.kv_cache import KvCache
    table = torch.zeros(1, 3, dtype=torch.int32, device='cuda')
    lengths = torch.full((1,), 40, dtype=torch.int32, device='cuda')
    q = _q(1, 1, 2, 64, 'float32')
    side = torch.cuda.Stream()
    pool = [torch.empty(1024, 1, 16, 64, device='cuda') for _ in range(2)]
    held = {x.data_ptr() for x in pool}
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        cache = KvCache(*pool)
        torch.cuda._sleep(400_000_000)
        out, lse = cache.attend(q, table, lengths)
    del cache, pool
    others = [torch.empty(1 << 20, dtype=torch.int32, device='cuda') for _ in range(4)]
    assert not side.query() and not held & {x.data_ptr() for x in others}
    torch.cuda.synchronize()
