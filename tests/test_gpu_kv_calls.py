"""Calls of the key-value cache beside each other on the GPU: evictions on several streams and in captured graphs, and what the
cache object itself keeps."""
import pytest

from tests.test_gpu_kv_cache import _make

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
