"""What the key-value cache's calls share and refuse, without a GPU: workspaces, aliases and the variant builds of its source."""
import ctypes

import pytest

from tests.test_cpu_kv_cache import _append, _attend, _pool

NOWHERE = 1000      # a device that no machine has: a call that is not refused before ends there, and launches nothing


def _host_cache(**pool):
    """A KvCache on the host whose buffers are never touched by a kernel: for the parts of a call before its launch."""
    import torch
    from tacotron_amd import _lib
    from tacotron_amd.kv_cache import KvCache
    c = object.__new__(KvCache)
    c.lib, c._need, c._none, c.device = _lib.load_library(), {}, torch.zeros(4, dtype=torch.int32), torch.device('cpu')
    c._pool = _pool(**pool)
    c._ref = ctypes.byref(c._pool)
    return c


def test_every_eviction_has_a_workspace_of_its_own():
    """The smallest one too: a sequence, one kv head and a budget of 1 need 16 bytes, two counts and an entry of each list."""
    c = _host_cache(kv_heads=1)
    for max_pages, budget in ((4, 1), (1024, 1), (4, 2), (2048, 1)):
        a, b = (c._workspace('taco_kv_evict_workspace_bytes', 1, max_pages, budget) for _ in range(2))
        assert a[1] == b[1] and a[0].numel() * a[0].element_size() >= a[1]
        assert len({a[0].data_ptr(), b[0].data_ptr(), c._none.data_ptr()}) == 3
    assert c._workspace('taco_kv_evict_workspace_bytes', 1, 4, 1)[1] == 16


def test_attention_of_a_short_memory_uses_no_workspace():
    """Where the buffer that all calls may be given stands for "none": the library asks for the least there is only where the
    kernel takes none, and for more wherever it takes one."""
    c = _host_cache(kv_heads=1)
    ws, need = c._workspace('taco_kv_attend_workspace_bytes', 1, 1, 4, True)
    assert ws is c._none and need == 16 == ws.numel() * ws.element_size()
    for dim, max_pages in ((64, 64), (128, 64), (256, 1), (256, 4)):
        c = _host_cache(kv_heads=1, head_dim=dim)
        (a, need), (b, _) = (c._workspace('taco_kv_attend_workspace_bytes', 1, 1, max_pages, False) for _ in range(2))
        assert need > 16 and len({a.data_ptr(), b.data_ptr(), c._none.data_ptr()}) == 3


@pytest.mark.parametrize('which', ['starts', 'counts', 'first'])
@pytest.mark.parametrize('shift,refused', [(0, True), (4, True), (-12, True), (16, False), (-16, False)])
def test_append_refuses_to_write_lengths_over_what_it_reads(which, shift, refused):
    """A launch's workgroups read starts, counts and first while one of them writes the new lengths."""
    from tacotron_amd import _lib
    at = dict(starts=1 << 16, counts=2 << 16, first=3 << 16)
    args = dict(at, B=4, k=16, v=16, lengths=at[which] + shift)
    assert _append(_lib.load_library(), _pool(device=NOWHERE), **args) < 0
    assert ('lengths_out' if refused else 'device') in _lib.last_error(), _lib.last_error()


def test_append_without_counts_and_firsts():
    from tacotron_amd import _lib
    lib = _lib.load_library()
    assert _append(lib, _pool(device=NOWHERE), starts=1 << 16, lengths=2 << 16) < 0 and 'device' in _lib.last_error()
    assert _append(lib, _pool(device=NOWHERE), starts=1 << 16, lengths=1 << 16) < 0 and 'lengths_out' in _lib.last_error()


@pytest.mark.parametrize('out,lse,refused', [
    (0, None, True), (-256, None, True), (1536 + 16, None, True),                # over the queries of the first or last sequence
    (528, None, True), (512, None, False),                                       # the gap between them holds it just so
    (-1024, None, False), (1536 + 512, None, False),                             # before and behind them all
    (None, 0, True), (None, 512, False), (None, 1536 + 508, True)])              # lse: on a query, in a gap, on the last of them
def test_attend_refuses_to_write_over_its_queries(out, lse, refused):
    """Queries [2, 2, 64] fp32, 1536 bytes from one sequence's to the next's (512 bytes each): waves read them as they come to
    a head, when others may have written theirs."""
    from tacotron_amd import _lib
    q = 1 << 20
    args = dict(B=2, q=q, qs=(384, 64), out=(1 << 21) if out is None else q + out, lse=(1 << 22) if lse is None else q + lse)
    assert _attend(_lib.load_library(), _pool(device=NOWHERE), **args) < 0
    assert ('overlap' if refused else 'device') in _lib.last_error(), _lib.last_error()


@pytest.mark.parametrize('B,qs,refused', [(2, (128, 64), False), (1, (384, 64), False), (2, (384, 64), True), (1, (128, 128), True)])
def test_attend_in_place_takes_contiguous_queries(B, qs, refused):
    from tacotron_amd import _lib
    q = 1 << 20
    assert _attend(_lib.load_library(), _pool(device=NOWHERE), B=B, q=q, qs=qs, out=q, lse=1 << 22) < 0
    assert ('overlap' if refused else 'device') in _lib.last_error(), _lib.last_error()


@pytest.mark.parametrize('kw', [dict(), dict(head_dim=256), dict(dtype=1), dict(head_dim=128, dtype=2)])
@pytest.mark.parametrize('with_mass', [0, 1])
def test_attend_refuses_a_workspace_one_byte_short(kw, with_mass):
    """Tables past what the kernel without a workspace takes."""
    from tacotron_amd import _lib
    lib, p = _lib.load_library(), _pool(device=NOWHERE, **kw)
    args = dict(B=3, table_ld=400, max_pages=400, qs=(1024, 256), q=1 << 16, out=1 << 20, lse=1 << 24, mass=(1 << 28) if with_mass else None, side_ld=6400)
    need = lib.taco_kv_attend_workspace_bytes(ctypes.byref(p), 3, 2, 400, with_mass)
    assert need > 16
    assert _attend(lib, p, ws_bytes=need - 1, **args) < 0 and 'workspace' in _lib.last_error()
    assert _attend(lib, p, ws_bytes=need, **args) < 0 and 'device' in _lib.last_error()


def test_take_status_refusals():
    from tacotron_amd import _lib
    lib = _lib.load_library()
    p = _pool(device=NOWHERE)
    assert lib.taco_kv_take_status(None, 16, None) < 0 and 'null' in _lib.last_error()
    assert lib.taco_kv_take_status(ctypes.byref(p), None, None) < 0 and 'null' in _lib.last_error()
    assert lib.taco_kv_take_status(ctypes.byref(_pool(status=None)), 16, None) < 0 and 'null' in _lib.last_error()
    assert lib.taco_kv_take_status(ctypes.byref(p), 16, None) < 0 and 'device' in _lib.last_error()


def test_gradients_are_refused_and_not_dropped():
    """A serving form: what would need a gradient is an error while gradients are recorded, wherever it enters."""
    import torch
    from tacotron_amd.engine import TacoError
    from tacotron_amd.kv_cache import KvCache
    c = _host_cache()
    c._index, c._esize, c.dtype, c.kv_heads = -1, 4, torch.float32, 2
    for t in (torch.zeros(2, 6, 64), torch.zeros(2, 3, 2, 64), torch.zeros(2, 65, 64)[:, 1:]):
        leaf = t.clone().requires_grad_()
        for x in (leaf, leaf * 2, leaf[:, 1:]):
            with pytest.raises(TacoError, match='gradient'):
                c._rows(x, 'q')
            with torch.no_grad():
                c._rows(x, 'q')
            c._rows(x.detach(), 'q')
    mass = torch.zeros(1, 2, 64, requires_grad=True)
    with pytest.raises(TacoError, match='gradient'):
        c._side(mass, 'mass', torch.float32, 1, 64)
    with torch.no_grad():
        assert c._side(mass, 'mass', torch.float32, 1, 64) == 64
    assert c._side(mass.detach(), 'mass', torch.float32, 1, 64) == 64
    pool = torch.zeros(4, 2, 16, 64)
    for k, v in ((pool.clone().requires_grad_(), pool), (pool, pool.clone().requires_grad_())):
        with pytest.raises(TacoError, match='gradient'):
            KvCache(k, v)


def test_attend_in_place_of_one_query_head():
    """One head: its stride says nothing."""
    from tacotron_amd import _lib
    args = dict(B=2, q=1 << 20, q_heads=1, out=1 << 20, lse=1 << 22)
    for qs, refused in (((64, 64), False), ((64, 4096), False), ((128, 64), True)):
        assert _attend(_lib.load_library(), _pool(device=NOWHERE, kv_heads=1), qs=qs, **args) < 0
        assert ('overlap' if refused else 'device') in _lib.last_error(), (qs, _lib.last_error())
