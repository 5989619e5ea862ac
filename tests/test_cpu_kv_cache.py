"""The paged key-value cache without a GPU: what the C entries and KvCache refuse (before any device call), the layout of
the pool struct, and the 64-bit reference the GPU tests compare with."""
import ctypes
import os
import re

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _pool(**kw):
    from tacotron_amd import _lib
    p = _lib.TacoKvPool()
    p.struct_size = ctypes.sizeof(p)
    p.num_pages, p.kv_heads, p.page_size, p.head_dim = 4, 2, 16, 64
    p.k, p.v, p.status = 4096, 8192, 12288        # never dereferenced: every call here is refused
    p.k_token_stride = p.v_token_stride = 64
    p.k_head_stride = p.v_head_stride = 1024
    p.k_page_stride = p.v_page_stride = 2048
    for n, x in kw.items():
        setattr(p, n, x)
    return p


def _append(lib, pool, **kw):
    a = dict(table=16, table_ld=4, B=1, max_pages=4, k=16, ks=(128, 128, 64), v=16, vs=(128, 128, 64), T=1, starts=16, counts=None,
             first=None, mass=None, positions=None, side_ld=64, lengths=16)
    a.update(kw)
    return lib.taco_kv_append(ctypes.byref(pool) if pool is not None else None, a['table'], a['table_ld'], a['B'], a['max_pages'],
                              a['k'], *a['ks'], a['v'], *a['vs'], a['T'], a['starts'], a['counts'], a['first'], a['mass'],
                              a['positions'], a['side_ld'], a['lengths'], None)


def _attend(lib, pool, **kw):
    a = dict(table=16, table_ld=4, B=1, max_pages=4, lengths=16, q=16, qs=(128, 64), q_heads=2, scale=1.0, out=16, lse=16, mass=None,
             side_ld=64, ws=16, ws_bytes=1 << 30)
    a.update(kw)
    return lib.taco_kv_attend(ctypes.byref(pool), a['table'], a['table_ld'], a['B'], a['max_pages'], a['lengths'], a['q'], *a['qs'],
                              a['q_heads'], a['scale'], a['out'], a['lse'], a['mass'], a['side_ld'], a['ws'], a['ws_bytes'], None)


def _evict(lib, pool, **kw):
    a = dict(table=16, table_ld=4, B=1, max_pages=4, lengths=16, mass=16, positions=16, side_ld=64, budget=8, recent=0, lo=16, mo=16,
             po=16, ws=16, ws_bytes=1 << 30)
    a.update(kw)
    return lib.taco_kv_evict(ctypes.byref(pool), a['table'], a['table_ld'], a['B'], a['max_pages'], a['lengths'], a['mass'],
                             a['positions'], a['side_ld'], a['budget'], a['recent'], a['lo'], a['mo'], a['po'], a['ws'], a['ws_bytes'], None)


def test_pool_struct_matches_header():
    from tacotron_amd import _lib
    hdr = open(os.path.join(ROOT, 'include', 'taco.h')).read()
    body = hdr[hdr.index('typedef struct TacoKvPool {'):hdr.index('} TacoKvPool;')]
    body = re.sub(r'/\*.*?\*/', '', body, flags=re.S)
    want = []
    for t, names in re.findall(r'^\s*(uint32_t|int32_t\*?|int64_t|void\*)\s+([\w, ]+);', body, flags=re.M):
        want += [(n.strip(), t) for n in names.split(',')]
    ctype = {'uint32_t': ctypes.c_uint32, 'int32_t': ctypes.c_int32, 'int64_t': ctypes.c_int64, 'void*': ctypes.c_void_p,
             'int32_t*': ctypes.c_void_p}
    assert [(n, ctype[t]) for n, t in want] == list(_lib.TacoKvPool._fields_)


@pytest.mark.parametrize('bad,text', [
    (dict(struct_size=8), 'struct_size'), (dict(k=None), 'null'), (dict(v=None), 'null'), (dict(status=None), 'null'),
    (dict(dtype=3), 'dtype'), (dict(dtype=-1), 'dtype'), (dict(num_pages=0), 'page'), (dict(kv_heads=0), 'kv_heads'),
    (dict(kv_heads=1025), 'kv_heads'), (dict(page_size=4), 'page_size'), (dict(page_size=24), 'page_size'),
    (dict(page_size=512), 'page_size'), (dict(head_dim=96), 'head_dim'), (dict(head_dim=512), 'head_dim'),
    (dict(k_page_stride=-64), 'stride'), (dict(v_token_stride=66), 'stride'), (dict(k=4104), 'boundary'), (dict(device=-1), 'device')])
def test_pools_that_are_refused(bad, text):
    from tacotron_amd import _lib
    lib = _lib.load_library()
    p = _pool(**bad)
    for call in (_append, _attend, _evict):
        assert call(lib, p) < 0 and text in _lib.last_error(), (call.__name__, _lib.last_error())
    assert lib.taco_kv_attend_workspace_bytes(ctypes.byref(p), 1, 2, 4, 1) == 0
    assert lib.taco_kv_evict_workspace_bytes(ctypes.byref(p), 1, 4, 8) == 0
    assert _append(lib, None) < 0


@pytest.mark.parametrize('call,bad,text', [
    (_append, dict(B=0), 'B must'), (_append, dict(B=65536), 'B must'), (_append, dict(max_pages=0), 'max_pages'),
    (_append, dict(max_pages=1 << 27, table_ld=1 << 27), 'max_pages'), (_append, dict(table_ld=3), 'table'), (_append, dict(table=None), 'table'),
    (_append, dict(k=None), 'null'), (_append, dict(v=20), 'boundary'), (_append, dict(ks=(128, 128, 63)), 'stride'),
    (_append, dict(T=0), 'T must'), (_append, dict(T=1 << 26), 'T must'), (_append, dict(starts=None), 'null'), (_append, dict(lengths=None), 'null'),
    (_append, dict(mass=16, side_ld=63), 'side'), (_append, dict(positions=16, side_ld=63), 'side'),
    (_attend, dict(q_heads=3), 'q_heads'), (_attend, dict(q_heads=0), 'q_heads'), (_attend, dict(q=None), 'null'), (_attend, dict(q=24), 'boundary'),
    (_attend, dict(out=None), 'null'), (_attend, dict(out=20), 'boundary'), (_attend, dict(lse=None), 'null'),
    (_attend, dict(lengths=None), 'null'), (_attend, dict(scale=float('nan')), 'scale'), (_attend, dict(scale=float('inf')), 'scale'), (_attend, dict(scale=3e38), 'scale'), (_attend, dict(B=65535, q_heads=65534), 'too many'),
    (_attend, dict(B=65535, max_pages=1 << 20, table_ld=1 << 20), 'too many'),
    (_attend, dict(mass=16, side_ld=32), 'side'), (_attend, dict(ws=None), 'workspace'),
    (_evict, dict(budget=0), 'budget'), (_evict, dict(recent=-1), 'recent'), (_evict, dict(recent=9), 'recent'),
    (_evict, dict(side_ld=10), 'side'), (_evict, dict(mass=None), 'null'), (_evict, dict(po=None), 'null'),
    (_evict, dict(ws_bytes=16), 'workspace'), (_evict, dict(ws=None), 'workspace')])
def test_arguments_that_are_refused(call, bad, text):
    from tacotron_amd import _lib
    lib = _lib.load_library()
    assert call(lib, _pool(), **bad) < 0 and text in _lib.last_error(), _lib.last_error()


def test_workspaces_grow_with_the_call():
    from tacotron_amd import _lib
    lib = _lib.load_library()
    p = ctypes.byref(_pool())
    assert lib.taco_kv_attend_workspace_bytes(p, 1, 2, 4, 0) >= 16
    assert lib.taco_kv_attend_workspace_bytes(p, 1, 3, 4, 0) == 0 and 'q_heads' in _lib.last_error()
    assert lib.taco_kv_evict_workspace_bytes(p, 2, 4, 8) >= 2 * 2 * 2 * 8 * 4
    assert lib.taco_kv_evict_workspace_bytes(p, 2, 4, 1 << 30) == lib.taco_kv_evict_workspace_bytes(p, 2, 4, 64)
    assert lib.taco_kv_evict_workspace_bytes(p, 2, 4, 0) == 0 and 'budget' in _lib.last_error()


def test_python_refuses_cpu_pools():
    import torch
    from tacotron_amd.engine import TacoError
    from tacotron_amd.kv_cache import KvCache
    t = torch.zeros(4, 2, 16, 64)
    for k, v, text in [(t, t, 'GPU'), (t[0], t[0], 'num_pages'), (t.double(), t.double(), 'float32'), (t, t[:2], 'agree'),
                       (t.transpose(2, 3), t, 'contiguous'), (t, t.half(), 'agree'), (None, t, 'tensor'),
                       (t[:1].expand(4, 2, 16, 64), t, 'expanded')]:
        with pytest.raises(TacoError, match=text):
            KvCache(k, v)


def test_reference_attention_and_eviction():
    """The oracle itself, on cases small enough to be done by hand."""
    import torch
    from tests import kv_reference as R
    k = torch.zeros(2, 1, 8, 64)
    v = torch.arange(16.).reshape(2, 1, 8, 1).expand(2, 1, 8, 64).contiguous()
    table = torch.tensor([[1, 0]], dtype=torch.int32)
    out, _, lse, _, w, _ = R.attend(torch.ones(1, 1, 64), k, v, table, [9], 1.0)
    assert np.allclose(out, (sum(range(8, 16)) + 0) / 9) and np.allclose(lse, np.log(9)) and np.allclose(w[0], 1 / 9)
    mass = np.array([3., 1., 5., 0., 5., 2.], np.float32)
    pos = np.arange(6, dtype=np.int32)
    assert R.survivors(mass, pos, 3, 0).tolist() == [0, 2, 4]
    assert R.survivors(mass, pos, 2, 1).tolist() == [2, 5]
    assert R.survivors(mass, pos, 2, 2).tolist() == [4, 5]
    kk = np.arange(6.).reshape(1, 1, 6, 1)
    k2, _, m2, p2, n2 = R.evict(kk, kk, mass[None, None], pos[None, None], [6], 3, 0)
    assert k2[0, 0, :3, 0].tolist() == [0, 4, 2] and p2[0, 0].tolist() == [0, 4, 2, -1, -1, -1] and n2.tolist() == [3]
    assert m2[0, 0].tolist() == [3, 5, 5, 0, 0, 0]
