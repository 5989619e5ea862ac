"""KvCache: a paged key-value cache on one GPU and the three calls that use it (include/taco.h, taco_kv_*): append rows,
attend one new token per sequence, evict by the attention tokens have drawn.

For decoders with dot-product attention over memories that are long, ragged or grow while they decode; the encoder memory of one
utterance (`TacoEngine.encode`, [T_in, 256]) is the simplest case: one kv head of dim 256, appended once, attended every step, the
collected `mass` being the alignments summed over the steps. (The Tacotron decoder itself attends additively and does not come here.)

The cache object holds the pool's geometry and a status word. Everything else - page tables, lengths, masses, positions -
is the caller's and is passed to each call, so one pool serves any number of batches and a captured HIP graph follows what
the tensors hold when it runs. Calls are queued on torch's current stream of the pool's device and synchronise nothing;
workspaces and results come from torch's allocator, so calls on several streams do not share any. A captured graph holds the
addresses of the pool and of the status word: the cache has to live as long as it is replayed. A serving form: no
gradients are recorded, and tensors that require one are refused while gradients are."""
import ctypes
import math

import torch

from . import _lib
from .engine import TacoError

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


class KvCache:
    def __init__(self, k_pages, v_pages):
        """k_pages, v_pages: [num_pages, kv_heads, page_size, head_dim] on a GPU, fp32 / bf16 / fp16; the rows of head_dim
        contiguous, the other strides free multiples of 16 bytes (a [num_pages, page_size, kv_heads, head_dim] pool is
        passed as its transpose(1, 2))."""
        for name, t in (('k_pages', k_pages), ('v_pages', v_pages)):
            if not isinstance(t, torch.Tensor) or t.dim() != 4 or t.dtype not in _DTYPES:
                raise TacoError('%s must be a tensor [num_pages, kv_heads, page_size, head_dim] of float32, bfloat16 or '
                                'float16' % name)
            if t.stride(3) != 1:
                raise TacoError('%s: rows of head_dim must be contiguous' % name)
            if any(n > 1 and st == 0 for n, st in zip(t.shape, t.stride())):
                raise TacoError('%s: an expanded tensor cannot be a pool' % name)
            if t.requires_grad:
                self._no_gradient(name)
        if k_pages.shape != v_pages.shape or k_pages.dtype != v_pages.dtype or k_pages.device != v_pages.device:
            raise TacoError('k_pages and v_pages must agree in shape, type and device')
        if k_pages.device.type != 'cuda':
            raise TacoError('KvCache needs a GPU; there is no CPU path')
        self.lib = _lib.load_library()
        self.k_pages, self.v_pages = k_pages, v_pages
        self.device, self.dtype, self._index = k_pages.device, k_pages.dtype, k_pages.device.index
        self.num_pages, self.kv_heads, self.page_size, self.head_dim = k_pages.shape
        own = torch.zeros(8, dtype=torch.int32, device=self.device)
        self._own, self._streams = own, set()
        with torch.cuda.device(self.device):
            if not torch.cuda.is_current_stream_capturing():
                torch.cuda.current_stream().synchronize()      # zeroed before a call of any stream may set a bit
        self._status, self._none = own[:1], own[4:]  # _none: 16 bytes, the workspace of attentions that use none
        p = _lib.TacoKvPool()
        p.struct_size = ctypes.sizeof(p)
        p.device, p.dtype = self.device.index, _DTYPES[self.dtype]
        p.num_pages, p.kv_heads, p.page_size, p.head_dim = k_pages.shape
        p.k, p.v, p.status = k_pages.data_ptr(), v_pages.data_ptr(), self._status.data_ptr()
        p.k_page_stride, p.k_head_stride, p.k_token_stride = k_pages.stride()[:3]
        p.v_page_stride, p.v_head_stride, p.v_token_stride = v_pages.stride()[:3]
        self._pool, self._ref = p, ctypes.byref(p)
        self._esize = k_pages.element_size()
        self._need = {}
        # the library's own checks of the geometry, now and not at the first call
        if not self.lib.taco_kv_evict_workspace_bytes(self._ref, 1, 1, 1):
            raise TacoError(_lib.last_error())

    @classmethod
    def empty(cls, num_pages, page_size, kv_heads, head_dim, dtype=torch.float32, device=0):
        """A cache over a pool of its own (uninitialised)."""
        shape = (num_pages, kv_heads, page_size, head_dim)
        device = torch.device('cuda', device) if isinstance(device, int) else torch.device(device)
        return cls(torch.empty(shape, dtype=dtype, device=device), torch.empty(shape, dtype=dtype, device=device))

    def status(self):
        """Synchronises the device; raises TacoError if any call since the last status() met a length outside its table's
        capacity or a page id outside the pool (which it treated as masked)."""
        torch.cuda.synchronize(self.device)
        taken = torch.empty_like(self._status)
        self._check(self.lib.taco_kv_take_status(self._ref, taken.data_ptr(), self._stream()))
        bits = int(taken.item())
        if bits:
            raise TacoError('KvCache: ' + ', '.join(m for b, m in ((1, 'a page id outside the pool'),
                                                                  (2, "a length outside the page table's capacity"))
                                                    if bits & b))

    # ---- argument checks
    def _check(self, rc):
        if rc != 0:
            raise TacoError(_lib.last_error())

    def _no_gradient(self, name):
        if torch.is_grad_enabled():
            raise TacoError('%s requires a gradient, and KvCache records none: pass it detached or call under torch.no_grad()' % name)

    # (get_device, an int, is -1 for host tensors; comparing devices builds objects)
    def _ints(self, t, name, B):
        if not isinstance(t, torch.Tensor) or t.dtype is not torch.int32 or t.get_device() != self._index or t.shape != (B,):
            raise TacoError('%s must be an int32 tensor [%d] on %s' % (name, B, self.device))
        return t if t.is_contiguous() else t.contiguous()

    def _table(self, t, B=None):
        """The page table, rows contiguous, its rows' distance and its shape."""
        if not isinstance(t, torch.Tensor) or t.dtype is not torch.int32 or t.get_device() != self._index or t.dim() != 2 or not t.numel():
            raise TacoError('page_table must be an int32 tensor [B, max_pages] on %s' % self.device)
        n, max_pages = t.shape
        if B is not None and n != B:
            raise TacoError('page_table must have a row for each of the %d sequences' % B)
        ld, one = t.stride()
        if one != 1 or ld < max_pages:
            t, ld = t.contiguous(), max_pages
        return t, ld, n, max_pages

    def _side(self, t, name, dtype, B, slots):
        if isinstance(t, torch.Tensor) and t.dtype is dtype and t.get_device() == self._index and t.dim() == 3 and t.is_contiguous():
            if t.requires_grad:
                self._no_gradient(name)
            n, h, ld = t.shape
            if n == B and h == self.kv_heads and ld >= slots:
                return ld
        raise TacoError('%s must be a contiguous %s tensor [%d, %d, at least %d] on %s'
                        % (name, str(dtype)[6:], B, self.kv_heads, slots, self.device))

    def _rows(self, t, name):
        """Rows of head_dim elements: contiguous, 16-byte aligned, or copied to be. Returns it and its strides."""
        if t.dtype is not self.dtype or t.get_device() != self._index:
            raise TacoError('%s must be %s on %s, as the pool' % (name, str(self.dtype)[6:], self.device))
        if t.requires_grad:
            self._no_gradient(name)
        st = t.stride()
        bits = t.data_ptr()
        for s in st[:-1]:
            bits |= s * self._esize
        if st[-1] != 1 or bits & 15:
            t = t.clone(memory_format=torch.contiguous_format)
            st = t.stride()
        return t, st

    def _workspace(self, query, *sizes):
        """Scratch of one call, from torch's allocator. Its size depends on the sizes alone and is asked for once."""
        need = self._need.get((query, sizes))
        if need is None:
            need = getattr(self.lib, query)(self._ref, *sizes)
            if not need:
                raise TacoError(_lib.last_error())
            if len(self._need) >= 256:
                self._need.clear()
            self._need[(query, sizes)] = need
        # The one buffer that calls share is for those that leave it alone: an attention that is said to need the least there
        # is. (An eviction of one head to one token uses all of its 16 bytes.)
        if need <= 16 and query == 'taco_kv_attend_workspace_bytes':
            return self._none, need
        return torch.empty(need, dtype=torch.uint8, device=self.device), need

    def _stream(self):
        """The stream a call is queued on. The cache holds the status word and the pool: torch's allocator is told of every
        stream that calls ran on, so that it waits for them before it gives that memory to other tensors."""
        # the handle alone: torch.cuda.current_stream builds an object around it
        s = torch._C._cuda_getCurrentRawStream(self._index)
        if s not in self._streams:
            for t in (self._own, self.k_pages, self.v_pages):
                t.record_stream(torch.cuda.current_stream(self.device))
            self._streams.add(s)
        return s

    # ---- the operators
    def append(self, k, v, page_table, starts, counts=None, first=None, mass=None, positions=None):
        """k, v [B, T, kv_heads, head_dim] -> slots starts[b] .. starts[b] + counts[b] - 1 (counts None: all T) of each
        sequence's pages. mass [B, kv_heads, slots] becomes 0 there, positions [B, kv_heads, slots] first[b] + t (first
        None: starts, which after an eviction are not the tokens' own any more). Returns the new lengths, starts + counts.
        The pages written must belong to one sequence; T * kv_heads is at most 2^25."""
        for name, t in (('k', k), ('v', v)):
            if not isinstance(t, torch.Tensor) or t.dim() != 4 or t.shape[2] != self.kv_heads or t.shape[3] != self.head_dim or not t.numel():
                raise TacoError('%s must be [B, T, %d, %d]' % (name, self.kv_heads, self.head_dim))
        if k.shape != v.shape:
            raise TacoError('k and v must have the same shape')
        B, T = k.shape[:2]
        (k, ks), (v, vs) = self._rows(k, 'k'), self._rows(v, 'v')
        table, table_ld, _, max_pages = self._table(page_table, B)
        ld = slots = max_pages * self.page_size
        starts = self._ints(starts, 'starts', B)
        counts = self._ints(counts, 'counts', B) if counts is not None else None
        first = self._ints(first, 'first', B) if first is not None else None
        if mass is not None:
            ld = self._side(mass, 'mass', torch.float32, B, slots)
        if positions is not None:
            pos_ld = self._side(positions, 'positions', torch.int32, B, slots)
            if mass is not None and pos_ld != ld:
                raise TacoError('mass and positions must have the same shape')
            ld = pos_ld
        lengths = torch.empty_like(starts)           # (quicker than torch.empty)
        self._check(self.lib.taco_kv_append(
            self._ref, table.data_ptr(), table_ld, B, max_pages,
            k.data_ptr(), ks[0], ks[1], ks[2], v.data_ptr(), vs[0], vs[1], vs[2], T,
            starts.data_ptr(), counts.data_ptr() if counts is not None else None,
            first.data_ptr() if first is not None else None, mass.data_ptr() if mass is not None else None,
            positions.data_ptr() if positions is not None else None, ld, lengths.data_ptr(), self._stream()))
        return lengths

    def attend(self, q, page_table, lengths, scale=None, mass=None):
        """One new token per sequence: q [B, q_heads, head_dim], q_heads a multiple of kv_heads (query head i reads kv head
        i // (q_heads // kv_heads)), over the first lengths[b] slots. Returns (out [B, q_heads, head_dim] in the pool's
        type, lse [B, q_heads] float32, natural log). scale: default 1 / sqrt(head_dim). mass [B, kv_heads, slots], if
        given, gains each slot's attention weight, summed over the query heads of its kv head. A sequence of length 0
        gives out 0, lse -inf."""
        if not isinstance(q, torch.Tensor) or q.dim() != 3 or q.shape[2] != self.head_dim or not q.numel():
            raise TacoError('q must be [B, q_heads, %d]' % self.head_dim)
        B, hq, _ = q.shape
        q, qs = self._rows(q, 'q')
        table, table_ld, _, max_pages = self._table(page_table, B)
        lengths = self._ints(lengths, 'lengths', B)
        ld = 0
        if mass is not None:
            ld = self._side(mass, 'mass', torch.float32, B, max_pages * self.page_size)
        ws, need = self._workspace('taco_kv_attend_workspace_bytes', B, hq, max_pages, mass is not None)
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        lse = torch.empty((B, hq), dtype=torch.float32, device=self.device)
        self._check(self.lib.taco_kv_attend(
            self._ref, table.data_ptr(), table_ld, B, max_pages, lengths.data_ptr(), q.data_ptr(), qs[0],
            qs[1], hq, 1.0 / math.sqrt(self.head_dim) if scale is None else float(scale), out.data_ptr(),
            lse.data_ptr(), mass.data_ptr() if mass is not None else None, ld, ws.data_ptr(), need, self._stream()))
        return out, lse

    def evict(self, page_table, lengths, mass, positions, budget, recent=0, out=None):
        """Cuts every (sequence, kv head) to min(lengths[b], budget) tokens: the newest (positions above the greatest one -
        `recent`), then those of the greatest mass (ties: the lower slot; a token never attended has 0). Survivors from
        beyond the budget fill the slots that became empty, so slots end up in no order; `positions` tells which token a
        slot holds. Returns (lengths, mass, positions), new tensors, or `out` = three tensors to write, each of which may
        be the matching input itself. Slots from the new length on get mass 0 and position -1 and their pages may be given
        away. The pages must belong to one sequence."""
        table, table_ld, B, max_pages = self._table(page_table)
        lengths = self._ints(lengths, 'lengths', B)
        slots = max_pages * self.page_size
        ld = self._side(mass, 'mass', torch.float32, B, slots)
        if self._side(positions, 'positions', torch.int32, B, slots) != ld:
            raise TacoError('mass and positions must have the same shape')
        budget, recent = int(budget), int(recent)
        if budget < 1 or not 0 <= recent <= budget:
            raise TacoError('evict needs 0 <= recent <= budget and budget >= 1 (got recent %d, budget %d)' % (recent, budget))
        budget, recent = min(budget, slots), min(recent, slots)
        if out is None:
            new = (torch.empty_like(lengths), torch.empty_like(mass), torch.empty_like(positions))
        else:
            new = tuple(out)
            if len(new) != 3 or new[0] is not self._ints(new[0], 'out[0]', B):
                raise TacoError('out must be contiguous (lengths, mass, positions) tensors')
            for name, dtype, t in (('out[1]', torch.float32, new[1]), ('out[2]', torch.int32, new[2])):
                if self._side(t, name, dtype, B, slots) != ld:
                    raise TacoError('%s must have the shape of its input' % name)
        ws, need = self._workspace('taco_kv_evict_workspace_bytes', B, max_pages, budget)
        self._check(self.lib.taco_kv_evict(
            self._ref, table.data_ptr(), table_ld, B, max_pages, lengths.data_ptr(), mass.data_ptr(),
            positions.data_ptr(), ld, budget, recent, new[0].data_ptr(), new[1].data_ptr(), new[2].data_ptr(),
            ws.data_ptr(), need, self._stream()))
        return new
