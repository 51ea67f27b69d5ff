"""Prompts of different lengths in one pass, and a paged KV cache: attention over packed prompts (`packed_attention`), and `KvPages` --
pages taken and filled (`reserve`, `append`), shared and copied (`fork`, `copy`), given back (`free`), moved together (`compact`), and
decode attention that reads a prefix shared by the whole batch once (`attend`). The C entry points are orc_attention_packed and
orc_kv_* of include/oracle_hip.h; tensors are bf16 or fp16 on one GPU, and every call runs on that GPU's current stream without waiting for it. There are no
derivatives: tensors that want a gradient, or have a tangent, are refused."""
import ctypes as C
import functools
import struct

import torch
from torch.autograd import forward_ad

from . import _lib

_DTYPES = {torch.bfloat16: 0, torch.float16: 1}
_ERRORS = ((1, 'a row outside the table'), (2, 'a row named twice (or a fork onto one of its sources)'), (4, 'a bad token count'),
           (8, 'a row longer than the table is wide'), (16, 'too few free pages'), (32, 'a fork onto a row that holds tokens'),
           (64, 'a page outside the pool'), (128, 'rows that do not share the prefix they were attended with'))


# strides as the C entries read them (an array of c_int64 takes four times as long to make)
_I64x4, _I64x8 = struct.Struct('4q').pack, struct.Struct('8q').pack
_raw_stream, _current = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice


class _Held:
    """Tensors that an object keeps and its calls read on whatever stream is current: noted once for every such stream but the one that they were made on, so
    that their memory is not given to others before that stream is through with it when the object is let go. (A captured graph's replays are not
    noted: who replays it keeps the object.)"""

    def _hold(self, *tensors):
        self._tensors, self._streams = tensors, {_raw_stream(tensors[0].get_device())} if tensors[0].is_cuda else set()

    def _note(self, device, stream):
        if stream in self._streams:
            return
        with torch.cuda.device(device):
            if not torch.cuda.is_current_stream_capturing():
                for t in self._tensors:
                    t.record_stream(torch.cuda.current_stream())
                self._streams.add(stream)


def _run(held, device, name, *args):
    """The C entry `name` with args and the current stream of `device`, with `device` the current one; it reads the tensors of `held`."""
    fn, i = getattr(_lib.lib(), name), device.index
    stream = _raw_stream(i)
    if stream not in held._streams:
        held._note(device, stream)
    if _current() == i:
        rc = fn(*args, stream)
    else:
        with torch.cuda.device(i):
            rc = fn(*args, stream)
    if rc != 0:
        _lib.check(rc, name)


def _chk(t, name, dim, dtype=None, device=None):
    if device is not None and type(t) is torch.Tensor and t.get_device() == device.index and t.dtype is dtype and t.dim() == dim and not t.requires_grad:
        return
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f'{name} must be a CUDA tensor')
    if t.dim() != dim:
        raise ValueError(f'{name} must have {dim} dimensions, got {tuple(t.shape)}')
    if dtype is None:
        if t.dtype not in _DTYPES:
            raise ValueError(f'{name} must be bfloat16 or float16, got {t.dtype}')
    elif t.dtype is not dtype:
        raise ValueError(f'{name} must be {dtype}, got {t.dtype}')
    if device is not None and t.device != device:
        raise ValueError(f'{name} is on {t.device}, not on {device}')
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f'{name} requires a gradient and the call has none: detach it, or call under torch.no_grad()')


def _no_tangents(**tensors):
    """Inside a level of forward-mode differentiation (nothing to look for outside)"""
    for name, t in tensors.items():
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise ValueError(f'{name} has a tangent and the call has no derivative: pass forward_ad.unpack_dual({name}).primal')


def _place(t, name):
    """(token stride, head stride, address) of (tokens, heads, head_dim)"""
    ts, hs, es = t.stride()
    p = t.data_ptr()
    if es != 1 or (ts | hs) & 7 or p & 15:
        n, heads, hd = t.shape
        ts, hs = ts if n > 1 else 0, hs if heads > 1 else 0      # the stride of one element does not matter
        if es != 1 and hd > 1:
            raise ValueError(f'{name}: the last dimension must be contiguous')
        if (ts | hs) & 7 or p & 15:
            raise ValueError(f'{name}: token and head strides must be multiples of 8 elements and the tensor must start on 16 bytes, '
                             f'got strides {tuple(t.stride())} at {p % 16} bytes past 16')
    return ts, hs, p


def _overlaps_itself(t):
    """whether two of t's elements may share memory (an output must not be an expanded view)"""
    need = 1
    for size, stride in sorted(zip(t.shape, t.stride()), key=lambda x: x[1]):
        if size > 1:
            if stride < need:
                return True
            need = stride * (size - 1) + need
    return False


def _ints(t, name, device, n=None):
    _chk(t, name, 1, torch.int32, device)
    if not t.is_contiguous():
        raise ValueError(f'{name} must be contiguous')
    if n is not None and t.numel() != n:
        raise ValueError(f'{name} must hold {n} values, got {t.numel()}')
    return t.data_ptr()


def _out(out, like, name='out'):
    if out is None:
        return None
    _chk(out, name, 3, like.dtype, like.device)
    if out.shape != like.shape:
        raise ValueError(f'{name} must have the shape {tuple(like.shape)}, got {tuple(out.shape)}')
    if _overlaps_itself(out):
        raise ValueError(f'{name} must not be an expanded view')
    return out


class PackedPlan(_Held):
    """The query tiles of prompts that lie one behind the other, `lens` tokens each (0 allowed), on `device`: made once for a batch
    and used for every layer. It holds for any number of heads. (Making it copies to the GPU and waits: not while a graph is captured.)"""

    def __init__(self, lens, device='cuda'):
        self.lens = [int(x) for x in lens]
        n = len(self.lens)
        if any(x < 0 or x > 0x7fffffff for x in self.lens) or sum(self.lens) > 0x7fffffff:
            raise ValueError('lengths must not be negative, nor add up to more than 2^31 - 1')
        self.total = sum(self.lens)
        lib = _lib.lib()
        arr = (C.c_int32 * max(n, 1))(*self.lens)
        self.n_work = lib.orc_attn_plan(arr, n, None, 0)
        if self.n_work < 0:
            _lib.check(self.n_work, 'orc_attn_plan')
        work = torch.empty(max(self.n_work, 1), 4, dtype=torch.int32)
        if lib.orc_attn_plan(arr, n, work.data_ptr(), self.n_work) < 0:
            _lib.check(-1, 'orc_attn_plan')
        self.work = work.to(device)
        self._hold(self.work)


def packed_attention(q, k, v, plan, scale=None, out=None):
    """Causal attention inside every prompt of `plan`: q (T, Hq, hd), k / v (T, Hkv, hd) with T >= plan.total, hd 64 or 128, Hq a multiple of
    Hkv; slices of a fused projection are taken as they are. scale defaults to hd ** -0.5. Rows of `out` behind the last prompt are left
    as they are (zero in a tensor made here). `out` may be q; one that lies over q in another way, or over k or v, is refused."""
    _chk(q, 'q', 3)
    dtype, device = q.dtype, q.device
    _chk(k, 'k', 3, dtype, device)
    _chk(v, 'v', 3, dtype, device)
    if forward_ad._current_level >= 0:
        _no_tangents(q=q, k=k, v=v, out=out)
    (tokens, hq, hd), (k_tokens, hkv, k_hd) = q.shape, k.shape
    if k.shape != v.shape or k_tokens != tokens or k_hd != hd:
        raise ValueError(f'q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not belong together')
    if hd not in (64, 128):
        raise ValueError(f'head_dim must be 64 or 128, got {hd}')
    if hkv < 1 or hq < 1 or hq % hkv:
        raise ValueError(f'{hq} query heads are not a multiple of {hkv} K/V heads')
    if plan.total > tokens:
        raise ValueError(f'the plan covers {plan.total} tokens, q has {tokens}')
    if plan.work.device != device:
        raise ValueError(f'the plan is on {plan.work.device}, not on {device}')
    scale = hd ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < 1e30:
        raise ValueError(f'scale must be positive and finite, got {scale}')
    out = _out(out, q)
    if out is None:
        out = (torch.empty_like if plan.total == tokens else torch.zeros_like)(q, memory_format=torch.contiguous_format)
    qt, qh, qp = _place(q, 'q')
    kt, kh, kp = _place(k, 'k')
    vt, vh, vp = _place(v, 'v')
    ot, oh, op = _place(out, 'out')
    _run(plan, device, 'orc_attention_packed', qp, kp, vp, op, _I64x8(qt, qh, kt, kh, vt, vh, ot, oh), plan.work.data_ptr(), plan.n_work, plan.total,
         hq, hkv, hd, _DTYPES[dtype], scale)
    return out


class KvPages(_Held):
    """A paged KV cache. kv (n_layers, 2, n_pages, n_kv_heads, page_size, head_dim) holds the tokens; table (max_rows, max_row_pages) the
    pages of every row (-1: none), lens (max_rows,) its tokens, refs (n_pages,) how many rows hold a page -- all on the GPU, so no call waits for it
    and all of them can be captured into a graph. Lists of rows and counts are int32 tensors there. A call whose lists are wrong, or that
    finds too few free pages, changes nothing and leaves a note that `check()` raises. The caller orders the calls on one cache (one
    stream, or events). A page that several rows hold is full and is not written again."""

    def __init__(self, n_layers, n_pages, n_kv_heads, head_dim, page_size=64, max_rows=64, max_row_pages=64, dtype=torch.bfloat16, device='cuda'):
        if min(n_layers, n_pages, n_kv_heads, max_rows, max_row_pages) < 1:
            raise ValueError('every size of the cache must be at least 1')
        if page_size not in (16, 32, 64, 128):
            raise ValueError(f'page_size must be 16, 32, 64 or 128, got {page_size}')
        if head_dim not in (64, 128):
            raise ValueError(f'head_dim must be 64 or 128, got {head_dim}')
        if dtype not in _DTYPES:
            raise ValueError(f'dtype must be bfloat16 or float16, got {dtype}')
        i32 = dict(dtype=torch.int32, device=device)
        self._adopt(torch.zeros(n_layers, 2, n_pages, n_kv_heads, page_size, head_dim, dtype=dtype, device=device),
                    torch.full((max_rows, max_row_pages), -1, **i32), torch.zeros(max_rows, **i32), torch.zeros(n_pages, **i32))

    @classmethod
    def wrap(cls, kv, table, lens, refs):
        """A cache over tensors that exist already, in the layout of the class; they are used, not copied."""
        self = cls.__new__(cls)
        self._adopt(kv, table, lens, refs)
        return self

    def _adopt(self, kv, table, lens, refs):
        _chk(kv, 'kv', 6)
        if forward_ad._current_level >= 0:
            _no_tangents(kv=kv)
        for t, name, dim in ((table, 'table', 2), (lens, 'lens', 1), (refs, 'refs', 1)):
            _chk(t, name, dim, torch.int32, kv.device)
        if not all(t.is_contiguous() for t in (kv, table, lens, refs)) or kv.data_ptr() % 16:
            raise ValueError('kv, table, lens and refs must be contiguous, and kv must start on 16 bytes')
        layers, two, n_pages, hkv, page, hd = kv.shape
        if two != 2 or page not in (16, 32, 64, 128) or hd not in (64, 128) or min(layers, n_pages, hkv) < 1:
            raise ValueError(f'kv must be (n_layers, 2, n_pages, n_kv_heads, 16 | 32 | 64 | 128, 64 | 128), got {tuple(kv.shape)}')
        if lens.numel() != table.shape[0] or refs.numel() != n_pages or not 1 <= table.shape[0] <= 65536 or not 1 <= table.shape[1] <= 1 << 20:
            raise ValueError(f'table {tuple(table.shape)}, lens {tuple(lens.shape)} and refs {tuple(refs.shape)} do not belong to {n_pages} pages')
        if n_pages * page > 0x7fffffff:
            raise ValueError('the pool holds more than 2^31 - 1 tokens')
        self.kv, self.table, self.lens, self.refs = kv, table, lens, refs
        self.device, self.dtype, self.n_layers, self.n_kv_heads, self.page_size, self.head_dim = kv.device, kv.dtype, layers, hkv, page, hd
        self.row_tokens = table.shape[1] * page      # the most a row can hold
        self.status = torch.zeros(1, dtype=torch.int32, device=kv.device)
        self._work = torch.zeros(8 + 4 * n_pages, dtype=torch.int32, device=kv.device)
        self._hold(kv, table, lens, refs, self.status, self._work)
        self._c = _lib.OrcKvPages(*[t.data_ptr() for t in (kv, table, lens, refs, self.status, self._work)], layers, n_pages, hkv, page, hd,
                                  table.shape[0], table.shape[1], _DTYPES[kv.dtype])
        self._ref = ref = C.byref(self._c)

        @functools.lru_cache(256)
        def attend_ws(n, hq, prefix):      # (no self in it, so no cycle keeps the pool)
            size = _lib.lib().orc_kv_attend_ws(ref, n, hq, prefix)
            if size < 0:
                _lib.check(-1, 'orc_kv_attend_ws')
            return size
        self._attend_ws = attend_ws

    def _call(self, name, *args):
        _run(self, self.device, name, self._ref, *args)

    def _rows(self, rows, name='rows', n=None):
        p = _ints(rows, name, self.device, n)
        if rows.numel() > 1024:
            raise ValueError(f'{name}: at most 1024 rows a call, got {rows.numel()}')
        return p

    def check(self):
        """Waits for the GPU and raises if a call since the last check was refused there."""
        bits = int(self.status.item())
        if bits:
            self.status.zero_()
            raise _lib.OracleHipError('KvPages: ' + '; '.join(text for bit, text in _ERRORS if bits & bit))

    def reserve(self, rows, counts=None, total=None):
        """Room for counts[i] more tokens (None: one) of every row: takes the lowest free pages and returns the new tokens' places (int32, `total` of
        them, the rows' tokens one behind the other, -1 behind the last) for `append`. total: the sum of counts, which the host has to know; it
        may be larger. The places hold until a `compact` in place, or until the row is freed."""
        r = self._rows(rows)
        n = rows.numel()
        c = None if counts is None else _ints(counts, 'counts', self.device, n)
        if total is None:
            if counts is not None:
                raise ValueError('total is needed with counts')
            total = n
        if not 0 <= total <= 1 << 20:
            raise ValueError(f'total must be 0..2^20, got {total}')
        slots = rows.new_empty(int(total))
        self._call('orc_kv_reserve', r, c, n, slots.data_ptr(), int(total))
        return slots

    def append(self, layer, slots, k, v):
        """k / v (T, n_kv_heads, head_dim) of one layer into the places of `reserve`, each named once; a place of -1 is skipped. k and v may be
        views of the cache, but not of the places that are written."""
        _chk(k, 'k', 3, self.dtype, self.device)
        _chk(v, 'v', 3, self.dtype, self.device)
        if forward_ad._current_level >= 0:
            _no_tangents(k=k, v=v)
        s = _ints(slots, 'slots', self.device)
        want = (slots.numel(), self.n_kv_heads, self.head_dim)
        if k.shape != want or v.shape != want:
            raise ValueError(f'k {tuple(k.shape)} and v {tuple(v.shape)} must be {want}')
        self._layer(layer)
        (kt, kh, kp), (vt, vh, vp) = _place(k, 'k'), _place(v, 'v')
        self._call('orc_kv_append', int(layer), s, want[0], kp, vp, _I64x4(kt, kh, vt, vh))

    def _layer(self, layer):
        if not 0 <= layer < self.n_layers:
            raise ValueError(f'layer {layer} outside 0..{self.n_layers - 1}')

    def _fork(self, src, dst, n_tokens, share):
        if n_tokens is not None and not 0 <= n_tokens <= 0x7fffffff:
            raise ValueError(f'n_tokens must not be negative, got {n_tokens}')
        n_tokens = -1 if n_tokens is None else int(n_tokens)
        self._call('orc_kv_fork', self._rows(src, 'src'), self._rows(dst, 'dst', src.numel()), src.numel(), n_tokens, share)

    def fork(self, src, dst, n_tokens=None):
        """The empty rows dst[i] become rows src[i] (their first n_tokens tokens): full pages are shared, the part page is copied. A row can be
        forked to many; no src row may be among dst. What was reserved for a src row is appended first, in every layer."""
        self._fork(src, dst, n_tokens, 1)

    def copy(self, src, dst, n_tokens=None):
        """As `fork`, with pages of their own for every token."""
        self._fork(src, dst, n_tokens, 0)

    def free(self, rows):
        """The rows give their pages back and hold no tokens."""
        self._call('orc_kv_free', self._rows(rows), rows.numel())

    def compact(self, into=None):
        """Held pages to the front of the pool: in place, the pages that stick out move into the holes, and places that `reserve` gave hold no
        more. into: another cache of the same geometry (n_pages may differ), which becomes a copy of this one without the holes; this one
        stays as it is. Too few pages there: a note that into.check() raises, and nothing is changed."""
        if into is not None and into.device != self.device:
            raise ValueError(f'into is on {into.device}, not on {self.device}')
        if into is not None:
            into._note(self.device, _raw_stream(self.device.index))
        self._call('orc_kv_compact', None if into is None else into._ref)

    def attend(self, layer, q, rows, prefix_tokens=0, limits=None, scale=None, out=None):
        """Attention of one token per query: q (n, Hq, hd), query i over the first limits[i] tokens (None: all) of row rows[i], Hq a multiple of
        n_kv_heads. The first prefix_tokens (a multiple of page_size) are on the same pages in every named row (`fork`) and are read
        once for all of them; a query that ends inside them (by its limit, or a shorter row) makes the call slower, up to three times. A row
        can be named more than once (several tokens of a question, with their limits). A query without tokens gives zeros (one whose scores are
        all -inf NaN); what lies behind a query's tokens is not seen, infinities and NaN included. `out` may be q; one that lies over q in
        another way, or over the pool, is refused."""
        _chk(q, 'q', 3, self.dtype, self.device)
        if forward_ad._current_level >= 0:
            _no_tangents(q=q, out=out)
        n, hq, hd = q.shape
        if hd != self.head_dim:
            raise ValueError(f'head_dim of q is {hd}, of the cache {self.head_dim}')
        if hq < 1 or hq % self.n_kv_heads:
            raise ValueError(f'{hq} query heads are not a multiple of {self.n_kv_heads} K/V heads')
        self._layer(layer)
        if not 0 <= prefix_tokens <= self.row_tokens or prefix_tokens % self.page_size:
            raise ValueError(f'prefix_tokens must be a multiple of page_size {self.page_size} inside a row, got {prefix_tokens}')
        r = self._rows(rows, n=n)
        lim = None if limits is None else _ints(limits, 'limits', self.device, n)
        scale = hd ** -0.5 if scale is None else float(scale)
        if not 0.0 < scale < 1e30:
            raise ValueError(f'scale must be positive and finite, got {scale}')
        out = _out(out, q)
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        size = self._attend_ws(n, hq, int(prefix_tokens))
        ws = q.new_empty(size >> 1) if size else None
        (qt, qh, qp), (ot, oh, op) = _place(q, 'q'), _place(out, 'out')
        self._call('orc_kv_attend', int(layer), qp, op, _I64x4(qt, qh, ot, oh), r, lim, n, hq, int(prefix_tokens), scale, ws.data_ptr() if size else None)
        return out
