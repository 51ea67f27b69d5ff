"""CPU: what the paged KV cache and the packed attention refuse, and the plan of packed prompts."""
import ctypes as C

import numpy as np
import pytest
import torch

import __graft_entry__
from oracle_amd import _lib
from oracle_amd.paged import KvPages, PackedPlan, packed_attention


@pytest.fixture(scope='module')
def lib():
    __graft_entry__.build()
    return _lib.lib()


@pytest.mark.parametrize('lens', [[], [0], [1], [5, 0, 128, 129, 1, 700], [256, 255, 257], [2305] * 3 + [1] * 40])
def test_plan_covers_every_row_once_and_runs_a_prompts_tiles_together(lib, lens):
    arr = (C.c_int32 * max(len(lens), 1))(*lens)
    n = lib.orc_attn_plan(arr, len(lens), None, 0)
    work = np.full((n + 1, 4), -7, dtype=np.int32)
    assert lib.orc_attn_plan(arr, len(lens), work.ctypes.data, n) == n
    assert (work[n] == -7).all()
    starts = np.cumsum([0] + lens).tolist()
    tile = 128
    want = [(s, x, q0, 0) for x, s in sorted(zip(lens, starts), key=lambda y: (-y[0], y[1])) for q0 in reversed(range(0, x, tile))]
    last = n // 4       # these by their keys alone
    want = want[:n - last] + sorted(want[n - last:], key=lambda y: (-min(y[2] + tile, y[1]), y[0]))
    assert [tuple(x) for x in work[:n].tolist()] == want


def test_plan_refusals(lib):
    arr = (C.c_int32 * 2)(5, -1)
    assert lib.orc_attn_plan(arr, 2, None, 0) == -1 and b'negative length' in lib.orc_last_error()
    assert lib.orc_attn_plan(None, 1, None, 0) == -1
    big = (C.c_int32 * 2)(0x7fffffff, 1)
    assert lib.orc_attn_plan(big, 2, None, 0) == -1
    out = np.zeros((1, 4), dtype=np.int32)
    two = (C.c_int32 * 2)(5, 5)
    assert lib.orc_attn_plan(two, 2, out.ctypes.data, 1) == -1 and b'capacity' in lib.orc_last_error()
    with pytest.raises(ValueError):
        PackedPlan([3, -1], device='cpu')
    with pytest.raises(ValueError):
        PackedPlan([0x7fffffff, 1], device='cpu')


PACKED_OK = dict(st=[1024, 128] * 4, n_work=1, total=4, hq=8, hkv=8, hd=128, dtype=0, scale=0.1, ptr=4096)


@pytest.mark.parametrize('change, text', [
    (dict(hq=9), b'multiple'), (dict(hkv=0), b'multiple'), (dict(hd=96), b'head_dim'), (dict(dtype=2), b'dtype'),
    (dict(scale=0.0), b'scale'), (dict(scale=float('nan')), b'scale'), (dict(scale=-1.0), b'scale'), (dict(scale=float('inf')), b'scale'),
    (dict(st=[1020] + [1024] * 7), b'strides'), (dict(st=[-8] + [1024] * 7), b'strides'), (dict(ptr=0), b'null'), (dict(ptr=4104), b'aligned'),
    (dict(n_work=-1), b'bad'), (dict(n_work=1 << 30), b'too many'), (dict(n_work=1 << 21), b'too many')])
def test_packed_attention_refusals_of_the_c_entry(lib, change, text):
    a = dict(PACKED_OK, **change)
    st = (C.c_int64 * 8)(*a['st'])
    p = a['ptr']
    rc = lib.orc_attention_packed(p, p, p, p, st, p, a['n_work'], a['total'], a['hq'], a['hkv'], a['hd'], a['dtype'], a['scale'], None)
    assert rc == -1 and text in lib.orc_last_error()


CACHE_OK = dict(kv=4096, table=4096, lens=4096, refs=4096, status=4096, work=4096, n_layers=2, n_pages=4, n_kv_heads=2, page_size=16, head_dim=64,
                max_rows=4, max_row_pages=4, dtype=0)


def cache(**change):
    return _lib.OrcKvPages(*[dict(CACHE_OK, **change)[n] for n, _ in _lib.OrcKvPages._fields_])


@pytest.mark.parametrize('change, text', [
    (dict(kv=0), b'null'), (dict(table=0), b'null'), (dict(lens=0), b'null'), (dict(refs=0), b'null'), (dict(status=0), b'null'), (dict(work=0), b'null'),
    (dict(n_layers=0), b'geometry'), (dict(n_pages=0), b'geometry'), (dict(n_kv_heads=0), b'geometry'), (dict(max_row_pages=0), b'geometry'),
    (dict(max_rows=0), b'rows'), (dict(max_rows=65537), b'rows'), (dict(page_size=24), b'page_size'), (dict(head_dim=32), b'head_dim'),
    (dict(dtype=3), b'dtype'), (dict(n_pages=1 << 28), b'2^31'), (dict(max_row_pages=(1 << 20) + 1), b'2^20'), (dict(kv=4104), b'aligned')])
def test_cache_refusals_of_the_c_entries(lib, change, text):
    c = cache(**change)
    st = (C.c_int64 * 4)(128, 64, 128, 64)
    calls = [lambda: lib.orc_kv_reserve(C.byref(c), 4096, None, 1, 4096, 1, None), lambda: lib.orc_kv_append(C.byref(c), 0, 4096, 1, 4096, 4096, st, None),
             lambda: lib.orc_kv_fork(C.byref(c), 4096, 4096, 1, -1, 1, None), lambda: lib.orc_kv_free(C.byref(c), 4096, 1, None),
             lambda: lib.orc_kv_compact(C.byref(c), None, None), lambda: lib.orc_kv_compact(C.byref(cache()), C.byref(c), None)]
    for call in calls:
        assert call() == -1 and text in lib.orc_last_error()


def test_call_refusals_of_the_c_entries(lib):
    c, st = C.byref(cache()), (C.c_int64 * 4)(128, 64, 128, 64)

    def refused(rc, text):
        assert rc == -1 and text in lib.orc_last_error(), lib.orc_last_error()

    refused(lib.orc_kv_reserve(c, 4096, None, 1025, 4096, 1, None), b'1024')
    refused(lib.orc_kv_reserve(c, 4096, None, 1, 4096, -1, None), b'2^20')
    refused(lib.orc_kv_reserve(c, 4096, None, 1, 4096, (1 << 20) + 1, None), b'2^20')
    refused(lib.orc_kv_reserve(c, None, None, 1, 4096, 1, None), b'null')
    refused(lib.orc_kv_reserve(c, 4096, None, 1, None, 1, None), b'null')
    refused(lib.orc_kv_append(c, 2, 4096, 1, 4096, 4096, st, None), b'layer')
    refused(lib.orc_kv_append(c, 0, 4096, -1, 4096, 4096, st, None), b'bad')
    refused(lib.orc_kv_append(c, 0, 4096, 1, 4104, 4096, st, None), b'aligned')
    refused(lib.orc_kv_append(c, 0, 4096, 1, 4096, 4096, (C.c_int64 * 4)(100, 64, 128, 64), None), b'strides')
    refused(lib.orc_kv_append(c, 0, None, 1, 4096, 4096, st, None), b'null')
    refused(lib.orc_kv_fork(c, 4096, 4096, 1025, -1, 1, None), b'1024')
    refused(lib.orc_kv_fork(c, None, 4096, 1, -1, 1, None), b'null')
    refused(lib.orc_kv_free(c, 4096, -1, None), b'1024')
    refused(lib.orc_kv_compact(c, c, None), b'share memory')
    refused(lib.orc_kv_compact(c, C.byref(cache(kv=8192, table=1 << 21, lens=1 << 22, refs=1 << 23)), None), b'share memory')   # the pool is 64 KiB
    refused(lib.orc_kv_compact(c, C.byref(cache(kv=1 << 20, table=1 << 21, lens=1 << 22, refs=1 << 23, page_size=32)), None), b'differ')

    def attend(**change):
        x = dict(dict(layer=0, q=4096, out=4096, st=st, rows=4096, limits=None, n=1, hq=2, prefix=0, scale=0.1, ws=4096, stream=None), **change)
        return lib.orc_kv_attend(c, *x.values())

    refused(attend(layer=2), b'layer')
    refused(attend(layer=-1), b'layer')
    refused(attend(hq=3), b'multiple')
    refused(attend(hq=0), b'multiple')
    refused(attend(n=1025), b'1024')
    refused(attend(prefix=8), b'prefix')
    refused(attend(prefix=80), b'prefix')
    refused(attend(prefix=-16), b'prefix')
    refused(attend(scale=0.0), b'scale')
    refused(attend(q=None), b'null')
    refused(attend(rows=None), b'null')
    refused(attend(out=4100), b'aligned')
    refused(attend(st=(C.c_int64 * 4)(128, 64, 128, 4)), b'strides')
    refused(attend(prefix=16, ws=None), b'null')
    assert lib.orc_kv_attend_ws(c, 1, 3, 0) == -1 and lib.orc_kv_attend_ws(c, 4, 2, 16) > 0


def test_python_entries_refuse_what_is_not_on_a_gpu():
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    plan = PackedPlan.__new__(PackedPlan)
    plan.total, plan.work = 4, torch.zeros(1, 4, dtype=torch.int32)
    with pytest.raises(ValueError, match='CUDA'):
        packed_attention(x, x, x, plan)
    with pytest.raises(ValueError, match='CUDA'):
        KvPages.wrap(torch.zeros(1, 2, 4, 2, 16, 64, dtype=torch.bfloat16), torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32),
                     torch.zeros(4, dtype=torch.int32))
    for bad in (dict(n_pages=0), dict(page_size=24), dict(head_dim=96), dict(dtype=torch.float32)):
        with pytest.raises(ValueError):
            KvPages(**dict(dict(n_layers=1, n_pages=4, n_kv_heads=2, head_dim=64, page_size=16, device='cpu'), **bad))
