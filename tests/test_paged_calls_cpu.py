"""CPU: calls of the packed attention and of the paged cache that the C entries have to tell apart before anything is launched."""
import ctypes as C
import os
import random

import pytest
import torch

import __graft_entry__
from oracle_amd import _lib

# What is not refused would be launched with addresses of no tensor: only where there is no GPU to launch it on.
pytestmark = pytest.mark.skipif(torch.cuda.device_count() > 0, reason='made-up addresses')
FAR = (1 << 40, 2 << 40, 3 << 40)


@pytest.fixture(scope='module')
def lib():
    if not os.path.exists(_lib.LIB_PATH):
        __graft_entry__.build()
    return _lib.lib()


def packed(lib, views, total, hq, hkv, hd):
    """views: (address, token stride, head stride) of q, k, v, out; what the call was refused for, None where it came to the launch"""
    st = (C.c_int64 * 8)(*[x for _, ts, hs in views for x in (ts, hs)])
    rc = lib.orc_attention_packed(*[p for p, _, _ in views], st, 4096, 1, total, hq, hkv, hd, 0, 0.1, None)
    assert rc == -1
    text = lib.orc_last_error().decode()
    return text if 'lies over' in text else None


def elements(p, ts, hs, tokens, heads, hd):
    return {p // 2 + t * ts + h * hs + d for t in range(tokens) for h in range(heads) for d in range(hd)}


def span(x):
    return min(x), max(x)


@pytest.mark.parametrize('seed', range(6))
def test_out_over_k_v_or_q_is_refused_and_slices_of_a_projection_are_not(lib, seed):
    r = random.Random(seed)
    hd, seen = 64, set()
    for _ in range(400):
        hkv, group, tokens = r.choice((1, 2, 3)), r.choice((1, 2)), r.choice((1, 2, 5))
        hq = hkv * group
        strides = lambda heads: r.choice(((heads * hd, hd), (3 * heads * hd, hd), (3 * heads * hd, 3 * hd), (hd, tokens * hd), (r.choice((8, 64, 96, 640)), r.choice((0, 8, 64, 72)))))    # noqa: E731
        a, b = strides(hq), strides(hkv)
        if r.random() < 0.6:
            b = a
        base, which = 1 << 20, r.choice(('q', 'k', 'v'))
        heads = hq if which == 'q' else hkv
        other = (base + 16 * r.randrange(-60, 90), *b)
        if other[0] == base and which == 'q':
            continue                                     # q itself: below
        views = [(FAR[i], heads_ * hd, hd) for i, heads_ in enumerate((hq, hkv, hkv))] + [(base, *a)]
        views['qkv'.index(which)] = other
        x, y = elements(base, *a, tokens, hq, hd), elements(*other, tokens, heads, hd)
        got = packed(lib, views, tokens, hq, hkv, hd)
        if x & y:
            seen.add('meet')
            assert got is not None and ('k or v' in got) == (which != 'q'), (views, which)
        elif a[0] == b[0] or tokens == 1 or span(x)[1] < span(y)[0] or span(y)[1] < span(x)[0]:
            seen.add('apart')
            assert got is None, (views, which, got)
    assert seen == {'meet', 'apart'}


def test_out_may_be_q_or_beside_it(lib):
    hq, hkv, hd, total = 8, 2, 128, 100
    row = (hq + 2 * hkv) * hd
    base = 1 << 20
    q, k, v = (base, row, hd), (base + 2 * hq * hd, row, hd), (base + 2 * (hq + hkv) * hd, row, hd)      # a fused projection's rows
    apart = (FAR[0], hq * hd, hd)
    assert packed(lib, [q, k, v, apart], total, hq, hkv, hd) is None
    assert packed(lib, [q, k, v, q], total, hq, hkv, hd) is None                                         # in place
    assert 'over q' in packed(lib, [q, k, v, (base - 2 * row, row, hd)], total, hq, hkv, hd)               # a row further
    assert 'over q' in packed(lib, [q, (FAR[1], 256, hd), (FAR[2], 256, hd), (base, hq * hd, hd)], total, hq, hkv, hd)   # its start, other strides
    assert 'k or v' in packed(lib, [apart, k, v, (base + 2 * 128, row, hd)], total, hq, hkv, hd)           # its last head is k's first
    assert 'k or v' in packed(lib, [apart, (FAR[1], 256, hd), (base, hq * hd, hd), (base, hq * hd, hd)], total, hq, hkv, hd)


def test_attend_refuses_an_out_over_its_queries_or_the_pool(lib):
    fields = dict(kv=1 << 30, table=4096, lens=4096, refs=4096, status=4096, work=4096, n_layers=2, n_pages=4, n_kv_heads=2, page_size=16, head_dim=64,
                  max_rows=4, max_row_pages=4, dtype=0)
    c = _lib.OrcKvPages(*[fields[n] for n, _ in _lib.OrcKvPages._fields_])
    pool = 2 * 2 * 4 * 2 * 16 * 64 * 2

    def attend(q, out, n=3, ts=512, out_ts=512):
        assert lib.orc_kv_attend(C.byref(c), 0, q, out, (C.c_int64 * 4)(ts, 64, out_ts, 64), 4096, None, n, 8, 0, 0.1, 4096, None) == -1
        text = lib.orc_last_error().decode()
        return text if 'lies over' in text else None

    q = 1 << 20
    assert attend(q, q) is None and attend(q, q + 3 * 1024) is None and attend(q, q - 3 * 1024) is None
    assert attend(q, q, n=1, out_ts=1024) is None                        # one query: its stride does not matter
    assert 'over q' in attend(q, q + 1024) and 'over q' in attend(q, q + 128) and 'over q' in attend(q, q, out_ts=1024)
    assert attend(q, (1 << 30) + pool) is None and attend(q, (1 << 30) - 3 * 1024) is None
    assert 'pool' in attend(q, (1 << 30) + pool - 1024) and 'pool' in attend(q, (1 << 30) - 3 * 1024 + 16)


# items of the prefix (wide columns and 16 at a time), of the rows' own tokens, and the waves that join
@pytest.mark.parametrize('hkv, hq, n, prefix', [(16384, 16384, 1024, 0), (16384, 16384, 1024, 64), (1, 1 << 17, 1024, 0), (1, 60000, 1024, 16 * 40 * 2044), (131072, 131072, 200, 64)])
def test_attend_refuses_what_no_launch_can_hold(lib, hkv, hq, n, prefix):
    fields = dict(kv=1 << 40, table=4096, lens=4096, refs=4096, status=4096, work=4096, n_layers=1, n_pages=4, n_kv_heads=hkv, page_size=16, head_dim=64,
                  max_rows=4, max_row_pages=1 << 20, dtype=0)
    c = _lib.OrcKvPages(*[fields[x] for x, _ in _lib.OrcKvPages._fields_])
    assert lib.orc_kv_attend_ws(C.byref(c), n, hq, prefix) == -1 and b'too many' in lib.orc_last_error()
    st = (C.c_int64 * 4)(hq * 64, 64, hq * 64, 64)
    assert lib.orc_kv_attend(C.byref(c), 0, 4096, 4096, st, 4096, None, n, hq, prefix, 0.1, 4096, None) == -1
    assert b'too many' in lib.orc_last_error()
    assert lib.orc_kv_attend_ws(C.byref(c), 1, hkv, 0) >= 0


# parts of the prefix whose tiles do not divide by their number: none of them is empty
@pytest.mark.parametrize('prefix, hkv, hq, n, parts', [
    (201 * 64, 1, 8, 40, 34 + 13),           # 128 columns at a time, 201 tiles: 34 parts of 6 (not 40, 6 of them empty), and 13 of own tokens
    (41 * 64, 1, 8, 40, 11 + 13),            # 41: 11 of 4
    (200 * 64, 2, 8, 40, 40 + 7),            # 40 of 5
    (16 * 256 + 32, 1, 2, 2, 17 + 16)])      # 16 columns at a time, tiles of 32 keys: 129 in 17 of 8
def test_no_part_of_a_prefix_is_empty(lib, prefix, hkv, hq, n, parts):
    fields = dict(kv=1 << 40, table=4096, lens=4096, refs=4096, status=4096, work=4096, n_layers=1, n_pages=4, n_kv_heads=hkv, page_size=32, head_dim=64,
                  max_rows=4, max_row_pages=4096, dtype=0)
    c = _lib.OrcKvPages(*[fields[x] for x, _ in _lib.OrcKvPages._fields_])
    assert lib.orc_kv_attend_ws(C.byref(c), n, hq, prefix) == n * hq * parts * (64 + 2) * 4
