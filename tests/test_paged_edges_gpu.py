"""GPU: calls of packed_attention and KvPages at the edges of what they allow. The oracle and its tolerance are test_paged_gpu's."""
import pytest
import torch

from oracle_amd._lib import OracleHipError
from oracle_amd.paged import KvPages, PackedPlan, packed_attention
from test_paged_gpu import attention64, close, filled, ints, packed64, qkv

pytestmark = pytest.mark.gpu
DEV = 'cuda'
BF, FP = torch.bfloat16, torch.float16


def cache(n, own, prefix=64, page=32, hkv=2, hd=64, dtype=FP, seed=1):
    c, dense = filled(n, prefix, own, page, hkv, hd, dtype, seed)
    return c, dense


# (2, 8, 2): 16 columns at a time; (12, 8, 2): two passes of them; (40, 8, 2): 128 at a time but for the queries that end early
@pytest.mark.parametrize('n, hq, hkv', [(1, 8, 2), (3, 8, 2), (6, 8, 2), (40, 8, 2)])
@pytest.mark.parametrize('hd, dtype', [(128, BF), (64, FP)])
def test_attend_odd_values_behind_a_query_are_not_seen(n, hq, hkv, hd, dtype):
    prefix = 640
    c, dense = filled(n, prefix, [i % 5 for i in range(n)], 64, hkv, hd, dtype, 60 + n)
    rows = ints(list(range(n)))
    limits = [(1, 64, 333, 639, 640, 1000, 0, -3, 500)[i % 9] for i in range(n)]
    q = torch.randn(n, hq, hd, device=DEV).to(dtype)
    for x, value in ((1, float('nan')), (1, float('inf')), (1, float('-inf')), (0, float('nan')), (0, float('inf'))):
        for token in (333, 600):
            c2 = KvPages.wrap(c.kv.clone(), c.table, c.lens, c.refs)
            c2.kv[1, x, int(c.table[0, token // 64]), :, token % 64, 7] = value
            out = c2.attend(1, q, rows, prefix_tokens=prefix, limits=ints(limits))
            c2.check()
            for i, (r, m) in enumerate(zip(range(n), limits)):
                m = min(m, dense[r][0].shape[1])
                if m <= 0:
                    assert (out[i] == 0).all()
                elif m <= token:
                    ref, tol = attention64(q[i], dense[r][0][:, :m], dense[r][1][:, :m], hd ** -0.5)
                    close(out[i], ref, tol, (x, value, token, i))
                elif x == 1:      # seen: only dim 7, and as it is
                    assert not torch.isfinite(out[i, :, 7]).any() and torch.isfinite(out[i, :, :7]).all() and torch.isfinite(out[i, :, 8:]).all()


def test_attend_into_its_own_queries():
    for n, prefix, own in ((3, 0, [5, 70, 0]), (3, 0, [700, 900, 31]), (3, 128, [5, 70, 0]), (20, 192, [9] * 20)):
        c, _ = cache(n, own, prefix=prefix, page=64)
        q = torch.randn(n, 8, 64, device=DEV).to(FP)
        rows = ints(list(range(n)))
        want = c.attend(1, q, rows, prefix_tokens=prefix)
        assert c.attend(1, q, rows, prefix_tokens=prefix, out=q) is q
        assert torch.equal(q, want)


def test_calls_of_nothing():
    none = ints([])
    q = torch.zeros(0, 4, 64, dtype=BF, device=DEV)
    k = torch.zeros(0, 2, 64, dtype=BF, device=DEV)
    for lens in ([], [0], [0, 0, 0]):
        assert packed_attention(q, k, k, PackedPlan(lens)).shape == (0, 4, 64)
    some = torch.ones(5, 4, 64, dtype=BF, device=DEV)
    assert (packed_attention(some, some[:, :2], some[:, :2], PackedPlan([0])) == 0).all()
    c = KvPages(1, 4, 2, 64, page_size=16, max_rows=3, max_row_pages=2)
    before = [x.clone() for x in (c.kv, c.table, c.lens, c.refs)]
    assert c.reserve(none).numel() == 0
    assert (c.reserve(none, none, total=3) == -1).all()
    assert c.reserve(ints([0, 2]), ints([0, 0]), total=0).numel() == 0
    c.append(0, none, k, k)
    c.fork(none, none), c.copy(none, none), c.free(none)
    c.fork(ints([0]), ints([1])), c.free(ints([1, 2])), c.compact()          # rows without tokens
    assert c.attend(0, q, none).shape == (0, 4, 64)
    assert (c.attend(0, some, ints([0, 1, 2, 1, 0])) == 0).all()
    c.check()
    assert all(torch.equal(x, y) for x, y in zip(before, (c.kv, c.table, c.lens, c.refs)))


def test_calls_of_1024_rows():
    rows, page = 1024, 16
    c = KvPages(1, 1200, 1, 64, page_size=page, max_rows=rows + 3, max_row_pages=4)
    src = rows + 1
    slots = c.reserve(ints([src]), ints([37]), total=37)
    k, v = (torch.randn(37, 1, 64, device=DEV).to(BF) for _ in range(2))
    c.append(0, slots, k, v)
    every = torch.randperm(rows, device=DEV).int()
    c.fork(torch.full((rows,), src, dtype=torch.int32, device=DEV), every)
    slots = c.reserve(every)
    k1, v1 = (torch.randn(rows, 1, 64, device=DEV).to(BF) for _ in range(2))
    c.append(0, slots, k1, v1)
    q = torch.randn(rows, 2, 64, device=DEV).to(BF)
    out, apart = c.attend(0, q, every, prefix_tokens=32), c.attend(0, q, every)
    c.check()
    assert int(c.refs.max()) == rows + 1 and int((c.refs > 0).sum()) == 3 + rows
    for i in range(0, rows, 41):
        kk, vv = torch.cat([k, k1[i:i + 1]]).transpose(0, 1), torch.cat([v, v1[i:i + 1]]).transpose(0, 1)
        ref, tol = attention64(q[i], kk, vv, 0.125)
        close(out[i], ref, tol, i)
        close(apart[i], ref, tol, i)
    c.free(every)
    c.check()
    assert int((c.refs > 0).sum()) == 3 and (c.lens[:rows] == 0).all() and (c.table[:rows] == -1).all()
    many = torch.zeros(rows + 1, dtype=torch.int32, device=DEV)
    for bad in (lambda: c.reserve(many), lambda: c.free(many), lambda: c.fork(many, many), lambda: c.attend(0, torch.zeros(rows + 1, 2, 64, dtype=BF, device=DEV), many)):
        with pytest.raises(ValueError, match='1024'):
            bad()


# tokens of 16-token pages over a prefix: within one part's list of pages, over several lists, and beyond what 128 columns at a time reach
@pytest.mark.parametrize('prefix', [32720, 150_000, 16 * (40 * 2044 + 3)])
@pytest.mark.parametrize('n', [1, 5])
def test_attend_long_prefix_of_small_pages(prefix, n):
    hq, hkv, hd, page = 8, 1, 64, 16
    prefix -= prefix % page
    pages = prefix // page
    kv = torch.empty(1, 2, pages + n, hkv, page, hd, dtype=FP, device=DEV).normal_()
    order = torch.randperm(pages + n, device=DEV).int()
    table = torch.full((n, pages + 1), -1, dtype=torch.int32, device=DEV)
    table[:, :pages] = order[:pages]
    table[:, pages] = order[pages:]
    lens = ints([prefix + 1 + i for i in range(n)])
    refs = torch.ones(pages + n, dtype=torch.int32, device=DEV)
    c = KvPages.wrap(kv, table, lens, refs)
    q = torch.randn(n, hq, hd, device=DEV).to(FP)
    out = c.attend(0, q, ints(list(range(n))), prefix_tokens=prefix)
    apart = c.attend(0, q, ints(list(range(n))))
    c.check()
    for i in range(n):
        mine = table[i].long()
        dense = [kv[0, x][mine].transpose(0, 1).flatten(1, 2)[:, :prefix + 1 + i] for x in (0, 1)]
        ref, tol = attention64(q[i], *dense, hd ** -0.5)
        close(out[i], ref, tol, i)
        close(apart[i], ref, tol, (i, 'apart'))


def test_a_pool_beyond_32_bits_of_bytes():
    hkv, page, hd, n_pages = 8, 128, 128, 17000                # 4.5 GB of K, as much of V
    c = KvPages(1, n_pages, hkv, hd, page_size=page, max_rows=4, max_row_pages=4)
    c.refs[:n_pages - 12] = 1                                  # the first row gets pages at the end
    lens = [300, 129]
    q, k, v = qkv(sum(lens), 16, hkv, hd, BF, 70)
    slots = c.reserve(ints([2, 0]), ints(lens), total=sum(lens))
    c.append(0, slots, k, v)
    c.refs[:n_pages - 12] = 0
    c.fork(ints([2]), ints([1]))
    c.copy(ints([0]), ints([3]))
    c.check()
    assert int(c.table[2].max()) >= n_pages - 12

    def look(c):
        out = c.attend(0, q[:4], ints([2, 0, 1, 3]))
        for i, (a, b) in enumerate(((0, 300), (300, 429), (0, 300), (300, 429))):
            ref, tol = attention64(q[i], k[a:b].transpose(0, 1), v[a:b].transpose(0, 1), hd ** -0.5)
            close(out[i], ref, tol, i)
        shared = c.attend(0, q[:2], ints([1, 2]), prefix_tokens=256)
        for i in range(2):
            ref, tol = attention64(q[i], k[:300].transpose(0, 1), v[:300].transpose(0, 1), hd ** -0.5)
            close(shared[i], ref, tol, i)
    look(c)
    other = KvPages(1, 16, hkv, hd, page_size=page, max_rows=4, max_row_pages=4)
    c.compact(other)
    look(other)
    c.compact()
    c.check(), other.check()
    assert int(c.table.max()) < 12
    look(c)


def test_strides_near_the_limit():
    ts, n = 1 << 23, 100                                       # 1.7 GB for 100 tokens
    room = torch.zeros(ts * n, dtype=BF, device=DEV)
    k, v = room.as_strided((n, 2, 64), (ts, 64, 1)), room.as_strided((n, 2, 64), (ts, 64, 1), 4096)
    q, k1, v1 = qkv(n, 4, 2, 64, BF, 71)
    k.copy_(k1), v.copy_(v1)
    assert torch.equal(packed_attention(q, k, v, PackedPlan([n])), packed_attention(q, k1, v1, PackedPlan([n])))
    c = KvPages(1, 8, 2, 64, page_size=16, max_rows=1, max_row_pages=8)
    slots = c.reserve(ints([0]), ints([n]), total=n)
    c.append(0, slots, k, v)
    ref, tol = attention64(q[0], k1.transpose(0, 1), v1.transpose(0, 1), 0.125)
    close(c.attend(0, q[:1], ints([0]))[0], ref, tol, 'append')


def test_many_short_prompts():
    lens = [i % 4 for i in range(3001)]
    q, k, v = qkv(sum(lens), 2, 1, 64, FP, 72)
    ref, tol = packed64(q, k, v, lens, 0.125)
    close(packed_attention(q, k, v, PackedPlan(lens)), ref, tol, 'short')


def test_calls_on_two_streams_at_once():
    c, _ = cache(20, [i for i in range(20)], prefix=640, page=64, seed=3)
    rows = ints(list(range(20)))
    lens = [700, 64, 333]
    q, k, v = qkv(sum(lens), 8, 2, 64, FP, 73)
    plan = PackedPlan(lens)
    q1, q2 = q[:20], q[20:40]
    want = [c.attend(1, q1, rows, prefix_tokens=640), c.attend(1, q2, rows, prefix_tokens=640), packed_attention(q, k, v, plan)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = [[], [], []]
    for _ in range(8):
        for s, g, call in zip(streams, got, (lambda: c.attend(1, q1, rows, prefix_tokens=640), lambda: c.attend(1, q2, rows, prefix_tokens=640),
                                             lambda: packed_attention(q, k, v, plan))):
            with torch.cuda.stream(s):
                g.append(call())
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(x, w) for x in g)


def test_a_question_from_fork_to_free_in_a_graph():
    """Two graphs of one cache, replayed in turn: fork a frame to questions, a token each, its attention, the rows given back, the pool compacted."""
    def make():
        c, _ = filled(2, 64, [21, 40], 32, 2, 64, FP, 18, extra=12)
        kv = torch.nan_to_num(c.kv)
        table, lens = torch.full((6, c.table.shape[1]), -1, dtype=torch.int32, device=DEV), torch.zeros(6, dtype=torch.int32, device=DEV)
        table[:2], lens[:2] = c.table, c.lens
        return KvPages.wrap(kv, table, lens, c.refs)
    c, d = make(), make()
    k, v = (torch.randn(3, 2, 64, device=DEV).to(FP) for _ in range(2))
    q = torch.randn(3, 4, 64, device=DEV).to(FP)
    dst = ints([4, 2, 5])

    def ask(x, src):
        x.fork(src, dst)
        slots = x.reserve(dst)
        x.append(1, slots, k, v)
        out = x.attend(1, q, dst, prefix_tokens=64)
        x.free(dst)
        x.compact()
        return out
    sources, graphs, outs = (ints([0, 0, 0]), ints([1, 0, 1])), [], []
    side = torch.cuda.Stream()
    for src in sources:
        g = torch.cuda.CUDAGraph()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(g, stream=side):
            outs.append(ask(c, src))
        graphs.append(g)
    for i in range(6):
        k.normal_(), v.normal_(), q.normal_()
        want = ask(d, sources[i % 2])
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[i % 2], want), i
        assert torch.equal(c.table, d.table) and torch.equal(c.lens, d.lens) and torch.equal(c.refs, d.refs) and torch.equal(c.kv, d.kv), i
    c.check(), d.check()


def test_compact_into_a_pool_that_is_too_small_or_the_same():
    c, _ = cache(3, [40, 9, 70], seed=5)
    c = KvPages.wrap(torch.nan_to_num(c.kv), c.table, c.lens, c.refs)
    live = int((c.refs > 0).sum())
    like = lambda pages: KvPages(2, pages, 2, 64, page_size=32, max_rows=3, max_row_pages=c.table.shape[1], dtype=FP)      # noqa: E731
    small, fits = like(live - 1), like(live)
    c.compact(small)
    c.check()
    with pytest.raises(OracleHipError, match='free pages'):
        small.check()
    assert (small.table == -1).all() and (small.lens == 0).all() and (small.refs == 0).all() and (small.kv == 0).all()
    c.compact(fits)
    c.check(), fits.check()
    assert (fits.refs > 0).all() and torch.equal(fits.lens, c.lens)
    with pytest.raises(OracleHipError, match='share memory'):
        c.compact(c)
    part = KvPages.wrap(c.kv.view(-1)[:c.kv.numel() // 2].view(1, *c.kv.shape[1:]), c.table.clone(), c.lens.clone(), c.refs.clone())
    whole = KvPages.wrap(c.kv.view(-1)[c.kv.numel() // 4:3 * (c.kv.numel() // 4)].view(1, *c.kv.shape[1:]), c.table.clone(), c.lens.clone(), c.refs.clone())
    with pytest.raises(OracleHipError, match='share memory'):
        part.compact(whole)


def test_tensors_that_want_gradients_are_refused():
    c, _ = cache(2, [3, 4])
    q, k, v = qkv(16, 4, 2, 64, FP, 6)
    plan, rows = PackedPlan([16]), ints([0, 1])
    want = packed_attention(q, k, v, plan)
    for i in range(3):
        x = [q, k, v]
        x[i] = x[i].clone().requires_grad_()
        with pytest.raises(ValueError, match='gradient'):
            packed_attention(*x, plan)
        with torch.no_grad():
            assert torch.equal(packed_attention(*x, plan), want)
    leaf = q[:2].clone().requires_grad_()
    with pytest.raises(ValueError, match='gradient'):
        c.attend(1, leaf, rows)
    c.attend(1, leaf.detach(), rows)
    with pytest.raises(ValueError, match='gradient'):
        c.append(1, c.reserve(rows), k[:2].clone().requires_grad_(), v[:2])
