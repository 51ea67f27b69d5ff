"""GPU: attention over packed prompts and the paged KV cache against plain implementations in 64 bits.

Tolerance of an attention output, derived before the first run. With eps/2 the half step of the 16-bit type, A = sum_j w_j |v_j| for the
softmax weights w: the output is rounded once (eps/2 |out|); the weights are rounded to 16 bits before the product with V, each by eps/2 of itself
(eps/2 A) while their sum is not; scores are fp32 sums of hd exact products (error <= hd 2^-24 sum|q k| <= hd 2^-24 S, S the largest such
sum over the row's keys) and go through exp with 2^-21 of their own: a weight is off by that relative amount, twice (numerator and sum); the output sum
runs over n keys in fp32 (n 2^-24 A)."""
import pytest
import torch

from oracle_amd._lib import OracleHipError
from oracle_amd.paged import KvPages, PackedPlan, packed_attention

pytestmark = pytest.mark.gpu
DEV = 'cuda'
BF, FP = torch.bfloat16, torch.float16


def attention64(q, k, v, scale):
    """q (Hq, hd) of one token, k / v (Hkv, n, hd): -> (out, tolerance without the output's own rounding), both (Hq, hd)"""
    hq, hd = q.shape
    hkv, n, _ = k.shape
    eps2 = torch.finfo(q.dtype).eps / 2
    q, k, v = q.double(), k.double(), v.double()
    k, v = k.repeat_interleave(hq // hkv, 0), v.repeat_interleave(hq // hkv, 0)
    w = torch.softmax((k * q[:, None]).sum(-1) * scale, -1)
    size = ((k * q[:, None]).abs().sum(-1) * scale).amax(-1, keepdim=True)
    out, mag = (w[..., None] * v).sum(1), (w[..., None] * v.abs()).sum(1)
    return out, mag * (eps2 + 2 * (hd * size * 2.0 ** -24 + 2.0 ** -20) + n * 2.0 ** -24)


def close(got, ref, tol, what):
    eps2 = torch.finfo(got.dtype).eps / 2
    err = (got.double() - ref).abs()
    bound = tol + eps2 * (ref.abs() + tol) + 1e-7      # 1e-7: below the least normal fp16 step
    assert torch.isfinite(got).all(), what
    worst = float((err / bound).max())
    assert worst <= 1.0, (what, worst)


def packed64(q, k, v, lens, scale):
    out, tol = torch.zeros(q.shape, dtype=torch.float64, device=q.device), torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    hq, hd = q.shape[1:]
    g, eps2, at = hq // k.shape[1], torch.finfo(q.dtype).eps / 2, 0
    for n in lens:
        qs, ks, vs = (x[at:at + n].double().transpose(0, 1).contiguous() for x in (q, k, v))
        ks, vs = ks.repeat_interleave(g, 0), vs.repeat_interleave(g, 0)
        seen = torch.ones(n, n, dtype=torch.bool, device=q.device).tril()
        kt = ks.transpose(1, 2).contiguous()
        w = torch.softmax((qs @ kt * scale).masked_fill(~seen, float('-inf')), -1)
        size = (qs.abs() @ kt.abs() * scale).masked_fill(~seen, 0).amax(-1, keepdim=True) if n else 0
        out[at:at + n] = (w @ vs).transpose(0, 1)
        tol[at:at + n] = ((w @ vs.abs()) * (eps2 + 2 * (hd * size * 2.0 ** -24 + 2.0 ** -20) + n * 2.0 ** -24)).transpose(0, 1)
        at += n
    return out, tol


def qkv(total, hq, hkv, hd, dtype, seed, qscale=2.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(total, hq + 2 * hkv, hd, generator=g, device=DEV).to(dtype)
    x[:, :hq] *= qscale
    return x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]


# ---------------------------------------------------------------------------------------------- packed prompts
@pytest.mark.parametrize('lens', [[1], [0, 2, 0], [63, 64, 65, 1], [127, 0, 128, 129], [255, 257, 31, 33, 32], [700, 5], [1025]], ids=str)
@pytest.mark.parametrize('hq, hkv, hd, dtype', [(4, 4, 128, BF), (8, 2, 64, FP), (6, 1, 128, FP), (16, 8, 64, BF)])
def test_packed_attention(lens, hq, hkv, hd, dtype):
    q, k, v = qkv(sum(lens), hq, hkv, hd, dtype, 1)
    out = packed_attention(q, k, v, PackedPlan(lens))
    ref, tol = packed64(q, k, v, lens, hd ** -0.5)
    close(out, ref, tol, lens)


def test_packed_attention_long_prompts():
    lens = [4200, 3900, 77]
    for hd, dtype in ((128, BF), (64, FP)):
        q, k, v = qkv(sum(lens), 16, 2, hd, dtype, 2)
        out = packed_attention(q, k, v, PackedPlan(lens), scale=0.11)
        at = 0
        for n in lens:      # every 53rd token of every prompt
            for t in range(0, n, 53):
                ref, tol = attention64(q[at + t], k[at:at + t + 1].transpose(0, 1), v[at:at + t + 1].transpose(0, 1), 0.11)
                close(out[at + t], ref, tol, (n, t))
            at += n


def test_packed_attention_large_scores_and_peaked_rows():
    lens = [300, 41]
    q, k, v = qkv(sum(lens), 4, 4, 128, BF, 3, qscale=40.0)
    k[0] *= 30
    out = packed_attention(q, k, v, PackedPlan(lens))
    ref, tol = packed64(q, k, v, lens, 128 ** -0.5)
    close(out, ref, tol, 'peaked')


def test_packed_attention_rows_behind_and_neighbours_do_not_matter():
    lens = [70, 0, 130]
    q, k, v = qkv(sum(lens) + 9, 4, 2, 128, BF, 4)
    plan = PackedPlan(lens)
    clean = packed_attention(q, k, v, plan)
    assert (clean[200:] == 0).all()
    for poison in (float('nan'), float('inf'), float('-inf'), torch.finfo(BF).min):
        k2, v2, q2 = k.clone(), v.clone(), q.clone()
        for x in (k2, v2, q2):
            x[70:] = poison           # the second prompt and what lies behind
        out = torch.full(q.shape, 7.0, dtype=BF, device=DEV)
        assert packed_attention(q2, k2, v2, plan, out=out) is out
        assert torch.equal(out[:70], clean[:70]) and (out[200:] == 7).all()
        k2, v2 = k.clone(), v.clone()
        k2[:70], v2[:70] = poison, poison
        k2[200:], v2[200:] = poison, poison
        assert torch.equal(packed_attention(q, k2, v2, plan)[70:200], clean[70:200])


@pytest.mark.parametrize('hd, dtype', [(128, BF), (64, FP)])
def test_packed_attention_odd_values_reach_only_who_sees_them(hd, dtype):
    lens, at = [200, 333], 200
    q, k, v = qkv(sum(lens), 4, 2, hd, dtype, 40)
    plan = PackedPlan(lens)
    clean = packed_attention(q, k, v, plan)
    inf, nan = float('inf'), float('nan')
    for t, kh, d, value in ((0, 0, 3, inf), (63, 1, 0, nan), (64, 0, hd - 1, -inf), (131, 1, 40, inf), (332, 0, 7, nan), (300, 1, 33, -inf)):
        odd = v.clone()
        odd[at + t, kh, d] = value
        out = packed_attention(q, k, odd, plan)
        want = clean.clone()
        want[at + t:, 2 * kh:2 * kh + 2, d] = value
        seen = torch.zeros_like(want, dtype=torch.bool)
        seen[at + t:, 2 * kh:2 * kh + 2, d] = True
        assert torch.equal(out[seen].isnan(), want[seen].isnan()) and torch.equal(out[seen].nan_to_num(1, 2, 3), want[seen].nan_to_num(1, 2, 3)), (t, value)
        close(out[~seen], clean[~seen].double(), torch.finfo(dtype).eps * clean[~seen].double().abs() + 2.0 ** -12, (t, value))
    odd = v.clone()
    odd[at + 10, 0, 5], odd[at + 100, 0, 5] = inf, -inf
    out = packed_attention(q, k, odd, plan)
    assert (out[at + 10:at + 100, :2, 5] == inf).all() and out[at + 100:, :2, 5].isnan().all() and torch.isfinite(out[at:at + 10]).all()
    odd = k.clone()
    odd[at + 150, 1] = nan
    out = packed_attention(q, odd, v, plan)
    assert out[at + 150:, 2:].isnan().all() and torch.isfinite(out[:at + 150]).all() and torch.isfinite(out[:, :2]).all()


def test_packed_attention_layouts_stream_and_graph():
    lens = [90, 33]
    q, k, v = qkv(123, 8, 4, 64, FP, 5)
    plan = PackedPlan(lens)
    want = packed_attention(q, k, v, plan)
    heads_first = lambda x: x.transpose(0, 1).contiguous().transpose(0, 1)      # noqa: E731
    out = torch.empty(8, 123, 64, dtype=FP, device=DEV).transpose(0, 1)
    assert torch.equal(packed_attention(heads_first(q), heads_first(k), heads_first(v), plan, out=out), want)
    inplace = q.clone()
    assert torch.equal(packed_attention(inplace, k, v, plan, out=inplace), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = packed_attention(q, k, v, plan)
    side.synchronize()
    assert torch.equal(other, want)
    graph = torch.cuda.CUDAGraph()
    qs = q.clone()
    with torch.cuda.graph(graph):
        captured = packed_attention(qs, k, v, plan)
    for i in range(3):
        qs.copy_(q if i % 2 == 0 else q * 0.5)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, packed_attention(qs, k, v, plan))


def test_packed_attention_refusals():
    q, k, v = qkv(16, 4, 2, 64, BF, 6)
    plan = PackedPlan([16])
    for bad in ((q.float(), k, v), (q, k.to(FP), v), (q, k[:8], v), (q, k, v[:, :1]), (q[:, :3], k, v), (q[..., :32], k[..., :32], v[..., :32]),
                (q[:8], k[:8], v[:8]), (q[0], k, v), (q.cpu(), k, v), (q.transpose(1, 2).contiguous().transpose(1, 2), k, v)):
        with pytest.raises(ValueError):
            packed_attention(*bad, plan)
    flat = torch.zeros(16 * 4 * 64 + 8, dtype=BF, device=DEV)
    with pytest.raises(ValueError, match='16 bytes'):
        packed_attention(flat[4:4 + 4096].view(16, 4, 64), k, v, plan)
    with pytest.raises(ValueError, match='expanded'):
        packed_attention(q, k, v, plan, out=torch.zeros(1, 4, 64, dtype=BF, device=DEV).expand(16, 4, 64))
    for scale in (0.0, -1.0, float('nan'), float('inf')):
        with pytest.raises(ValueError):
            packed_attention(q, k, v, plan, scale=scale)
    with pytest.raises(ValueError, match='plan'):
        packed_attention(q, k, v, PackedPlan([16], device='cpu'))


# ---------------------------------------------------------------------------------------------- pages
class Model:
    """The cache on the host: lists, and the tokens as rows of (layers, 2, heads, hd)."""

    def __init__(self, c):
        self.ps, self.width = c.page_size, c.table.shape[1]
        self.table, self.lens, self.refs = c.table.tolist(), c.lens.tolist(), c.refs.tolist()
        self.kv = c.kv.clone()

    def take(self):
        p = self.refs.index(0)
        self.refs[p] = 1
        return p

    def reserve(self, rows, counts):
        slots = []
        for r, n in zip(rows, counts):
            for t in range(self.lens[r], self.lens[r] + n):
                if t % self.ps == 0:
                    self.table[r][t // self.ps] = self.take()
                slots.append(self.table[r][t // self.ps] * self.ps + t % self.ps)
            self.lens[r] += n
        return slots

    def append(self, layer, slots, k, v):
        for i, s in enumerate(slots):
            if s >= 0:
                self.kv[layer, 0, s // self.ps, :, s % self.ps] = k[i]
                self.kv[layer, 1, s // self.ps, :, s % self.ps] = v[i]

    def fork(self, src, dst, n_tokens=None, share=True):
        for s, d in zip(src, dst):
            n = self.lens[s] if n_tokens is None else min(n_tokens, self.lens[s])
            for j in range(-(-n // self.ps)):
                part = min(self.ps, n - j * self.ps)
                if share and part == self.ps:
                    self.table[d][j] = self.table[s][j]
                    self.refs[self.table[s][j]] += 1
                else:
                    self.table[d][j] = self.take()
                    self.kv[:, :, self.table[d][j], :, :part] = self.kv[:, :, self.table[s][j], :, :part]
            self.lens[d] = n

    def free(self, rows):
        for r in rows:
            for j, p in enumerate(self.table[r]):
                if p >= 0:
                    self.refs[p] -= 1
                self.table[r][j] = -1
            self.lens[r] = 0

    def compact(self):
        live = sum(x > 0 for x in self.refs)
        holes = [i for i in range(live) if self.refs[i] == 0]
        for s, d in zip([i for i in range(live, len(self.refs)) if self.refs[i] > 0], holes):
            self.kv[:, :, d] = self.kv[:, :, s]
            self.refs[d], self.refs[s] = self.refs[s], 0
            self.table = [[d if p == s else p for p in row] for row in self.table]

    def same(self, c, what):
        assert c.table.tolist() == self.table, what
        assert c.lens.tolist() == self.lens, what
        assert c.refs.tolist() == self.refs, what
        assert torch.equal(c.kv, self.kv), what


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def new_cache(page=16, hd=64, hkv=2, layers=2, n_pages=60, rows=9, width=12, dtype=BF, seed=0):
    c = KvPages(layers, n_pages, hkv, hd, page_size=page, max_rows=rows, max_row_pages=width, dtype=dtype)
    c.kv.copy_(torch.randn(c.kv.shape, generator=torch.Generator().manual_seed(seed)).to(dtype))     # what lies behind the last token of a page
    return c


@pytest.mark.parametrize('page, hd, dtype', [(16, 64, BF), (32, 128, FP), (128, 64, FP), (64, 128, BF)])
def test_pages_follow_the_model(page, hd, dtype):
    import random
    r = random.Random(page + hd)
    c = new_cache(page, hd, dtype=dtype)
    m = Model(c)
    tok = 0
    for step in range(60):
        empty, full = [i for i in range(9) if m.lens[i] == 0], [i for i in range(9) if m.lens[i] > 0]
        free = sum(x == 0 for x in m.refs)
        op = r.choice(('reserve', 'reserve', 'fork', 'copy', 'free', 'compact'))
        if op == 'reserve':
            rows = r.sample(range(9), r.randint(1, 9))
            counts = [min(r.choice((0, 1, page - 1, page, page + 1, 3 * page + 5)), 12 * page - m.lens[x]) for x in rows]
            if sum(x // page + 1 for x in counts) > free:
                continue
            one = all(x == 1 for x in counts)
            extra = r.choice((0, 3))
            slots = c.reserve(ints(rows), None if one and not extra else ints(counts), None if one and not extra else sum(counts) + extra)
            want = m.reserve(rows, counts)
            assert slots.tolist() == want + [-1] * (slots.numel() - len(want)), step
            g = torch.Generator(device=DEV).manual_seed(step)
            for layer in range(2):
                k, v = torch.randn(2, slots.numel(), 2, hd, generator=g, device=DEV).to(dtype).unbind(0)
                c.append(layer, slots, k, v)
                m.append(layer, slots.tolist(), k, v)
            tok += sum(counts)
        elif op in ('fork', 'copy') and empty and full:
            dst = r.sample(empty, r.randint(1, len(empty)))
            src = [r.choice(full) for _ in dst]
            n_tokens = r.choice((None, None, 0, 1, page, 2 * page + 3))
            need = sum(1 if op == 'fork' else -(-m.lens[s] // page) for s in src)
            if need > free:
                continue
            (c.fork if op == 'fork' else c.copy)(ints(src), ints(dst), n_tokens)
            m.fork(src, dst, n_tokens, op == 'fork')
        elif op == 'free' and full:
            rows = r.sample(range(9), r.randint(1, 4))
            c.free(ints(rows))
            m.free(rows)
        elif op == 'compact':
            c.compact()
            m.compact()
        c.check()
        m.same(c, (step, op))
    assert tok > 100


def test_refused_calls_change_nothing_and_say_why():
    c = new_cache(n_pages=8, rows=4, width=4)
    slots = c.reserve(ints([0, 1]), ints([40, 16]), total=56)
    c.append(0, slots, *torch.randn(2, 56, 2, 64, device=DEV).to(BF).unbind(0))
    c.check()
    m = Model(c)
    cases = [('outside', lambda: c.reserve(ints([0, 4]))), ('outside', lambda: c.reserve(ints([-1]))), ('twice', lambda: c.reserve(ints([1, 0, 1]))),
             ('count', lambda: c.reserve(ints([2, 3]), ints([5, 6]), total=10)), ('count', lambda: c.reserve(ints([2]), ints([-1]), total=10)),
             ('wide', lambda: c.reserve(ints([0]), ints([25]), total=25)), ('free pages', lambda: c.reserve(ints([2, 3]), ints([64, 64]), total=128)),
             ('outside', lambda: c.fork(ints([4]), ints([2]))), ('outside', lambda: c.fork(ints([0]), ints([-5]))), ('twice', lambda: c.fork(ints([0, 0]), ints([2, 2]))),
             ('twice', lambda: c.fork(ints([0, 2]), ints([2, 3]))), ('holds', lambda: c.fork(ints([0]), ints([1]))),
             ('free pages', lambda: c.copy(ints([0, 0]), ints([2, 3]))), ('outside', lambda: c.free(ints([0, 9]))), ('twice', lambda: c.free(ints([1, 1])))]
    for text, call in cases:
        got = call()
        with pytest.raises(OracleHipError, match=text):
            c.check()
        c.check()
        m.same(c, text)
        if got is not None:
            assert (got == -1).all()
            c.append(1, got, *torch.randn(2, got.numel(), 2, 64, device=DEV).to(BF).unbind(0))      # writes nothing
            m.same(c, text)
    c.append(0, ints([-1, 8 * 16, 2 ** 31 - 1]), *torch.ones(2, 3, 2, 64, device=DEV, dtype=BF).unbind(0))
    m.same(c, 'slots outside the pool')
    saved = c.table.clone()
    c.table[0, 0] = 8
    c.fork(ints([0]), ints([2]))
    with pytest.raises(OracleHipError, match='pool'):
        c.check()
    c.table.copy_(saved)
    m.same(c, 'a bad page')
    for bad in (lambda: c.reserve(torch.tensor([0], dtype=torch.int32)), lambda: c.reserve(torch.tensor([0], device=DEV)), lambda: c.reserve(ints([0]), ints([1])),
                lambda: c.reserve(ints([0]), ints([1, 2]), total=3), lambda: c.reserve(ints([0]), total=-1), lambda: c.reserve(ints([[0]])),
                lambda: c.reserve(ints(list(range(1025)))), lambda: c.fork(ints([0, 1]), ints([2])), lambda: c.fork(ints([0]), ints([2]), n_tokens=-2), lambda: c.fork(ints([0]), ints([2]), n_tokens=-1),
                lambda: c.append(2, ints([0]), *torch.zeros(2, 1, 2, 64, device=DEV, dtype=BF).unbind(0)),
                lambda: c.append(0, ints([0]), *torch.zeros(2, 2, 2, 64, device=DEV, dtype=BF).unbind(0)),
                lambda: c.append(0, ints([0]), *torch.zeros(2, 1, 2, 64, device=DEV, dtype=FP).unbind(0))):
        with pytest.raises(ValueError):
            bad()
    m.same(c, 'host refusals')


def test_compact_into_another_cache():
    c = new_cache(n_pages=40, rows=6)
    c.reserve(ints([0, 1, 2, 3]), ints([50, 0, 33, 100]), total=183)
    c.fork(ints([3, 0]), ints([4, 5]))
    c.free(ints([0, 3]))
    live = int((c.refs > 0).sum())
    before = Model(c)
    for size in (live, live + 5):
        d = new_cache(n_pages=size, rows=6, seed=9)
        old = d.kv.clone()
        c.compact(into=d)
        c.check(), d.check()
        before.same(c, 'the source')
        pages = [p for p, n in enumerate(before.refs) if n > 0]
        place = {p: i for i, p in enumerate(pages)}
        assert d.table.tolist() == [[place.get(p, -1) for p in row] for row in before.table] and d.lens.tolist() == before.lens
        assert d.refs.tolist() == [before.refs[p] for p in pages] + [0] * (size - live)
        assert torch.equal(d.kv[:, :, :live], c.kv[:, :, pages]) and torch.equal(d.kv[:, :, live:], old[:, :, live:])
    small = new_cache(n_pages=live - 1, rows=6, seed=9)
    m = Model(small)
    c.compact(into=small)
    with pytest.raises(OracleHipError, match='free pages'):
        small.check()
    m.same(small, 'too small')
    with pytest.raises(OracleHipError, match='differ'):
        c.compact(into=new_cache(n_pages=40, rows=7))
    with pytest.raises(OracleHipError, match='share'):
        c.compact(into=c)


def test_append_takes_slices_of_a_projection():
    c = new_cache(hkv=3, hd=128)
    slots = c.reserve(ints([2, 0]), ints([17, 5]), total=22)
    _, k, v = qkv(22, 6, 3, 128, BF, 7)
    m = Model(c)
    c.append(1, slots, k, v)
    m.append(1, slots.tolist(), k, v)
    m.same(c, 'slices')


# ---------------------------------------------------------------------------------------------- decode over a shared prefix
def filled(n, prefix, own, page, hkv, hd, dtype, seed, extra=2):
    """n rows of prefix + own[i] tokens; unused places of the pool hold NaN. -> (cache, dense K, dense V per row)"""
    import random
    r = random.Random(seed)
    shared = prefix // page
    width = shared + max(-(-max(own) // page), 1) + 1
    live = shared + sum(-(-x // page) for x in own)
    kv = torch.full((2, 2, live + extra, hkv, page, hd), float('nan'), dtype=dtype, device=DEV)
    order = r.sample(range(live + extra), live)
    table = torch.full((n, width), -1, dtype=torch.int32)
    head, at = order[:shared], shared
    g = torch.Generator(device=DEV).manual_seed(seed)
    fill = lambda: torch.randn(hkv, page, hd, generator=g, device=DEV).to(dtype)       # noqa: E731
    for p in head:
        for x in (0, 1):
            kv[1, x, p] = fill()
    dense = []
    for i in range(n):
        mine = order[at:at + -(-own[i] // page)]
        at += len(mine)
        table[i, :shared + len(mine)] = torch.tensor(head + mine, dtype=torch.int32)
        for j, p in enumerate(mine):
            m = min(page, own[i] - j * page)
            for x in (0, 1):
                kv[1, x, p, :, :m] = fill()[:, :m]
        pages = torch.tensor(head + mine, dtype=torch.long, device=DEV)
        dense.append([kv[1, x][pages].transpose(0, 1).flatten(1, 2)[:, :prefix + own[i]] for x in (0, 1)])
    refs = torch.zeros(live + extra, dtype=torch.int32)
    for p in table.flatten().tolist():
        if p >= 0:
            refs[p] += 1
    c = KvPages.wrap(kv, table.to(DEV), ints([prefix + x for x in own]), refs.to(DEV))
    return c, dense


@pytest.mark.parametrize('n, prefix, own, page', [
    (1, 0, [1], 16), (3, 0, [0, 5, 700], 64), (2, 16, [0, 1], 16), (5, 48, [0, 3, 16, 17, 33], 16), (4, 640, [31, 32, 33, 200], 32),
    (7, 1024, [0, 1, 2, 3, 127, 128, 129], 128), (20, 192, list(range(20)), 64), (3, 2304, [300, 1, 64], 64)], ids=str)
@pytest.mark.parametrize('hq, hkv, hd, dtype', [(4, 4, 128, BF), (8, 2, 64, FP), (24, 1, 128, FP), (40, 8, 64, BF)])
def test_attend(n, prefix, own, page, hq, hkv, hd, dtype):
    c, dense = filled(n, prefix, own, page, hkv, hd, dtype, n + prefix)
    q = (torch.randn(n, hq, hd, device=DEV) * 2).to(dtype)
    order = torch.randperm(n).tolist()
    out = c.attend(1, q, ints(order), prefix_tokens=prefix)
    c.check()
    for i, r in enumerate(order):
        if prefix + own[r] == 0:
            assert (out[i] == 0).all()
            continue
        ref, tol = attention64(q[i], *dense[r], hd ** -0.5)
        close(out[i], ref, tol, (i, r))
    if prefix:      # the same without the sharing
        apart = c.attend(1, q, ints(order))
        for i, r in enumerate(order):
            ref, tol = attention64(q[i], *dense[r], hd ** -0.5)
            close(apart[i], ref, tol, (i, r, 'apart'))


def test_attend_limits_rows_named_often_and_rows_outside():
    c, dense = filled(3, 64, [40, 0, 9], 32, 2, 128, BF, 11)
    rows = [0, 0, 0, 2, 1, 0, 7, -1, 2, 0, 2]
    limits = [104, 70, 65, 73, 64, 64, 5, 5, 33, 0, 1000]
    q = (torch.randn(len(rows), 6, 128, device=DEV) * 2).to(BF)
    out = c.attend(1, q, ints(rows), prefix_tokens=64, limits=ints(limits), scale=0.3)
    c.check()
    for i, (r, n) in enumerate(zip(rows, limits)):
        if r not in (0, 1, 2) or n == 0:
            assert (out[i] == 0).all()
            continue
        n = min(n, dense[r][0].shape[1])
        ref, tol = attention64(q[i], dense[r][0][:, :n], dense[r][1][:, :n], 0.3)
        close(out[i], ref, tol, (i, r, n))


@pytest.mark.parametrize('n, hq, hkv', [(2, 4, 2), (6, 8, 2), (40, 8, 2)])
def test_attend_odd_values_come_out_as_they_are(n, hq, hkv):
    c, _ = filled(n, 96, [5 + i % 7 for i in range(n)], 32, hkv, 64, FP, 50 + n)
    rows = ints(list(range(n)))
    q = torch.randn(n, hq, 64, device=DEV).to(FP)
    clean = c.attend(1, q, rows, prefix_tokens=96)
    page, g = int(c.table[0, 2]), hq // hkv
    for value in (float('inf'), float('-inf'), float('nan')):
        c.kv[1, 1, page, 1, 31, 9] = value            # the prefix's last token
        out = c.attend(1, q, rows, prefix_tokens=96)
        odd = torch.zeros_like(out, dtype=torch.bool)
        odd[:, g:2 * g, 9] = True
        assert (out[odd].isnan().all() if value != value else (out[odd] == value).all()) and torch.equal(out[~odd], clean[~odd])


def test_attend_many_columns_and_wide_groups():
    for n, hq, hkv, hd in ((70, 16, 2, 128), (5, 64, 1, 64), (1, 96, 1, 128)):
        own = [(7 * i) % 45 for i in range(n)]
        c, dense = filled(n, 320, own, 64, hkv, hd, BF, n)
        q = (torch.randn(n, hq, hd, device=DEV) * 2).to(BF)
        out = c.attend(1, q, ints(list(range(n))), prefix_tokens=320)
        for i in range(n):
            ref, tol = attention64(q[i], *dense[i], hd ** -0.5)
            close(out[i], ref, tol, (n, i))


def test_attend_pages_outside_the_pool_are_not_read():
    c, dense = filled(3, 0, [40, 70, 16], 16, 2, 64, FP, 13)
    q = torch.randn(3, 4, 64, device=DEV).to(FP)
    c.table[0, 1], c.table[1, 0], c.table[1, 4], c.table[2, 0] = 10 ** 9, -1, c.refs.numel(), -77
    out = c.attend(1, q, ints([0, 1, 2]))
    keep = [[*range(16), *range(32, 40)], [*range(16, 64)], []]
    for i in range(3):
        if not keep[i]:
            assert (out[i] == 0).all()
            continue
        ref, tol = attention64(q[i], dense[i][0][:, keep[i]], dense[i][1][:, keep[i]], 0.125)
        close(out[i], ref, tol, i)


def test_attend_notices_rows_that_do_not_share():
    c, _ = filled(3, 64, [5, 6, 7], 32, 2, 64, FP, 14)
    q = torch.randn(3, 4, 64, device=DEV).to(FP)
    c.attend(1, q, ints([2, 0, 1]), prefix_tokens=64)
    c.check()
    c.table[1, 1] = c.table[1, 2]
    c.attend(1, q, ints([2, 0, 1]), prefix_tokens=64)
    with pytest.raises(OracleHipError, match='share'):
        c.check()


def test_attend_a_freed_first_row_does_not_take_the_prefix_away():
    c, dense = filled(4, 64, [5, 6, 7, 0], 32, 2, 128, BF, 15)
    c.free(ints([2]))
    q = torch.randn(4, 4, 128, device=DEV).to(BF)
    out = c.attend(1, q, ints([2, 0, 1, 3]), prefix_tokens=64)
    c.check()
    assert (out[0] == 0).all()
    for i, r in ((1, 0), (2, 1), (3, 3)):
        ref, tol = attention64(q[i], *dense[r], 128 ** -0.5)
        close(out[i], ref, tol, i)


def test_attend_layouts_stream_graph_and_refusals():
    c, _ = filled(4, 128, [5, 60, 7, 0], 64, 2, 128, BF, 16)
    rows = ints([0, 1, 2, 3])
    q = torch.randn(4, 8, 128, device=DEV).to(BF)
    want = c.attend(1, q, rows, prefix_tokens=128)
    out = torch.empty(8, 4, 128, dtype=BF, device=DEV).transpose(0, 1)
    assert torch.equal(c.attend(1, q.transpose(0, 1).contiguous().transpose(0, 1), rows, prefix_tokens=128, out=out), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = c.attend(1, q, rows, prefix_tokens=128)
    side.synchronize()
    assert torch.equal(other, want)
    for bad in (lambda: c.attend(2, q, rows), lambda: c.attend(1, q.to(FP), rows), lambda: c.attend(1, q[:, :3], rows), lambda: c.attend(1, q[..., :64], rows),
                lambda: c.attend(1, q, rows[:3]), lambda: c.attend(1, q, rows, prefix_tokens=32), lambda: c.attend(1, q, rows, prefix_tokens=64 * 9),
                lambda: c.attend(1, q, rows, limits=rows[:2]), lambda: c.attend(1, q, rows, scale=0.0), lambda: c.attend(1, q, rows.long()),
                lambda: c.attend(1, q, rows, out=q[:2])):
        with pytest.raises(ValueError):
            bad()


def test_a_decode_step_in_a_graph_grows_the_rows():
    c, dense = filled(3, 64, [5, 30, 31], 32, 2, 64, FP, 17)
    c.table[:, 4:] = -1
    d, _ = filled(3, 64, [5, 30, 31], 32, 2, 64, FP, 17)
    rows = ints([1, 0, 2])
    k, v = torch.randn(2, 3, 2, 64, device=DEV).to(FP).unbind(0)
    q = torch.randn(3, 4, 64, device=DEV).to(FP)

    def step(x):
        slots = x.reserve(rows)
        x.append(1, slots, k, v)
        return x.attend(1, q, rows, prefix_tokens=64)

    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        captured = step(c)
    for i in range(3):
        k.normal_(), v.normal_(), q.normal_()
        want = step(d)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, want), i
        assert torch.equal(c.table, d.table) and torch.equal(c.lens, d.lens) and torch.equal(c.refs, d.refs)
    c.check(), d.check()


# ---------------------------------------------------------------------------------------------- together
def test_frames_and_questions_together():
    """Prompts in one packed pass, their K / V into pages, each frame forked to its questions, the questions' tokens over the shared
    prefix, answers token by token, rows that end, a compacted pool -- against dense attention of every row."""
    layers, hq, hkv, hd, page = 2, 8, 4, 128, 32
    lens = [150, 96]                                      # two frames
    c = KvPages(layers, 40, hkv, hd, page_size=page, max_rows=10, max_row_pages=8)
    dense = {r: [([], []) for _ in range(layers)] for r in range(10)}
    plan = PackedPlan(lens)
    slots = c.reserve(ints([0, 1]), ints(lens), total=sum(lens))
    for layer in range(layers):
        q, k, v = qkv(sum(lens), hq, hkv, hd, BF, 30 + layer)
        ref, tol = packed64(q, k, v, lens, hd ** -0.5)
        close(packed_attention(q, k, v, plan), ref, tol, 'prompts')
        c.append(layer, slots, k, v)
        for r, a, b in ((0, 0, 150), (1, 150, 246)):
            dense[r][layer] = ([*k[a:b]], [*v[a:b]])
    c.fork(ints([0, 0, 0, 1, 1]), ints([2, 3, 4, 5, 6]))
    for r, s in ((2, 0), (3, 0), (4, 0), (5, 1), (6, 1)):
        dense[r] = [([*a], [*b]) for a, b in dense[s]]

    def tokens(rows, counts, prefix, seed):
        """counts[i] more tokens of row rows[i]; every one attends to all before it"""
        slots = c.reserve(ints(rows), ints(counts), total=sum(counts))
        who = [r for r, n in zip(rows, counts) for _ in range(n)]
        first = {r: len(dense[r][0][0]) for r in rows}
        limits = [first[r] + j + 1 for r, n in zip(rows, counts) for j in range(n)]
        for layer in range(layers):
            q, k, v = qkv(len(who), hq, hkv, hd, BF, seed + layer)
            c.append(layer, slots, k, v)
            for i, r in enumerate(who):
                dense[r][layer][0].append(k[i])
                dense[r][layer][1].append(v[i])
            out = c.attend(layer, q, ints(who), prefix_tokens=prefix, limits=ints(limits))
            for i, r in enumerate(who):
                kk, vv = (torch.stack(x[:limits[i]]).transpose(0, 1) for x in dense[r][layer])
                ref, tol = attention64(q[i], kk, vv, hd ** -0.5)
                close(out[i], ref, tol, (seed, i, r))
        c.check()

    tokens([2, 3, 4], [7, 1, 12], 128, 40)                # the questions of the first frame, then of the second
    tokens([5, 6], [3, 33], 96, 50)
    for step in range(3):
        tokens([2, 3, 4], [1, 1, 1], 128, 60 + 10 * step)
    c.free(ints([3, 0]))
    tokens([2, 4], [1, 1], 128, 100)                      # the frame's own row is gone, its pages are not
    c.compact()
    held = int((c.refs > 0).sum())
    assert (c.refs[:held] > 0).all() and (c.refs[held:] == 0).all()
    tokens([4, 2], [1, 1], 128, 110)
    bigger = KvPages(layers, 64, hkv, hd, page_size=page, max_rows=10, max_row_pages=8)
    c.compact(into=bigger)
    c = bigger
    tokens([6, 5], [1, 1], 96, 120)
