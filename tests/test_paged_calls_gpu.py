"""GPU: calls of packed_attention and KvPages that their documentation allows and that are easily got wrong. The oracle and its tolerance
are test_paged_gpu's."""
import pytest
import torch
from torch.autograd import forward_ad

from oracle_amd._lib import OracleHipError
from oracle_amd.paged import KvPages, PackedPlan, packed_attention
from test_paged_gpu import attention64, close, filled, ints, qkv

pytestmark = pytest.mark.gpu
DEV = 'cuda'
BF, FP = torch.bfloat16, torch.float16


# Columns that see keys of an item and columns that end in front of it, in turn, where a NaN behind some limits makes the item run column by column: a
# column without keys must not disturb the one before it, whose parts are still being joined.
@pytest.mark.parametrize('n, hq, hkv', [(16, 1, 1), (8, 4, 2), (32, 2, 2), (64, 8, 2)])
@pytest.mark.parametrize('hd, dtype', [(128, BF), (64, FP)])
def test_attend_columns_without_keys_behind_columns_with_keys(n, hq, hkv, hd, dtype):
    prefix = 1024
    c, dense = filled(n, prefix, [i % 3 for i in range(n)], 64, hkv, hd, dtype, 80 + n)
    for token in (200, 500, 900):
        c.kv[1, 1, int(c.table[0, token // 64]), :, token % 64, 7] = float('nan')
    q, rows = torch.randn(n, hq, hd, device=DEV).to(dtype), ints(list(range(n)))
    for most in (180, 499, 899):                      # of each item: some columns end inside, every other one at once
        limits = [most - 37 * (i % 5) if i % 2 == 0 else (0, -1, 1)[i // 2 % 3] for i in range(n)]
        first = c.attend(1, q, rows, prefix_tokens=prefix, limits=ints(limits))
        for _ in range(30):
            assert torch.equal(c.attend(1, q, rows, prefix_tokens=prefix, limits=ints(limits)).nan_to_num(99.0), first.nan_to_num(99.0))
        c.check()
        for i, m in enumerate(limits):
            if m <= 0:
                assert (first[i] == 0).all()
            else:
                k, v = (x[:, :m] for x in dense[i])
                ref, tol = attention64(q[i], k, v, hd ** -0.5)
                keep = [d for d in range(hd) if d != 7 or m <= 200]       # `dense` was taken before the NaN went in
                close(first[i][:, keep], ref[:, keep], tol[:, keep], (most, i))
                assert 7 in keep or first[i, :, 7].isnan().all()


def test_packed_attention_into_slices_of_the_projection():
    lens, hq, hkv, hd = [90, 33], 4, 4, 64
    q, k, v = qkv(sum(lens), hq, hkv, hd, FP, 90)
    plan = PackedPlan(lens)
    want = packed_attention(q, k, v, plan)
    rows = torch.cat([q, k, v], 1)                                                   # (T, heads of q, k, v, hd)
    kv = rows[:, hq:].clone()
    out = rows[:, :hq]
    assert packed_attention(out, rows[:, hq:2 * hq], rows[:, 2 * hq:], plan, out=out) is out
    assert torch.equal(out, want) and torch.equal(rows[:, hq:], kv)
    heads = torch.stack([q, k, v], 2)                                                # (T, heads, q k v, hd)
    out = heads[:, :, 0]
    assert packed_attention(out, heads[:, :, 1], heads[:, :, 2], plan, out=out) is out
    assert torch.equal(out, want) and torch.equal(heads[:, :, 1], k)
    rows = torch.cat([q, k, v], 1)
    for out, text in ((rows[:, hq:2 * hq], 'k or v'), (rows[:, 2 * hq:], 'k or v'), (rows[:, 1:1 + hq], 'k or v')):
        with pytest.raises(OracleHipError, match=text):
            packed_attention(rows[:, :hq], rows[:, hq:2 * hq], rows[:, 2 * hq:], plan, out=out)
    room = torch.zeros(sum(lens) + 1, hq, hd, dtype=FP, device=DEV)
    with pytest.raises(OracleHipError, match='over q'):
        packed_attention(room[1:], k, v, plan, out=room[:-1])


def test_attend_into_the_pool_or_a_shifted_query_is_refused():
    c, _ = filled(3, 0, [5, 70, 2], 64, 2, 64, FP, 91)
    rows, room = ints([0, 1, 2]), torch.zeros(4, 4, 64, dtype=FP, device=DEV)
    with pytest.raises(OracleHipError, match='over q'):
        c.attend(1, room[1:], rows, out=room[:-1])
    before = c.kv.clone()
    with pytest.raises(OracleHipError, match='over the pool'):
        c.attend(1, room[1:], rows, out=c.kv.view(-1)[:3 * 4 * 64].view(3, 4, 64))
    assert torch.equal(c.kv.view(torch.int16), before.view(torch.int16))


def test_tensors_with_a_tangent_are_refused():
    c, _ = filled(2, 0, [3, 4], 32, 2, 64, FP, 92)
    q, k, v = qkv(16, 4, 2, 64, FP, 92)
    plan, rows = PackedPlan([16]), ints([0, 1])
    slots = c.reserve(rows)
    c.append(1, slots, k[:2], v[:2])                  # (what `filled` leaves in a free place is NaN)
    want, one = packed_attention(q, k, v, plan), c.attend(1, q[:2], rows)
    with forward_ad.dual_level():
        dual = lambda x: forward_ad.make_dual(x, torch.ones_like(x))      # noqa: E731
        for i in range(3):
            x = [q, k, v]
            x[i] = dual(x[i])
            for mode in (torch.enable_grad(), torch.no_grad()):
                with mode, pytest.raises(ValueError, match='tangent'):
                    packed_attention(*x, plan)
        for call in (lambda: packed_attention(q, k, v, plan, out=dual(torch.empty_like(q))), lambda: c.attend(1, dual(q[:2]), rows),
                     lambda: c.attend(1, q[:2], rows, out=dual(torch.empty_like(q[:2]))), lambda: c.append(1, slots, dual(k[:2]), v[:2]),
                     lambda: c.append(1, slots, k[:2], dual(v[:2])), lambda: KvPages.wrap(dual(c.kv), c.table, c.lens, c.refs)):
            with pytest.raises(ValueError, match='tangent'):
                call()
        assert torch.equal(packed_attention(forward_ad.unpack_dual(dual(q)).primal, k, v, plan), want)      # without one: as outside
        assert torch.equal(c.attend(1, q[:2], rows), one)


# A row whose last, part page is not one of the pool's: its next tokens have no place (page * page_size may even come out as another page's)
@pytest.mark.parametrize('bad', [-1, 40, (1 << 28) + 1, -(1 << 28)])
def test_reserve_refuses_a_part_page_outside_the_pool(bad):
    c, _ = filled(3, 0, [21, 5, 16], 16, 2, 64, FP, 93, extra=6)
    c.table[0, 1] = bad
    before = [x.clone() for x in (c.table, c.lens, c.refs)]
    for rows, counts in ((ints([0]), None), (ints([1, 0, 2]), ints([3, 20, 1])), (ints([2, 1, 0]), ints([0, 0, 1]))):
        slots = c.reserve(rows, counts, total=None if counts is None else 44)
        with pytest.raises(OracleHipError, match='a page outside the pool'):
            c.check()
        assert (slots == -1).all() and all(torch.equal(x, y) for x, y in zip(before, (c.table, c.lens, c.refs)))
    assert (c.reserve(ints([0, 1, 2]), ints([0, 2, 1]), total=3) >= 0).all()      # no token for that row: its page does not matter
    c.check()


# Scores of -inf at every token a query sees: the softmax is 0 / 0, as packed_attention has it; a query without tokens keeps its zeros
@pytest.mark.parametrize('n, prefix, hq, hkv', [(4, 0, 4, 2), (4, 64, 4, 2), (40, 64, 8, 2), (300, 0, 4, 2)])
def test_scores_of_minus_infinity_alone_give_nan(n, prefix, hq, hkv):
    hd, own = 64, [(0, 3, 70, 17)[i % 4] for i in range(n)]
    c, dense = filled(n, prefix, own, 32, hkv, hd, BF, 94)
    q = torch.randn(n, hq, hd, device=DEV).to(BF)
    q[..., 5] = q[..., 5].abs() + 1
    rows, limits = ints(list(range(n))), [prefix + own[i] if i % 3 else (1, 0, prefix + 2)[i // 3 % 3] for i in range(n)]
    for kh in range(hkv):
        c2 = KvPages.wrap(c.kv.clone(), c.table, c.lens, c.refs)
        c2.kv[1, 0, :, kh, :, 5] = float('-inf')
        for lim in (None, limits):
            out = c2.attend(1, q, rows, prefix_tokens=prefix, limits=None if lim is None else ints(lim))
            for i in range(n):
                m = min(prefix + own[i], prefix + own[i] if lim is None else lim[i])
                if m <= 0:
                    assert (out[i] == 0).all()
                    continue
                g = slice(kh * hq // hkv, (kh + 1) * hq // hkv)
                assert out[i, g].isnan().all(), i
                k, v = (x[:, :m] for x in dense[i])
                ref, tol = attention64(q[i], k, v, hd ** -0.5)
                rest = [h for h in range(hq) if not g.start <= h < g.stop]
                close(out[i, rest], ref[rest], tol[rest], i)
        c2.check()
        if not prefix:                                                     # no page of the pool is no token
            gone = c2.table.clone()
            gone[2] = -1
            assert (KvPages.wrap(c2.kv, gone, c.lens, c.refs).attend(1, q, rows)[2] == 0).all()
    k, v = q[:3, :hkv].clone(), q[:3, :hkv]
    k[..., 5] = float('-inf')
    assert packed_attention(q[:3], k, v, PackedPlan([3])).isnan().all()


@pytest.mark.parametrize('prefix, n, hd', [(201 * 64, 40, 64), (201 * 64, 40, 128), (16 * 256 + 32, 2, 64)])
def test_attend_prefixes_whose_tiles_do_not_divide_by_their_parts(prefix, n, hd):
    c, dense = filled(n, prefix, [i % 4 for i in range(n)], 32, 1, hd, BF, 95)
    q = torch.randn(n, 8 if n > 2 else 2, hd, device=DEV).to(BF)
    out = c.attend(1, q, ints(list(range(n))), prefix_tokens=prefix)
    c.check()
    for i in range(0, n, 7):
        ref, tol = attention64(q[i], *dense[i], hd ** -0.5)
        close(out[i], ref, tol, i)


# What a plan or a cache made for itself is not given to others while a stream that used it is still at it
def test_a_plan_or_cache_let_go_while_another_stream_uses_it():
    lens = [70, 300]
    q, k, v = qkv(sum(lens), 4, 2, 64, FP, 96)
    plan = PackedPlan(lens)
    want = packed_attention(q, k, v, plan)
    c, _ = filled(3, 0, [5, 40, 9], 32, 2, 64, FP, 97)
    rows = ints([0, 1, 2])
    one, side = c.attend(1, q[:3], rows), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)
        out, two = packed_attention(q, k, v, plan), c.attend(1, q[:3], rows)
    held = {t.data_ptr(): t.numel() for t in (plan.work, c.status, c._work)}
    del plan, c
    assert not side.query()                                            # still asleep
    fresh = [torch.empty(n, dtype=torch.int32, device=DEV) for n in held.values() for _ in range(64)]
    assert not held.keys() & {t.data_ptr() for t in fresh}
    side.synchronize()
    assert torch.equal(out, want) and torch.equal(two, one)


# All scores -inf and an infinity in V: 0 / 0 is NaN in every dim, the one of the infinity too
@pytest.mark.parametrize('hd, dtype', [(128, BF), (64, FP)])
def test_scores_of_minus_infinity_over_an_infinite_value_give_nan(hd, dtype):
    for lens in ([1, 1], [3, 70], [64, 130]):
        q, k, v = (x.clone() for x in qkv(sum(lens), 4, 2, hd, dtype, 98))
        q[..., 5] = q[..., 5].abs() + 1
        clean = packed_attention(q, k, v, PackedPlan(lens))
        k[:lens[0], 1, 5], v[0, 1, 19] = float('-inf'), float('inf')
        out = packed_attention(q, k, v, PackedPlan(lens))
        assert out[:lens[0], 2:].isnan().all() and torch.equal(out[:, :2], clean[:, :2]) and torch.equal(out[lens[0]:], clean[lens[0]:])
        c = KvPages(1, 40, 2, hd, page_size=16, max_rows=2, max_row_pages=20, dtype=dtype)
        c.append(0, c.reserve(ints([0, 1]), ints(lens), total=sum(lens)), k, v)
        out = c.attend(0, q[-2:], ints([0, 1]))
        assert out[0, 2:].isnan().all() and torch.isfinite(out[0, :2]).all() and torch.isfinite(out[1]).all()
