"""What is measured of the paged KV cache and of the attention over packed prompts (oracle_amd/paged.py): the cases, their inputs,
a plain form of every operator in elementary torch operations (`own = False`) and the calls a user makes (`own = True`)."""
import math
import random

import torch

own = False

DTYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16}
DEV = 'cuda'


# ------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # packed prompts ------------------------------------------------------------------------------
        # four short text prompts on the reduced test model (4 heads of 128): latency
        dict(name='packed_tiny', op='packed', n=4, lo=9, hi=61, pick=1, hq=4, hkv=4, hd=128, dtype='bf16'),
        # a batch of 8 frames: image tokens + prompts of 640..900 tokens on the 7B model's 32 heads
        dict(name='packed_frames', op='packed', n=8, lo=640, hi=900, pick=2, hq=32, hkv=32, hd=128, dtype='bf16'),
        # many prompts of very different lengths, grouped heads of 64, fp16; empty and one-token prompts among them
        dict(name='packed_ragged_hd64', op='packed', n=48, lo=0, hi=2305, pick=3, hq=16, hkv=4, hd=64, dtype='fp16'),
        # two long documents with grouped heads
        dict(name='packed_long_gqa', op='packed', n=2, lo=15001, hi=24001, pick=4, hq=32, hkv=8, hd=128, dtype='bf16'),
        # decode over a shared prefix -------------------------------------------------------------------
        # two questions about one view (576 image tokens) on the reduced model: latency
        dict(name='prefix_tiny', op='attend', n=2, prefix=576, lo=3, hi=40, pick=5, hq=4, hkv=4, hd=128, page=64, dtype='bf16'),
        # 16 questions about one frame on the 7B model: 2304 shared tokens (4 views), answers of up to 300 tokens
        dict(name='prefix_frame', op='attend', n=16, prefix=2304, lo=1, hi=300, pick=6, hq=32, hkv=32, hd=128, page=64, dtype='bf16'),
        # 96 rows over a 32k-token context with grouped heads, suffixes up to 2000 tokens
        dict(name='prefix_long_gqa', op='attend', n=96, prefix=32768, lo=0, hi=2001, pick=7, hq=32, hkv=8, hd=128, page=128, dtype='bf16'),
        # filling the cache -----------------------------------------------------------------------------
        # the scatter of one decode step of one layer: 32 new tokens
        dict(name='append_step', op='append', n=32, lo=1, hi=1, pick=8, layers=1, hkv=32, hd=128, page=64, dtype='bf16'),
        # rows are freed and admitted again: pages of 8 prompts are taken and filled in four layers
        dict(name='admit_prompts', op='append', n=8, lo=640, hi=900, pick=9, layers=4, hkv=32, hd=128, page=64, dtype='bf16'),
        # pages -----------------------------------------------------------------------------------------
        # one frame's rows forked to 24 questions, shared but for the part page
        dict(name='fork_questions', op='fork', n=24, parents=2, lo=2000, hi=2400, pick=10, layers=8, hkv=8, hd=128, page=64, dtype='bf16'),
        # three rows copied in full
        dict(name='copy_rows', op='copy', n=3, parents=3, lo=100, hi=4000, pick=11, layers=16, hkv=8, hd=64, page=16, dtype='fp16'),
        # a fragmented pool moved, without its holes, into another one
        dict(name='compact_pool', op='compact', n=40, parents=40, lo=200, hi=1100, pick=12, layers=8, hkv=8, hd=128, page=32, dtype='bf16'),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(('packed', 'packed', 'packed', 'attend', 'attend', 'attend', 'append', 'fork', 'copy', 'compact'))
    hkv = rng.choice((1, 2, 4, 8, 32))
    hq = hkv * rng.choice((1, 2, 4, 8) if hkv <= 8 else (1,))
    hd = rng.choice((64, 128, 128))
    c = dict(op=op, hkv=hkv, hd=hd, dtype=rng.choice(('bf16', 'bf16', 'fp16')), pick=rng.randrange(1 << 20))
    if op == 'packed':
        n = _log_int(rng, 1, 48)
        hi = _log_int(rng, 2, max(3, 32768 // n))
        c.update(n=n, lo=rng.choice((0, 1, hi // 2)), hi=hi, hq=hq)
        while work(c)['flops'] > 6.0e12:                             # no dearer than the long documents above
            c['hi'] = c['hi'] * 3 // 4
            c['lo'] = min(c['lo'], c['hi'])
    elif op == 'attend':
        page = rng.choice((16, 32, 64, 128))
        n = _log_int(rng, 1, 96)
        c.update(n=n, page=page, prefix=page * rng.choice((0, 1, _log_int(rng, 1, 32768 // page), _log_int(rng, 1, 32768 // page))),
                 lo=0, hi=_log_int(rng, 1, 2000), hq=hq)
    else:
        page = rng.choice((16, 32, 64, 128))
        hkv = c['hkv'] = min(hkv, 8)
        layers = rng.choice((1, 2, 4, 8))
        n = _log_int(rng, 1, 40)
        hi = _log_int(rng, 1, 900)
        c.update(n=n, page=page, layers=layers, lo=rng.choice((0, 1)), hi=hi)
        if op in ('fork', 'copy'):
            c['parents'] = max(1, n // rng.choice((1, 2, 5)))
        elif op == 'compact':
            c['parents'] = n
    return c


def _lengths(c):
    """The lengths of a case: spread over lo..hi (over the logarithm where hi is far above lo), with both ends among them."""
    r = random.Random(c['pick'])
    n, lo, hi = c.get('parents', c['n']), c['lo'], c['hi']
    out = []
    for _ in range(n):
        if hi > 10 * max(lo, 1) and r.random() < 0.5:
            out.append(min(hi, max(lo, _log_int(r, max(lo, 1), hi))))
        else:
            out.append(r.randint(lo, hi))
    if n > 1:
        out[r.randrange(n)] = lo
    out[r.randrange(n)] = hi
    return out


def _pages(tokens, page):
    return -(-tokens // page)


# ------------------------------------------------------------------------------------------------- inputs
def _randn(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEV, dtype=torch.float32) * scale).to(dtype)


def _state(c, seed):
    """The paged cache of a case: pool, page table, lengths and reference counts, with pages in no particular order."""
    g = torch.Generator(device=DEV).manual_seed(seed * 7919 + 17)
    r = random.Random(seed * 104729 + 5)
    page, layers, dt = c['page'], c.get('layers', 1), DTYPES[c['dtype']]
    op, n = c['op'], c['n']
    lens = _lengths(c)
    if op == 'attend':
        shared = c['prefix'] // page
        own_pages = [_pages(x, page) for x in lens]
        width = shared + max(own_pages + [1])
        rows, live = n, shared + sum(own_pages)
        n_pages = live + 3
        order = r.sample(range(n_pages), live)
        table = [[-1] * width for _ in range(rows)]
        at = shared
        for i in range(rows):
            table[i][:shared] = order[:shared]
            table[i][shared:shared + own_pages[i]] = order[at:at + own_pages[i]]
            at += own_pages[i]
        total = [c['prefix'] + x for x in lens]
    else:
        own_pages = [_pages(x, page) for x in lens]
        width = max(own_pages + [1]) + 1
        first = len(lens)                                            # rows that hold tokens from the start
        rows = first + (n if op in ('fork', 'copy') else 0)
        live = sum(own_pages)
        each = [_pages(lens[i % first], page) for i in range(n)]
        n_pages = {'append': 2 * live, 'fork': live + n, 'copy': live + sum(each), 'compact': live + live // 2}[op] + 5
        order = r.sample(range(n_pages), live)
        table = [[-1] * width for _ in range(rows)]
        at = 0
        for i in range(first):
            table[i][:own_pages[i]] = order[at:at + own_pages[i]]
            at += own_pages[i]
        total = lens + [0] * (rows - first)
    refs = [0] * n_pages
    for row in table:
        for p in row:
            if p >= 0:
                refs[p] += 1
    kv = torch.empty(layers, 2, n_pages, c['hkv'], page, c['hd'], dtype=dt, device=DEV)
    for layer in range(layers):
        kv[layer] = _randn(g, kv.shape[1:], dt)
    as_dev = lambda x: torch.tensor(x, dtype=torch.int32).to(DEV)    # noqa: E731
    return dict(case=c, kv=kv, table=as_dev(table), lens=as_dev(total), refs=as_dev(refs), lengths=lens), g, r


def prepare(case, seed):
    c = dict(case)
    dt = DTYPES[c['dtype']]
    if c['op'] == 'packed':
        g = torch.Generator(device=DEV).manual_seed(seed * 7919 + 11)
        lens = _lengths(c)
        total = sum(lens)
        # one fused projection's output, as a model hands it over: q, k and v are slices of its rows
        qkv = _randn(g, (total, c['hq'] + 2 * c['hkv'], c['hd']), dt)
        qkv[:, :c['hq']] *= 2.0
        s = dict(case=c, lengths=lens, q=qkv[:, :c['hq']], k=qkv[:, c['hq']:c['hq'] + c['hkv']], v=qkv[:, c['hq'] + c['hkv']:])
        if own:
            from oracle_amd.paged import PackedPlan
            s['plan'] = PackedPlan(lens, device=DEV)
        return s
    s, g, r = _state(c, seed)
    n, page = c['n'], c['page']
    dev = lambda x: torch.tensor(x, dtype=torch.int32).to(DEV)       # noqa: E731
    if c['op'] == 'attend':
        s['q'] = _randn(g, (n, c['hq'], c['hd']), dt, 2.0)
        s['rows'] = dev(r.sample(range(n), n))                       # the batch lists its rows in an order of its own
        s['longest'] = max(s['lengths'])
    elif c['op'] == 'append':
        total = sum(s['lengths'])
        s['k'] = [_randn(g, (total, c['hkv'], c['hd']), dt) for _ in range(c['layers'])]
        s['v'] = [_randn(g, (total, c['hkv'], c['hd']), dt) for _ in range(c['layers'])]
        s['rows'], s['counts'], s['total'] = dev(list(range(n))), dev(s['lengths']), total
        if c['hi'] == 1 and c['lo'] == 1:                            # a decode step: its places in the pool are known already
            t = s['table'][:, 0]
            s['slots'] = (t * page).to(torch.int32).contiguous()
    elif c['op'] in ('fork', 'copy'):
        p = c['parents']
        s['src'], s['dst'] = dev([i % p for i in range(n)]), dev([p + i for i in range(n)])
        s['src_host'] = [i % p for i in range(n)]
    else:
        live = sum(_pages(x, page) for x in s['lengths'])
        s['into'] = dict(kv=torch.zeros(c['layers'], 2, live + 2, c['hkv'], page, c['hd'], dtype=dt, device=DEV),
                         table=torch.full_like(s['table'], -1), lens=torch.zeros_like(s['lens']),
                         refs=torch.zeros(live + 2, dtype=torch.int32, device=DEV))
    if own:
        from oracle_amd.paged import KvPages
        s['pages'] = KvPages.wrap(s['kv'], s['table'], s['lens'], s['refs'])
        if c['op'] == 'compact':
            s['pages_into'] = KvPages.wrap(**s['into'])
    return s


# ------------------------------------------------------------------------------------------------- one pass
def run(s):
    return {'packed': _packed, 'attend': _attend, 'append': _append, 'fork': _fork, 'copy': _fork, 'compact': _compact}[s['case']['op']](s)


def _softmax_product(q, k, v, visible, scale):
    """q (H, M, hd), k / v (H, N, hd) float; visible (M, N) or broadcastable, or None."""
    x = torch.matmul(q * scale, k.transpose(1, 2).contiguous())
    if visible is not None:
        x = x.masked_fill(~visible, float('-inf'))
    p = torch.exp(x - x.amax(-1, keepdim=True))
    return torch.matmul(p, v) / p.sum(-1, keepdim=True)


def _packed(s):
    c = s['case']
    if own:
        from oracle_amd.paged import packed_attention
        return packed_attention(s['q'], s['k'], s['v'], s['plan'])
    out = torch.empty_like(s['q'], memory_format=torch.contiguous_format)
    at, group = 0, c['hq'] // c['hkv']
    for length in s['lengths']:
        if length:
            q, k, v = (s[x][at:at + length].transpose(0, 1).float().contiguous() for x in 'qkv')
            k, v = k.repeat_interleave(group, 0), v.repeat_interleave(group, 0)
            for lo in range(0, length, 1024):
                hi = min(lo + 1024, length)
                visible = torch.arange(hi, device=DEV)[None, :] <= torch.arange(lo, hi, device=DEV)[:, None]
                o = _softmax_product(q[:, lo:hi], k[:, :hi], v[:, :hi], visible, c['hd'] ** -0.5)
                out[at + lo:at + hi] = o.transpose(0, 1).to(out.dtype)
        at += length
    return out


def _attend(s):
    c = s['case']
    if own:
        return s['pages'].attend(0, s['q'], s['rows'], prefix_tokens=c['prefix'])
    n, group, hd, hkv, page = c['n'], c['hq'] // c['hkv'], c['hd'], c['hkv'], c['page']
    rows = s['rows'].long()
    lens, table = s['lens'][rows].long(), s['table'][rows].long()
    shared, wide = c['prefix'] // page, _pages(max(s['longest'], 1), page)
    q = s['q'].float().view(n, hkv, group, hd) * hd ** -0.5
    k, v = s['kv'][0, 0], s['kv'][0, 1]
    tail = table[:, shared:shared + wide].clamp_min(0)
    tail_k = k[tail].float().permute(0, 2, 1, 3, 4).reshape(n, hkv, -1, hd)      # (n, hkv, tokens, hd)
    tail_v = v[tail].float().permute(0, 2, 1, 3, 4).reshape(n, hkv, -1, hd)
    x = torch.matmul(q, tail_k.transpose(2, 3).contiguous())                     # (n, hkv, group, tokens)
    there = torch.arange(x.shape[-1], device=DEV)[None, :] < (lens - c['prefix'])[:, None]
    x = x.masked_fill(~there[:, None, None, :], float('-inf'))
    top = x.amax(-1, keepdim=True)
    if shared:
        head_k = k[table[0, :shared]].float().transpose(0, 1).reshape(hkv, -1, hd)
        head_v = v[table[0, :shared]].float().transpose(0, 1).reshape(hkv, -1, hd)
        y = torch.matmul(q.permute(1, 0, 2, 3).reshape(hkv, n * group, hd), head_k.transpose(1, 2).contiguous())
        y = y.view(hkv, n, group, -1).permute(1, 0, 2, 3)
        top = torch.maximum(top, y.amax(-1, keepdim=True))
    top = top.masked_fill(torch.isinf(top), 0.0)                                 # a row without tokens: zeros
    p = torch.exp(x - top)
    total, o = p.sum(-1, keepdim=True), torch.matmul(p, tail_v)
    if shared:
        p = torch.exp(y - top)
        total = total + p.sum(-1, keepdim=True)
        p = p.permute(1, 0, 2, 3).reshape(hkv, n * group, -1)
        o = o + torch.matmul(p, head_v).view(hkv, n, group, hd).permute(1, 0, 2, 3)
    return (o / total.clamp_min(1e-30)).reshape(n, c['hq'], hd).to(s['q'].dtype)


def _plain_free(s, rows):
    """Takes the pages of `rows` (host list) back."""
    t = s['table'][rows]
    held = t[t >= 0].long()
    s['refs'].index_add_(0, held, torch.full_like(held, -1, dtype=torch.int32))
    s['table'][rows] = -1
    s['lens'][rows] = 0


def _plain_take(s, count):
    return (s['refs'] == 0).nonzero().flatten()[:count]                          # the lowest free pages


def _append(s):
    c = s['case']
    page = c['page']
    if own:
        p = s['pages']
        if 'slots' in s:
            for layer in range(c['layers']):
                p.append(layer, s['slots'], s['k'][layer], s['v'][layer])
            return [s['kv']]
        p.free(s['rows'])
        slots = p.reserve(s['rows'], s['counts'], total=s['total'])
        for layer in range(c['layers']):
            p.append(layer, slots, s['k'][layer], s['v'][layer])
        return [s['kv'], s['table'], s['lens'], s['refs'], slots]
    if 'slots' in s:
        slots = s['slots'].long()
        for layer in range(c['layers']):
            s['kv'][layer, 0, slots // page, :, slots % page] = s['k'][layer]
            s['kv'][layer, 1, slots // page, :, slots % page] = s['v'][layer]
        return [s['kv']]
    rows = list(range(c['n']))
    _plain_free(s, rows)
    need = [_pages(x, page) for x in s['lengths']]
    got, at, slots = _plain_take(s, sum(need)), 0, []
    s['refs'][got] = 1
    for i, length in enumerate(s['lengths']):
        mine = got[at:at + need[i]]
        at += need[i]
        s['table'][i, :need[i]] = mine.int()
        t = torch.arange(length, device=DEV)
        slots.append(mine[t // page] * page + t % page)
    s['lens'][:] = s['counts']
    slots = torch.cat(slots)
    for layer in range(c['layers']):
        s['kv'][layer, 0, slots // page, :, slots % page] = s['k'][layer]
        s['kv'][layer, 1, slots // page, :, slots % page] = s['v'][layer]
    return [s['kv'], s['table'], s['lens'], s['refs'], slots.int()]


def _fork(s):
    """The children are freed (a first pass finds them empty) and forked, or copied in full, again."""
    c = s['case']
    n, page, parents = c['n'], c['page'], c['parents']
    if own:
        p = s['pages']
        p.free(s['dst'])
        (p.fork if c['op'] == 'fork' else p.copy)(s['src'], s['dst'])
    else:
        _plain_free(s, list(range(parents, parents + n)))
        for i in range(n):
            src, dst = s['src_host'][i], parents + i
            length = s['lengths'][src]
            keep = length // page if c['op'] == 'fork' else 0
            used = _pages(length, page)
            fresh = _plain_take(s, used - keep)
            old = s['table'][src, keep:used].long()
            s['table'][dst, :keep] = s['table'][src, :keep]
            s['table'][dst, keep:used] = fresh.int()
            s['refs'][s['table'][dst, :used].long()] += 1
            s['lens'][dst] = length
            part = length % page
            whole = used - keep - (1 if part else 0)
            if whole:
                s['kv'][:, :, fresh[:whole]] = s['kv'][:, :, old[:whole]]
            if part:                                                             # the tokens behind the last are left as they were
                s['kv'][:, :, fresh[-1], :, :part] = s['kv'][:, :, old[-1], :, :part]
    return [s['kv'], s['table'], s['lens'], s['refs']]


def _compact(s):
    t = s['into']
    if own:
        s['pages'].compact(into=s['pages_into'])
    else:
        live = (s['refs'] > 0).nonzero().flatten()
        place = torch.full_like(s['refs'], -1)
        place[live] = torch.arange(live.numel(), device=DEV, dtype=torch.int32)
        t['kv'][:, :, :live.numel()] = s['kv'][:, :, live]
        t['table'][:] = torch.where(s['table'] >= 0, place[s['table'].clamp_min(0).long()], -1)
        t['lens'][:] = s['lens']
        t['refs'][:] = 0
        t['refs'][:live.numel()] = s['refs'][live]
    return [t['kv'], t['table'], t['lens'], t['refs']]


# ------------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    c = case
    lens, item = _lengths(c), 2
    if c['op'] == 'packed':
        total = sum(lens)
        return {'bytes': item * total * c['hd'] * (2 * c['hq'] + 2 * c['hkv']), 'flops': 4 * c['hd'] * c['hq'] * sum(x * (x + 1) // 2 for x in lens)}
    token = 2 * c['hkv'] * c['hd'] * item                                        # K and V of one token in one layer
    if c['op'] == 'attend':
        table = 4 * (c['prefix'] // c['page'] + sum(_pages(x, c['page']) for x in lens))
        return {'bytes': token * (c['prefix'] + sum(lens)) + 2 * item * c['n'] * c['hq'] * c['hd'] + table,
                'flops': 4 * c['hd'] * c['hq'] * sum(c['prefix'] + x for x in lens)}
    if c['op'] == 'append':
        return {'bytes': 2 * token * sum(lens) * c['layers'] + 8 * sum(lens), 'flops': 0}
    if c['op'] in ('fork', 'copy'):
        each = [lens[i % c['parents']] for i in range(c['n'])]
        moved = sum(x % c['page'] if c['op'] == 'fork' else x for x in each)
        return {'bytes': 2 * token * moved * c['layers'] + 16 * sum(_pages(x, c['page']) for x in each), 'flops': 0}
    live = sum(_pages(x, c['page']) for x in lens)
    return {'bytes': 2 * token * c['page'] * live * c['layers'] + 24 * live, 'flops': 0}


# ------------------------------------------------------------------------------------------------- the definition, in 64 bits
def exact(case, seed):
    c = case
    s = prepare(case, seed)
    if c['op'] == 'packed':
        return _exact_packed(c, s)
    if c['op'] == 'attend':
        return _exact_attend(c, s)
    page = c['page']
    kv, table, lens, refs = s['kv'], s['table'].tolist(), s['lens'].tolist(), s['refs'].tolist()
    pages_of = lambda tokens: (tokens + page - 1) // page                        # noqa: E731
    place = lambda row, t: (table[row][t // page], t % page)                     # noqa: E731

    def take():
        p = refs.index(0)
        refs[p] = 1
        return p

    def give(row):
        for j, p in enumerate(table[row]):
            if p >= 0:
                refs[p] -= 1
                table[row][j] = -1
        lens[row] = 0

    result = kv.double()
    if c['op'] == 'append':
        if 'slots' in s:
            for i, x in enumerate(s['slots'].tolist()):
                for layer in range(c['layers']):
                    result[layer, 0, x // page, :, x % page] = s['k'][layer][i].double()
                    result[layer, 1, x // page, :, x % page] = s['v'][layer][i].double()
            return [result]
        slots, at = [], 0
        for row in range(c['n']):
            give(row)
        for row, count in enumerate(s['counts'].tolist()):
            for j in range(pages_of(count)):
                table[row][j] = take()
            lens[row] = count
            for j in range(pages_of(count)):
                m = min(page, count - j * page)
                for layer in range(c['layers']):
                    result[layer, 0, table[row][j], :, :m] = s['k'][layer][at:at + m].double().transpose(0, 1)
                    result[layer, 1, table[row][j], :, :m] = s['v'][layer][at:at + m].double().transpose(0, 1)
                at += m
            slots += [place(row, t)[0] * page + place(row, t)[1] for t in range(count)]
        return [result] + [torch.tensor(x, dtype=torch.int32) for x in (table, lens, refs, slots)]
    if c['op'] in ('fork', 'copy'):
        for row in s['dst'].tolist():
            give(row)
        for src, dst in zip(s['src'].tolist(), s['dst'].tolist()):
            lens[dst] = lens[src]
            for j in range(pages_of(lens[src])):
                m = min(page, lens[src] - j * page)
                if c['op'] == 'fork' and m == page:
                    table[dst][j] = table[src][j]
                    refs[table[src][j]] += 1
                else:
                    table[dst][j] = take()
                    result[:, :, table[dst][j], :, :m] = result[:, :, table[src][j], :, :m]
        return [result] + [torch.tensor(x, dtype=torch.int32) for x in (table, lens, refs)]
    moved, counts = s['into']['kv'].double(), [0] * s['into']['refs'].numel()
    new = {}
    for p, held in enumerate(refs):
        if held > 0:
            new[p] = len(new)
            counts[new[p]] = held
    src = torch.tensor(list(new), device=DEV)
    moved[:, :, :len(new)] = result[:, :, src]
    return [moved] + [torch.tensor(x, dtype=torch.int32) for x in ([[new.get(p, -1) for p in row] for row in table], lens, counts)]


def _exact_packed(c, s):
    out = torch.zeros(s['q'].shape, dtype=torch.float64, device=DEV)
    start, group = 0, c['hq'] // c['hkv']
    for length in s['lengths']:
        end = start + length
        for h in range(c['hq']):
            k, v = s['k'][start:end, h // group].double(), s['v'][start:end, h // group].double()
            for a in range(0, length, 4096):
                b = min(length, a + 4096)
                weight = (s['q'][start + a:start + b, h].double() @ k[:b].T.contiguous()) / math.sqrt(c['hd'])
                weight += torch.full_like(weight, float('-inf')).triu(a + 1)
                out[start + a:start + b, h] = torch.softmax(weight, dim=1) @ v[:b]
        start = end
    return out


def _exact_attend(c, s):
    out = torch.zeros(s['q'].shape, dtype=torch.float64, device=DEV)
    group = c['hq'] // c['hkv']
    lens, table = s['lens'].tolist(), s['table']
    for i, row in enumerate(s['rows'].tolist()):
        length = lens[row]
        if not length:
            continue
        mine = table[row, :_pages(length, c['page'])].long()
        k, v = (s['kv'][0, x][mine].double().transpose(0, 1).flatten(1, 2)[:, :length] for x in (0, 1))      # (hkv, length, hd)
        q = s['q'][i].double().view(c['hkv'], group, c['hd'])
        for h in range(c['hkv']):
            out[i, h * group:(h + 1) * group] = torch.softmax(q[h] @ k[h].T.contiguous() / math.sqrt(c['hd']), dim=1) @ v[h]
    return out
