"""A cache in pages that many sequences share, and attention over it and over an encoder's states, as cases that can be timed and
compared.

  attend  kernels.paged_attend: grouped-query attention of a chunk of new tokens (one up to a long prompt) of a batch of sequences over
          the pages that their tables name
  append  kernels.paged_append: new key / value rows into those pages
  pages   kernels.pages_fork, pages_take, pages_trim, pages_compact: sequences forked (shared pages, copied when they are written),
          cut back, and a pool's pages moved together
  cross   kernels.cross_attend: attention to an encoder's states of another length, with lengths and a mask of their keys

The plain forms are elementary torch operations in 32 bits on the same tensors. Layouts that are part of the interface: a layer's pool is
k, v (pages, KV heads, rows of a page, D); table (sequences, most pages of one) int32 names a sequence's pages in order, -1 behind them;
lens int32 are the rows held, refs int32 the users of each page, bit p % 32 of word p / 32 of free says that page p has none.
"""
import math
import random

import torch

own = False
DEV = 'cuda'
DT = dict(bf16=torch.bfloat16, f16=torch.float16)


def listed():
    return [
        # one generated token behind the prefix of one observation: latency only
        dict(name='attend_token', kind='attend', B=1, M=1, P=968, Hq=8, Hk=1, D=256, T=64, causal=True, ragged=False, dtype='bf16'),
        # a decode step of a batch of sequences of several thousand rows, grouped heads
        dict(name='attend_batch', kind='attend', B=32, M=1, P=8192, Hq=16, Hk=8, D=128, T=64, causal=True, ragged=True, dtype='bf16'),
        # generated tokens behind very long contexts
        dict(name='attend_long', kind='attend', B=2, M=1, P=131000, Hq=8, Hk=1, D=256, T=256, causal=True, ragged=True, dtype='f16'),
        # the action tokens of several robots: every token sees its prefix and all action tokens
        dict(name='attend_actions', kind='attend', B=8, M=50, P=800, Hq=8, Hk=1, D=256, T=16, causal=False, ragged=False, dtype='bf16'),
        # parts of long prompts behind the parts before them
        dict(name='attend_chunk', kind='attend', B=4, M=2048, P=4096, Hq=16, Hk=8, D=128, T=64, causal=True, ragged=True, dtype='bf16'),
        # a decode step of a batch: one row each into a page that is partly filled
        dict(name='append_step', kind='append', B=64, M=1, P=1000, H=8, D=128, T=64, ragged=True, dtype='bf16'),
        # prompts of different lengths behind what the pages hold already
        dict(name='append_prompt', kind='append', B=6, M=2000, P=777, H=8, D=128, T=64, ragged=True, dtype='bf16'),
        # eight continuations of each of two prompts tried for a few rows and given back: shared pages, the last one copied
        dict(name='pages_fork', kind='fork', S=2, n=8, P=968, M=10, L=18, H=1, D=256, T=64, dtype='bf16'),
        # half of 48 sequences have ended: the others' pages move together, in all layers
        dict(name='pages_compact', kind='compact', S=48, P=1000, L=18, H=1, D=256, T=64, dtype='bf16'),
        # action tokens to the states of one observation, many narrow heads
        dict(name='cross_token', kind='cross', B=1, M=50, N=600, Hq=32, Hk=32, D=48, ragged=False, mask=False, dtype='bf16'),
        # the same for a batch of robots whose cameras and texts differ
        dict(name='cross_batch', kind='cross', B=16, M=129, N=1500, Hq=32, Hk=32, D=64, ragged=True, mask=True, dtype='f16'),
        # a long sequence to a long one
        dict(name='cross_long', kind='cross', B=2, M=4096, N=4096, Hq=16, Hk=16, D=128, ragged=True, mask=False, dtype='bf16'),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(('attend', 'attend', 'attend', 'cross', 'cross', 'append', 'fork', 'compact'))
    T = rng.choice((16, 32, 64, 64, 128, 256))
    dtype = rng.choice(('bf16', 'f16'))
    if kind == 'append':
        H, D = rng.choice(((1, 256), (1, 128), (2, 64), (4, 128), (8, 128), (8, 80), (16, 64)))
        B = _log_int(rng, 1, 64)
        return dict(kind='append', B=B, M=_log_int(rng, 1, 12000 // B), P=_log_int(rng, 1, 2000) - 1, H=H, D=D, T=T, ragged=rng.random() < 0.6, dtype=dtype)
    if kind in ('fork', 'compact'):
        H, D = rng.choice(((1, 256), (1, 128), (8, 128), (8, 64)))
        L = rng.choice((1, 4, 18)) if H == 1 else rng.choice((1, 2))
        P = _log_int(rng, 1, 1000)
        if kind == 'fork':
            return dict(kind='fork', S=rng.randint(1, 8), n=rng.randint(1, 8), P=P, M=_log_int(rng, 1, 100), L=L, H=H, D=D, T=T, dtype=dtype)
        return dict(kind='compact', S=_log_int(rng, 2, 48), P=P, L=L, H=H, D=D, T=T, dtype=dtype)
    most = {c['name']: work(c)['flops'] for c in listed()}
    while True:
        M = 1 if rng.random() < 0.4 else _log_int(rng, 1, 3000)
        B = _log_int(rng, 1, 32)
        if kind == 'attend':
            Hk, G, D = rng.choice(((1, 8, 256), (1, 5, 256), (8, 2, 128), (2, 7, 128), (4, 4, 64), (16, 1, 64), (1, 16, 128), (8, 4, 96)))
            case = dict(kind='attend', B=B, M=M, P=_log_int(rng, 1, 130000) - 1, Hq=Hk * G, Hk=Hk, D=D, T=T, causal=rng.random() < 0.8,
                        ragged=rng.random() < 0.6, dtype=dtype)
            keys = case['P'] + M
        else:
            Hk, G, D = rng.choice(((32, 1, 48), (32, 1, 64), (16, 1, 72), (16, 1, 128), (8, 2, 128), (8, 1, 256), (1, 8, 256), (20, 1, 80)))
            keys = _log_int(rng, 1, 20000)
            case = dict(kind='cross', B=B, M=M, N=keys, Hq=Hk * G, Hk=Hk, D=D, ragged=rng.random() < 0.5, mask=rng.random() < 0.5, dtype=dtype)
        w = work(case)
        if w['flops'] <= most['attend_chunk'] and w['bytes'] <= 5e8 and B * M * case['Hq'] * keys <= 8e8:
            return case


def _ragged(n, B, ragged):
    """The first sequence's n rows and, ragged, the others' down to half of it."""
    return [n - (b * n) // (2 * B) if ragged else n for b in range(B)]


def _counts(case):
    """Rows held before and new rows of a batch's sequences."""
    return _ragged(case['P'], case['B'], case['ragged']), _ragged(case['M'], case['B'], case['ragged'])


def _hidden(n, b):
    """Keys lo .. hi - 1 of a sequence of n are masked: a camera's that is not there."""
    return (n * (b % 5)) // 7, (n * (b % 5)) // 7 + (n * (1 + b % 3)) // 8


def _seen(case):
    """Keys that the rows of each sequence see in a cross case."""
    lens = _ragged(case['N'], case['B'], case['ragged'])
    return [n - (min(_hidden(n, b)[1], n) - _hidden(n, b)[0] if case['mask'] else 0) for b, n in enumerate(lens)]


def _pages(n, T):
    return (n + T - 1) // T


# ---------------------------------------------------------------------------------------------------------------- prepare
def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _bookkeeping(tables, lens, most, pages):
    """One buffer of a pool's bookkeeping (table, lens, refs, free, lack one after the other) for sequences that hold these pages."""
    B, words = len(tables), (pages + 31) // 32
    refs, table = [0] * pages, []
    for t in tables:
        table += t + [-1] * (most - len(t))
        for p in t:
            refs[p] += 1
    free = [0] * words
    for p, r in enumerate(refs):
        if r == 0:
            free[p // 32] |= 1 << (p % 32)
    free = [w - (1 << 32) if w >= 1 << 31 else w for w in free]
    return _ints(table + list(lens) + refs + free + [0]), (B, most, pages, words)


def _views(flat, sizes):
    B, most, pages, words = sizes
    table, lens, refs, free, lack = flat.split([B * most, B, pages, words, 1])
    return dict(table=table.view(B, most), lens=lens, refs=refs, free=free, lack=lack)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    pick = random.Random(seed)
    dt = DT[case['dtype']]
    st = dict(case=case)

    def normal(*shape, by=1.0):
        return (torch.randn(*shape, generator=g, device=DEV) * by).to(dt)

    if case['kind'] == 'cross':
        B, M, N, D = case['B'], case['M'], case['N'], case['D']
        st['q'] = normal(B * M, case['Hq'], D, by=2.0)
        kv = normal(B, N, 2, case['Hk'], D)                       # the states' keys and values come side by side from one product
        st['k'], st['v'] = kv[:, :, 0], kv[:, :, 1]
        lens = _ragged(N, B, case['ragged'])
        st['lens'] = _ints(lens)
        st['mask'] = None
        if case['mask']:
            lo, hi = (torch.tensor(x, device=DEV)[:, None] for x in zip(*[_hidden(n, b) for b, n in enumerate(lens)]))
            j = torch.arange(N, device=DEV)
            st['mask'] = (j < lo) | (j >= hi)
        return st
    T = case['T']
    H, D = case.get('H', case.get('Hk')), case['D']
    if case['kind'] in ('attend', 'append'):
        start, new = _counts(case)
        lens = [s + n for s, n in zip(start, new)]
        held = [_pages(n, T) for n in lens]
        pages = sum(held) + 3
        order = pick.sample(range(pages), sum(held))              # a pool in use: a sequence's pages lie anywhere
        at = [sum(held[:b]) for b in range(len(held) + 1)]
        flat, sizes = _bookkeeping([order[at[b]:at[b + 1]] for b in range(len(held))], lens, max(held) + 1, pages)
        cu = [sum(new[:b]) for b in range(len(new) + 1)]
        st.update(_views(flat, sizes), start=_ints(start), cu=_ints(cu), most=max(new), longest=max(lens))
        st['pk'], st['pv'] = normal(pages, H, T, D), normal(pages, H, T, D)
        if case['kind'] == 'append':
            st['k'], st['v'] = normal(cu[-1], H, D), normal(cu[-1], H, D)
        else:
            st['q'] = normal(cu[-1], case['Hq'], D, by=2.0)
        return st
    L, P, S = case['L'], case['P'], case['S']
    if case['kind'] == 'fork':
        n, each = case['n'], _pages(P, T)
        pages = S * each + S * n * (_pages(P + case['M'], T) - P // T) + 2
        order = pick.sample(range(pages), S * each)
        tables = [order[s * each:(s + 1) * each] for s in range(S)] + [[] for _ in range(S * n)]
        flat, sizes = _bookkeeping(tables, [P] * S + [0] * (S * n), _pages(P + case['M'], T), pages)
        st.update(src=_ints([s for s in range(S) for _ in range(n)]), dst=_ints(range(S, S + S * n)),
                  new=_ints([0] * S + [case['M']] * (S * n)), keep=_ints([P] * S + [0] * (S * n)))
    else:
        each = _pages(P, T)
        pages = S * each
        used = _in_use(case)
        pick.shuffle(used)
        tables = [used[s * each:(s + 1) * each] for s in range(S // 2)]
        flat, sizes = _bookkeeping(tables + [[] for _ in range(S - S // 2)], [P] * (S // 2) + [0] * (S - S // 2), each, pages)
    st.update(_views(flat, sizes), flat=flat, saved=flat.clone())
    st['pk'], st['pv'] = normal(L, pages, H, T, D), normal(L, pages, H, T, D)
    return st


def _in_use(case):
    """The pages still held in a compact case: S sequences grew in turn, and those with an odd number have ended."""
    S, each = case['S'], _pages(case['P'], case['T'])
    return [p for p in range(S * each) if p % S < 2 * (S // 2) and p % S % 2 == 0]


# -------------------------------------------------------------------------------------------------------------------- run
def run(st):
    case = st['case']
    kind = case['kind']
    if own:
        from yanlongvla_amd import kernels
        if kind == 'cross':
            return kernels.cross_attend(st['q'], st['k'], st['v'], lens=st['lens'], mask=st['mask'])
        pool = kernels.Pages(st['pk'], st['pv'])
        if kind == 'attend':
            return kernels.paged_attend(st['q'], pool, st['table'], st['lens'], causal=case['causal'], cu=st['cu'], most=st['most'],
                                        keys=st['longest'])
        if kind == 'append':
            kernels.paged_append(pool, st['k'], st['v'], st['table'], st['lens'], st['start'], cu=st['cu'], most=st['most'])
            return dict(k=st['pk'], v=st['pv'])
        st['flat'].copy_(st['saved'])
        book = kernels.PageTable(st['table'], st['lens'], st['refs'], st['free'], st['lack'], case['T'])
        if kind == 'compact':
            kernels.pages_compact(book, pool)
            return dict(table=st['table'], refs=st['refs'], k=st['pk'], v=st['pv'])
        kernels.pages_fork(book, st['src'], st['dst'])
        start = kernels.pages_take(book, pool, st['new'])
        tried = st['table'].clone()
        kernels.pages_trim(book, st['keep'])
        return dict(start=start, tried=tried, table=st['table'], lens=st['lens'], refs=st['refs'], k=st['pk'], v=st['pv'])
    if kind == 'cross':
        return _cross(st)
    if kind == 'attend':
        return _attend(st)
    if kind == 'append':
        return _append(st)
    st['flat'].copy_(st['saved'])
    if kind == 'compact':
        _compact(st)
        return dict(table=st['table'], refs=st['refs'], k=st['pk'], v=st['pv'])
    _fork(st)
    start = _take(st)
    tried = st['table'].clone()
    _trim(st)
    return dict(start=start, tried=tried, table=st['table'], lens=st['lens'], refs=st['refs'], k=st['pk'], v=st['pv'])


def _softmax(q, k, v, seen):
    """q (B, H, R, D), k and v (B, H, N, D) in FP32, seen (B, 1, R or 1, N): the means of v, zeros for a row that sees nothing."""
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()) / math.sqrt(q.shape[-1])
    s = s.masked_fill(~seen, float('-inf'))
    p = (s - s.amax(-1, keepdim=True).clamp(min=-1e30)).exp()
    return torch.matmul(p, v) / p.sum(-1, keepdim=True).clamp(min=1e-30)


def _cross(st):
    case = st['case']
    B, M, Hk, D = case['B'], case['M'], case['Hk'], case['D']
    G = case['Hq'] // Hk
    q = st['q'].float().view(B, M, Hk, G, D).permute(0, 2, 1, 3, 4).reshape(B, Hk, M * G, D)
    k, v = (t.float().transpose(1, 2).contiguous() for t in (st['k'], st['v']))
    seen = torch.arange(case['N'], device=DEV) < st['lens'][:, None]
    if st['mask'] is not None:
        seen = seen & st['mask']
    o = _softmax(q, k, v, seen[:, None, None])
    return o.view(B, Hk, M, G, D).permute(0, 2, 1, 3, 4).reshape(B * M, case['Hq'], D).to(st['q'].dtype)


def _attend(st):
    case, table, most = st['case'], st['table'].long(), st['most']
    B, Hk, D = case['B'], case['Hk'], case['D']
    G = case['Hq'] // Hk
    k, v = (t[table.clamp(min=0)].transpose(1, 2).reshape(B, Hk, -1, D).float() for t in (st['pk'], st['pv']))
    rows = torch.arange(st['q'].shape[0], device=DEV)
    b = torch.searchsorted(st['cu'].long(), rows, right=True) - 1
    i = rows - st['cu'].long()[b]
    q = torch.zeros(B, most, case['Hq'], D, device=DEV)
    q[b, i] = st['q'].float()
    q = q.view(B, most, Hk, G, D).permute(0, 2, 1, 3, 4).reshape(B, Hk, most * G, D)
    lens, count = st['lens'].long()[:, None], st['cu'].long().diff()[:, None]
    end = torch.minimum(lens, lens - count + 1 + torch.arange(most, device=DEV)) if case['causal'] else lens.expand(B, most)
    seen = torch.arange(k.shape[2], device=DEV) < end.repeat_interleave(G, 1)[:, None, :, None]
    o = _softmax(q, k, v, seen)
    o = o.view(B, Hk, most, G, D).permute(0, 2, 1, 3, 4).reshape(B, most, case['Hq'], D)
    return o[b, i].to(st['q'].dtype)


def _append(st):
    T = st['case']['T']
    rows = torch.arange(st['k'].shape[0], device=DEV)
    b = torch.searchsorted(st['cu'].long(), rows, right=True) - 1
    at = st['start'].long()[b] + rows - st['cu'].long()[b]
    page = st['table'].long()[b, at // T]
    st['pk'][page, :, at % T] = st['k']
    st['pv'][page, :, at % T] = st['v']
    return dict(k=st['pk'], v=st['pv'])


def _fork(st):
    src, dst, table, refs = st['src'].long(), st['dst'].long(), st['table'], st['refs']
    table[dst] = table[src]
    st['lens'][dst] = st['lens'][src]
    taken = table[dst]
    refs.index_add_(0, taken.clamp(min=0).long().flatten(), (taken >= 0).int().flatten())


def _take(st):
    T, table, lens, refs = st['case']['T'], st['table'], st['lens'], st['refs']
    start, new = lens.clone(), st['new']
    b = torch.arange(lens.shape[0], device=DEV)
    have, want = (start + T - 1) // T, (start + new + T - 1) // T
    last = table[b, (have - 1).clamp(min=0).long()]
    copied = (new > 0) & (start % T != 0) & (refs[last.clamp(min=0).long()] > 1)
    need = want - have + copied.int()
    order = torch.argsort((refs > 0).int(), stable=True)          # the free pages from the lowest on
    first = need.cumsum(0) - need                                  # (the cases have as many as they need)
    at = first[:, None] + torch.arange(table.shape[1], device=DEV)
    got = order[at.clamp(max=order.shape[0] - 1)].int()           # (B, most): the pages that a sequence may take, in order
    for to, frm in zip(got[copied, 0].long(), last[copied].long()):
        st['pk'][:, to] = st['pk'][:, frm]
        st['pv'][:, to] = st['pv'][:, frm]
    refs.index_add_(0, last[copied].long(), torch.full_like(last[copied], -1))
    slot = torch.arange(table.shape[1], device=DEV)[None] - (have - copied.int())[:, None]
    put = (slot >= 0) & (slot < need[:, None])
    table.copy_(torch.where(put, got.gather(1, slot.clamp(0, table.shape[1] - 1)), table))
    refs.index_add_(0, table[put].long(), torch.ones_like(table[put]))
    lens.add_(new)
    return start


def _trim(st):
    T, table, lens, keep = st['case']['T'], st['table'], st['lens'], st['keep']
    end = torch.minimum(lens, keep)
    drop = (torch.arange(table.shape[1], device=DEV) >= ((end + T - 1) // T)[:, None]) & (table >= 0)
    st['refs'].index_add_(0, table[drop].long(), torch.full_like(table[drop], -1))
    table.masked_fill_(drop, -1)
    lens.copy_(end)


def _compact(st):
    table, refs = st['table'], st['refs']
    used = refs > 0
    p = torch.arange(refs.shape[0], device=DEV)
    U = used.sum()
    src, dst = (used & (p >= U)).nonzero()[:, 0], (~used & (p < U)).nonzero()[:, 0]
    for t in (st['pk'], st['pv']):
        t[:, dst] = t[:, src]
    to = p.int()
    to[src] = dst.int()
    table.copy_(torch.where(table >= 0, to[table.clamp(min=0).long()], table))
    refs[dst] = refs[src]
    refs[src] = 0


# ------------------------------------------------------------------------------------------------------------------- work
def work(case):
    """Every input read once, every output written once: of the pages and states the rows that are seen, of a pool's pages those that
    move or are copied, read and written."""
    if case['kind'] in ('fork', 'compact'):
        T = case['T']
        page = 2 * case['L'] * case['H'] * T * case['D'] * 2
        held = _pages(case['P'], T)
        if case['kind'] == 'fork':
            n = case['S'] * case['n']
            copied = n if case['P'] % T else 0
            return dict(bytes=2 * copied * page + 4 * n * (4 * held + 8), flops=n * held)
        used = _in_use(case)
        moved = sum(p >= len(used) for p in used)
        return dict(bytes=2 * moved * page + 4 * (3 * len(used) + case['S'] * held), flops=case['S'] * held)
    B, D = case['B'], case['D']
    if case['kind'] == 'cross':
        rows, seen = case['M'], _seen(case)
        return dict(bytes=2 * D * (2 * sum(seen) * case['Hk'] + 2 * B * rows * case['Hq']) + (B * case['N'] if case['mask'] else 0),
                    flops=4 * rows * sum(seen) * case['Hq'] * D)
    start, new = _counts(case)
    if case['kind'] == 'append':
        return dict(bytes=2 * 2 * 2 * sum(new) * case['H'] * D + 8 * B, flops=sum(new) * case['H'] * D)
    seen = sum(n * (s + n) - (n * (n - 1) // 2 if case['causal'] else 0) for s, n in zip(start, new))
    keys = sum(s + n for s, n in zip(start, new))
    return dict(bytes=2 * D * (2 * keys * case['Hk'] + 2 * sum(new) * case['Hq']) + 4 * keys // case['T'], flops=4 * seen * case['Hq'] * D)


# ------------------------------------------------------------------------------------------ the same results in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    if case['kind'] == 'cross':
        out = torch.zeros(st['q'].shape, dtype=torch.float64, device=DEV)
        M, G = case['M'], case['Hq'] // case['Hk']
        for b, n in enumerate(st['lens'].tolist()):
            on = torch.arange(n, device=DEV) if st['mask'] is None else st['mask'][b, :n].nonzero()[:, 0]
            for h in range(case['Hq'] if len(on) else 0):
                s = st['q'][b * M:(b + 1) * M, h].double() @ st['k'][b, on, h // G].double().t() * case['D'] ** -0.5
                out[b * M:(b + 1) * M, h] = torch.softmax(s, 1) @ st['v'][b, on, h // G].double()
        return out
    T = case['T']
    table, lens = st['table'].tolist(), st['lens'].tolist()
    if case['kind'] == 'attend':
        out = torch.zeros(st['q'].shape, dtype=torch.float64, device=DEV)
        cu, G = st['cu'].tolist(), case['Hq'] // case['Hk']
        for b, n in enumerate(lens):
            m = cu[b + 1] - cu[b]
            for h in range(case['Hk']):
                k, v = (torch.cat([t[p, h] for p in table[b] if p >= 0])[:n].double() for t in (st['pk'], st['pv']))
                for f in range(h * G, h * G + G):
                    s = st['q'][cu[b]:cu[b + 1], f].double() @ k.t() / case['D'] ** 0.5
                    if case['causal']:
                        s += torch.full((m, n), -math.inf, dtype=torch.float64, device=DEV).triu(n - m + 1)
                    out[cu[b]:cu[b + 1], f] = torch.softmax(s, 1) @ v
        return out
    if case['kind'] == 'append':
        cu, start = st['cu'].tolist(), st['start'].tolist()
        out = dict(k=st['pk'].double(), v=st['pv'].double())
        for b in range(case['B']):
            at = start[b]
            while at < lens[b]:                                    # a run of rows that lie in one page
                end = min(lens[b], (at // T + 1) * T)
                for name in 'kv':
                    rows = st[name][cu[b] + at - start[b]:cu[b] + end - start[b]].double()
                    out[name][table[b][at // T], :, at % T:at % T + end - at] = rows.transpose(0, 1)
                at = end
        return out
    refs = st['refs'].tolist()
    pool = dict(k=st['pk'].double(), v=st['pv'].double())
    whole = lambda x: torch.tensor(x, dtype=torch.float64, device=DEV)              # noqa: E731
    if case['kind'] == 'compact':
        high = [p for p in range(len(refs)) if refs[p] and p >= sum(r > 0 for r in refs)]
        low = [p for p in range(len(refs)) if not refs[p]][:len(high)]
        for a, z in zip(high, low):
            for t in pool.values():
                t[:, z] = t[:, a]
            refs[a], refs[z] = 0, refs[a]
        to = dict(zip(high, low))
        return dict(table=whole([[to.get(p, p) for p in r] for r in table]), refs=whole(refs), **pool)
    new, keep = st['new'].tolist(), st['keep'].tolist()
    for s, d in zip(st['src'].tolist(), st['dst'].tolist()):
        table[d], lens[d] = list(table[s]), lens[s]
        for p in table[d]:
            if p >= 0:
                refs[p] += 1
    start = list(lens)
    spare = [p for p in range(len(refs)) if not refs[p]]
    shared = [r > 1 for r in refs]
    for b in range(len(lens)):
        have = _pages(lens[b], T)
        if new[b] and lens[b] % T and shared[table[b][have - 1]]:
            a, z = table[b][have - 1], spare.pop(0)
            for t in pool.values():
                t[:, z] = t[:, a]
            table[b][have - 1] = z
            refs[a] -= 1
            refs[z] += 1
        lens[b] += new[b]
        for j in range(have, _pages(lens[b], T)):
            table[b][j] = spare.pop(0)
            refs[table[b][j]] += 1
    tried = [list(r) for r in table]
    for b in range(len(lens)):
        lens[b] = min(lens[b], keep[b])
        for j in range(_pages(lens[b], T), len(table[b])):
            if table[b][j] >= 0:
                refs[table[b][j]] -= 1
            table[b][j] = -1
    return dict(start=whole(start), tried=whole(tried), table=whole(table), lens=whole(lens), refs=whole(refs), **pool)
