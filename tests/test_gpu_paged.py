"""GPU tests of attention over a cache in pages and of cross attention against 64 bits, and of rows into pages. Sizes and masks where it can go
wrong: one row, no rows, lengths at and around a page's and a tile's end, ragged batches, grouped heads, head sizes that fill no tile, rows that
see nothing, rows of no sequence, keys and values that are not finite where no row sees them, views, offsets past 32 bits, other streams,
replays.

Tolerance of an output, elementwise: half a step of its type (eps / 2 relative), plus what the rounded probabilities and their sum change: each
is off by at most d of itself (half a step: BF16 2^-8, FP16 2^-11), so a weight by 2 d and an output by 2 d sum p |v|. A score is a sum of
D products in FP32, off by at most e = D 2^-24 scale sum |q k|, and a weight with its sum by 2 e of itself; 1e-5 more for the exponentials
(2^-22) and the sum of up to 64 terms a lane and tile."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda'
BF, HF = torch.bfloat16, torch.float16


@pytest.fixture(scope='module', autouse=True)
def _lib():
    from yanlongvla_amd import _lib
    _lib.lib()
    torch.cuda.init()


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def rand(*shape, seed, dt=BF, by=1.0):
    return (torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV) * by).to(dt)


def formula(q, k, v, seen, scale=None):
    """q (m, D), k and v (n, D), seen (m, n) of one head: outputs and sum p |v| in 64 bits; keys that a row does not see do not count at all."""
    q, k, v = q.double(), k.double(), v.double()
    s = (q @ k.t()) * (scale if scale is not None else 1 / math.sqrt(q.shape[1]))
    s = torch.where(seen, s, torch.full_like(s, -math.inf))
    top = s.amax(1, keepdim=True)
    p = torch.where(seen, torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top)), torch.zeros_like(s))
    l = p.sum(1, keepdim=True)
    p = torch.where(l > 0, p / l, p)
    finite = torch.where(v.isfinite(), v, torch.zeros_like(v))
    o = p @ finite
    for j in (~v.isfinite()).any(1).nonzero()[:, 0].tolist():              # what is not finite reaches the rows that see it
        o = o + torch.where(seen[:, j:j + 1], torch.where(v[j].isfinite(), 0.0, v[j]), torch.zeros_like(v[j]))
    e = q.shape[1] * 2.0 ** -24 * (scale if scale is not None else 1 / math.sqrt(q.shape[1])) * torch.where(seen, q.abs() @ k.abs().t(), 0.0)
    return o, p @ finite.abs(), torch.where(e.isfinite(), e, torch.zeros_like(e)).amax(1, keepdim=True)


def close(got, o, a, e, dt):
    d = torch.finfo(dt).eps / 2
    nan = o.isnan()
    assert torch.equal(got.isnan(), nan)
    inf = o.isinf()
    assert torch.equal(got.double()[inf], o[inf])
    ok = ~(nan | inf)
    err = (got.double() - o).abs()[ok]
    tol = (torch.finfo(dt).eps / 2 * o.abs() + (2 * d + 2 * e + 1e-5) * a)[ok] + 1e-7
    assert (err <= tol).all(), float((err / tol).max())


class Pool:
    """A pool whose pages lie in random order, sequences of these lengths, and what stands at no sequence's rows: NaN."""

    def __init__(self, lens, H, D, T, dt=BF, seed=0, extra=3, fill=math.nan, room=1):
        from yanlongvla_amd import kernels as K
        held = [(n + T - 1) // T for n in lens]
        pages = sum(held) + extra
        g = torch.Generator().manual_seed(seed)
        order = torch.randperm(pages, generator=g).tolist()
        N = max(held) + room
        self.table = torch.full((len(lens), N), -1, dtype=torch.int32)
        self.pages = K.Pages(*(torch.full((pages, H, T, D), fill, dtype=dt, device=DEV) for _ in range(2)))
        self.k, self.v, at = [], [], 0
        for b, n in enumerate(lens):
            self.table[b, :held[b]] = torch.tensor(order[at:at + held[b]], dtype=torch.int32)
            k, v = rand(n, H, D, seed=seed + 10 * b + 1, dt=dt), rand(n, H, D, seed=seed + 10 * b + 2, dt=dt)
            for j in range(held[b]):
                p, rows = order[at + j], min(T, n - j * T)
                self.pages.k[p, :, :rows] = k[j * T:j * T + rows].transpose(0, 1)
                self.pages.v[p, :, :rows] = v[j * T:j * T + rows].transpose(0, 1)
            at += held[b]
            self.k.append(k)
            self.v.append(v)
        self.table = self.table.to(DEV)
        self.lens = ints(lens)

    def set_value(self, b, j, value, T):
        """Value row j of sequence b, in the pool too."""
        self.v[b][j] = value
        self.pages.v[int(self.table[b, j // T]), :, j % T] = value


def check(got, q, pool, lens, new, causal, dt, scale=None):
    at = 0
    H = pool.pages.k.shape[1]
    G = q.shape[1] // H
    for b, (n, m) in enumerate(zip(lens, new)):
        i, j = torch.arange(m, device=DEV)[:, None], torch.arange(n, device=DEV)[None]
        seen = (j <= n - m + i) if causal else torch.ones(m, n, dtype=torch.bool, device=DEV)
        for h in range(q.shape[1] if m else 0):
            close(got[at:at + m, h], *formula(q[at:at + m, h], pool.k[b][:, h // G], pool.v[b][:, h // G], seen, scale), dt)
        at += m


SIZES = [  # lens, new rows, Hq, H, D, T
    ([1], [1], 1, 1, 64, 16), ([17], [1], 8, 1, 256, 16), ([64, 65, 63], [1, 1, 1], 16, 8, 128, 64), ([968], [1], 8, 1, 256, 64),
    ([300, 1, 129, 31], [1, 1, 1, 1], 6, 2, 96, 32), ([5000, 2], [1, 1], 8, 8, 64, 128), ([40000], [1], 8, 1, 128, 256), ([33], [3], 16, 1, 48, 16),
    ([128], [128], 4, 4, 128, 64), ([700], [200], 8, 2, 128, 32), ([257, 64, 300], [100, 64, 3], 8, 1, 256, 16), ([1500], [1000], 3, 3, 72, 64),
    ([129], [129], 5, 1, 8, 16), ([500, 499], [77, 20], 14, 2, 80, 64), ([850, 850], [50, 50], 8, 1, 256, 64), ([400], [129], 2, 2, 200, 16),
    ([70, 0, 200], [33, 0, 34], 4, 4, 64, 16), ([6200], [2048], 2, 1, 128, 64), ([90], [9], 14, 7, 16, 32),
]


@pytest.mark.parametrize('lens,new,Hq,H,D,T', SIZES)
@pytest.mark.parametrize('causal', [True, False])
@pytest.mark.parametrize('dt', [BF, HF])
def test_paged_attend(lens, new, Hq, H, D, T, causal, dt):
    from yanlongvla_amd import kernels as K
    pool = Pool(lens, H, D, T, dt, seed=D + T)
    q = rand(sum(new), Hq, D, seed=7, dt=dt, by=2.0)
    cu = ints([sum(new[:b]) for b in range(len(new) + 1)])
    got = K.paged_attend(q, pool.pages, pool.table, pool.lens, causal=causal, cu=cu, most=max(new))
    check(got, q, pool, lens, new, causal, dt)
    for keys in (0, max(lens), 10 ** 6):                                     # the split changes the order of sums alone
        check(K.paged_attend(q, pool.pages, pool.table, pool.lens, causal=causal, cu=cu, most=max(new), keys=keys), q, pool, lens, new, causal, dt)
    if len(set(new)) == 1:                                                   # equal shares: the same bits
        assert torch.equal(K.paged_attend(q, pool.pages, pool.table, pool.lens, causal=causal), got)


@pytest.mark.parametrize('scale', [0.0, 1e-3, 1.0, 30.0])
@pytest.mark.parametrize('M', [1, 70])
def test_score_scales(scale, M):
    """Means at 0, one key at 30."""
    from yanlongvla_amd import kernels as K
    lens, dt = [300], HF
    pool = Pool(lens, 2, 64, 64, dt, seed=3)
    q = rand(M, 4, 64, seed=8, dt=dt, by=2.0)
    got = K.paged_attend(q, pool.pages, pool.table, pool.lens, scale=scale)
    check(got, q, pool, lens, [M], True, dt, scale)


@pytest.mark.parametrize('M,G', [(7, 1), (40, 1), (5, 3), (200, 2)])
def test_rows_that_see_nothing_and_rows_of_no_sequence(M, G):
    """More new rows than a sequence holds: the first of them see nothing and are zeros. Rows before, between and behind the sequences stay."""
    from yanlongvla_amd import kernels as K
    H, D, T, dt = 2, 64, 16, BF
    lens = [3, M]
    pool = Pool(lens, H, D, T, dt, seed=1)
    rows = 2 + 2 * M + 5
    q = rand(rows, H * G, D, seed=2, dt=dt)
    o = torch.full_like(q, 7.0)
    cu = ints([2, 2 + M, 2 + 2 * M])
    K.paged_attend(q, pool.pages, pool.table, pool.lens, o=o, causal=True, cu=cu, most=M)
    check(o[2:2 + 2 * M], q[2:2 + 2 * M], pool, lens, [M, M], True, dt)
    assert (o[2:2 + M - 3] == 0).all()
    assert (o[:2] == 7).all() and (o[2 + 2 * M:] == 7).all()
    K.paged_attend(q, pool.pages, pool.table, ints([0, -5]), o=o, causal=False, cu=cu, most=M)   # nothing at all
    assert (o[2:2 + 2 * M] == 0).all() and (o[:2] == 7).all()
    part = torch.full_like(q, 7.0)                                           # rows of a sequence past `most`
    K.paged_attend(q, pool.pages, pool.table, pool.lens, o=part, causal=True, cu=cu, most=M - 2)
    assert (part[2 + M - 2:2 + M] == 7).all() and torch.equal(part[2 + M:2 + 2 * M - 2], K.paged_attend(q, pool.pages, pool.table, pool.lens, cu=cu, most=M)[2 + M:2 + 2 * M - 2])


@pytest.mark.parametrize('value', [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize('M,Hq,H,D', [(4, 2, 2, 64), (16, 1, 1, 128), (90, 2, 1, 128), (300, 4, 2, 64), (70, 2, 2, 256), (150, 1, 1, 96)])
@pytest.mark.parametrize('dt', [BF, HF])
def test_later_values_that_are_not_finite(value, M, Hq, H, D, dt):
    """A value row that is not finite reaches the rows that see it, and no row before it."""
    from yanlongvla_amd import kernels as K
    lens, T = [M + 37], 16
    pool = Pool(lens, H, D, T, dt, seed=5)
    for j in (37 + M // 2, 37 + M - 1):
        pool.set_value(0, j, value, T)
    q = rand(M, Hq, D, seed=6, dt=dt)
    got = K.paged_attend(q, pool.pages, pool.table, pool.lens)
    check(got, q, pool, lens, [M], True, dt)
    assert got[:M // 2].isfinite().all() and not got[M // 2:].isfinite().any()


@pytest.mark.parametrize('M', [1, 100])
def test_keys_that_are_not_finite(M):
    """NaN among the keys a row sees makes the row NaN; a key that makes every score of a row -inf, too; -inf of some scores takes those keys out."""
    from yanlongvla_amd import kernels as K
    H, D, T = 1, 64, 64
    pool = Pool([200], H, D, T, BF, seed=5)
    q = rand(M, 2, D, seed=6).abs() + 0.1
    pool.pages.k[int(pool.table[0, 0]), :, 3] = -math.inf
    pool.k[0][3] = -math.inf
    got = K.paged_attend(q, pool.pages, pool.table, pool.lens)
    check(got, q, pool, [200], [M], True, BF)
    pool.pages.k[int(pool.table[0, 1]), :, 5] = math.nan
    assert K.paged_attend(q, pool.pages, pool.table, pool.lens).isnan().all()
    pool.pages.k.fill_(-math.inf)
    assert K.paged_attend(q, pool.pages, pool.table, pool.lens).isnan().all()


def test_views_and_other_layouts():
    """Queries that are a part of a q | k | v row, pools of another order, the pool of a layer among several."""
    from yanlongvla_amd import kernels as K
    lens, Hq, H, D, T = [150, 90], 8, 2, 64, 32
    pool = Pool(lens, H, D, T, seed=4)
    for m in (1, 40):
        qkv = rand(2 * m, Hq + 2 * H, D, seed=m)
        q = qkv[:, :Hq]
        want = K.paged_attend(q.contiguous(), pool.pages, pool.table, pool.lens)
        assert torch.equal(K.paged_attend(q, pool.pages, pool.table, pool.lens), want)
        swapped = K.Pages(*(t.transpose(1, 2).contiguous().transpose(1, 2) for t in pool.pages))
        assert torch.equal(K.paged_attend(q, swapped, pool.table, pool.lens), want)
        both = torch.stack([torch.stack(list(pool.pages), 1), torch.zeros_like(torch.stack(list(pool.pages), 1))])
        assert torch.equal(K.paged_attend(q, K.Pages(both[0, :, 0], both[0, :, 1]), pool.table, pool.lens), want)


def test_offsets_past_32_bits():
    """A pool of 5 GiB for keys alone: the last pages hold the rows."""
    from yanlongvla_amd import kernels as K
    H, D, T, pages = 8, 128, 64, 40960
    k = torch.zeros(pages, H, T, D, dtype=BF, device=DEV)
    v = torch.zeros(pages, H, T, D, dtype=BF, device=DEV)
    small = Pool([250, 300], H, D, T, seed=9, extra=0)
    n = small.pages.k.shape[0]
    k[-n:], v[-n:] = small.pages.k, small.pages.v
    table = torch.where(small.table >= 0, small.table + (pages - n), small.table)
    for m in (1, 60):
        q = rand(2 * m, 16, D, seed=m)
        assert torch.equal(K.paged_attend(q, K.Pages(k, v), table, small.lens), K.paged_attend(q, small.pages, small.table, small.lens))
    new = rand(2, H, D, seed=3)
    K.paged_append(K.Pages(k, v), new, new, table, small.lens, small.lens - 1)
    at = [int(table[b, (n_ - 1) // T]) for b, n_ in enumerate((250, 300))]
    for b, n_ in enumerate((250, 300)):
        assert torch.equal(k[at[b], :, (n_ - 1) % T], new[b]) and torch.equal(v[at[b], :, (n_ - 1) % T], new[b])


@pytest.mark.parametrize('H,D,T,dt', [(1, 256, 64, BF), (8, 128, 16, HF), (3, 72, 32, BF), (2, 8, 128, HF)])
@pytest.mark.parametrize('odd', [False, True])
def test_append(H, D, T, dt, odd):
    """Rows behind others, in views whose rows are not aligned too; rows past the length, past the table or of an entry without a page are dropped."""
    from yanlongvla_amd import kernels as K
    lens, start, new = [70, 9, 130, 40], [65, 0, 3, 40], [5, 9, 127, 0]
    pool = Pool(lens, H, D, T, dt, seed=1, fill=0.0)
    wide = rand(sum(new), 2 * H * D + 3, seed=4, dt=dt)
    k, v = (wide[:, o:o + H * D].unflatten(1, (H, D)) for o in ((1, 1 + H * D) if odd else (0, H * D)))
    if not odd:
        k, v = k.contiguous(), v.contiguous()
    cu = ints([sum(new[:b]) for b in range(5)])
    K.paged_append(pool.pages, k, v, pool.table, pool.lens, ints(start), cu, max(new))
    want = [t.clone() for t in pool.pages]
    for b in range(4):
        for i in range(new[b]):
            p = start[b] + i
            assert torch.equal(pool.pages.k[int(pool.table[b, p // T]), :, p % T], k[int(cu[b]) + i])
            assert torch.equal(pool.pages.v[int(pool.table[b, p // T]), :, p % T], v[int(cu[b]) + i])
    bad = pool.table.clone()
    bad[0] = 10 ** 6
    K.paged_append(pool.pages, v, k, bad, ints([70, 9, 3, 40]), ints([65, 10 ** 9, 3, -4]), cu, max(new))
    assert torch.equal(pool.pages.k, want[0]) and torch.equal(pool.pages.v, want[1])


def test_streams_and_replays():
    """Calls on another stream, and a captured step (room, rows, attention) replayed many times with work between, against eager steps."""
    from yanlongvla_amd import kernels as K
    B, H, Hq, D, T, steps = 3, 2, 4, 128, 16, 40
    k, v, q = rand(steps, B, H, D, seed=1), rand(steps, B, H, D, seed=2), rand(steps, B, Hq, D, seed=3)

    def fresh():
        return K.kv_pages(20, H, D, DEV, T), K.page_table(B, 6, 20, DEV, T), torch.ones(B, dtype=torch.int32, device=DEV)

    def step(pool, pt, one, kk, vv, qq):
        start = K.pages_take(pt, pool, one)
        K.paged_append(pool, kk, vv, pt.table, pt.lens, start)
        return K.paged_attend(qq, pool, pt.table, pt.lens)

    pool, pt, one = fresh()
    want = [step(pool, pt, one, k[t], v[t], q[t]) for t in range(steps)]
    side = torch.cuda.Stream()
    pool2, pt2, one2 = fresh()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = [step(pool2, pt2, one2, k[t], v[t], q[t]) for t in range(steps)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    pool3, pt3, one3 = fresh()
    kk, vv, qq = k[0].clone(), v[0].clone(), q[0].clone()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(pool3, pt3, one3, kk, vv, qq)
    torch.cuda.current_stream().wait_stream(side)
    K.pages_trim(pt3, torch.zeros(B, dtype=torch.int32, device=DEV))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(pool3, pt3, one3, kk, vv, qq)
    for t in range(steps):
        kk.copy_(k[t]), vv.copy_(v[t]), qq.copy_(q[t])
        graph.replay()
        assert torch.equal(out, want[t])
        (out.float() @ out.float().transpose(-1, -2).contiguous()).sum().item()
    assert torch.equal(pt3.table, pt.table) and torch.equal(pt3.lens, pt.lens)


# ------------------------------------------------------------------------------------------------------------- cross
CROSS = [  # B, M, T, Hq, H, D
    (1, 1, 1, 1, 1, 48), (2, 50, 600, 32, 32, 48), (3, 1, 77, 8, 8, 64), (2, 129, 300, 4, 2, 128), (4, 5, 64, 16, 16, 72), (1, 300, 65, 4, 4, 80),
    (2, 33, 2000, 8, 1, 256), (1, 17, 5000, 2, 2, 24), (5, 64, 31, 6, 3, 104),
]


def cross_check(got, q, k, v, lens, mask, M, dt):
    B, T, H, D = k.shape
    G = q.shape[1] // H
    for b in range(B):
        on = torch.arange(T, device=DEV) < (T if lens is None else int(lens[b]))
        if mask is not None:
            on = on & mask[b]
        for h in range(q.shape[1]):
            close(got[b * M:(b + 1) * M, h], *formula(q[b * M:(b + 1) * M, h], k[b, :, h // G], v[b, :, h // G], on.expand(M, T)), dt)


@pytest.mark.parametrize('B,M,T,Hq,H,D', CROSS)
@pytest.mark.parametrize('kind', ['all', 'lens', 'mask', 'both'])
@pytest.mark.parametrize('dt', [BF, HF])
def test_cross_attend(B, M, T, Hq, H, D, kind, dt):
    """Keys that no row sees hold NaN and infinities; the last sequence's mask leaves nothing."""
    from yanlongvla_amd import kernels as K
    kv = rand(B, T, 2, H, D, seed=T, dt=dt)
    k, v = kv[:, :, 0], kv[:, :, 1]
    q = rand(B * M, Hq, D, seed=M, dt=dt, by=2.0)
    lens = ints([max(0, T - 13 * b) for b in range(B)]) if kind in ('lens', 'both') else None
    mask = None
    if kind in ('mask', 'both'):
        mask = torch.rand(B, T, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV) < 0.7
        if B > 1:
            mask[-1] = False
            mask[0, :min(T, 130)] = False                                    # whole tiles
            mask[0, -1] = True
    off = torch.zeros(B, T, dtype=torch.bool, device=DEV)
    if lens is not None:
        off |= torch.arange(T, device=DEV) >= lens[:, None]
    if mask is not None:
        off |= ~mask
    k[off], v[off] = math.nan, math.inf
    got = K.cross_attend(q, k, v, lens, mask)
    finite = torch.where(off[:, :, None, None], torch.zeros_like(v), v)      # (a masked key is not seen, whatever it holds)
    cross_check(got, q, torch.where(off[:, :, None, None], torch.zeros_like(k), k), finite, lens, mask, M, dt)
    if kind == 'mask' and B > 1:
        assert (got[-M:] == 0).all()


def test_cross_ragged_queries_views_and_replays():
    from yanlongvla_amd import kernels as K
    new, T, H, D = [3, 40, 0, 7], 200, 4, 64
    B = len(new)
    k, v = rand(B, T, H, D, seed=1), rand(B, T, H, D, seed=2)
    qkv = rand(sum(new) + 3, 3 * H, D, seed=3)
    q = qkv[:, H:2 * H]
    cu = ints([sum(new[:b]) for b in range(B + 1)])
    o = torch.full((sum(new) + 3, H, D), 7.0, dtype=BF, device=DEV)
    K.cross_attend(q, k, v, o=o, cu=cu, most=40)
    assert (o[sum(new):] == 7).all()
    for b in range(B):
        if new[b]:
            part = q[int(cu[b]):int(cu[b + 1])]
            for h in range(H):
                want = formula(part[:, h], k[b, :, h], v[b, :, h], torch.ones(new[b], T, dtype=torch.bool, device=DEV))
                close(o[int(cu[b]):int(cu[b + 1]), h], *want, BF)
    # keys as (B, H, T, D), and mask rows that lie apart
    kt, vt = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (k, v))
    mask = torch.ones(B, 2 * T, dtype=torch.bool, device=DEV)[:, :T]
    o2 = torch.full_like(o, 7.0)
    K.cross_attend(q, kt, vt, o=o2, cu=cu, most=40, mask=mask)
    assert torch.equal(o, o2)
    qq = q.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        K.cross_attend(qq, k, v, cu=cu, most=40)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):                                                       # two graphs at once: each has its own workspace
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = K.cross_attend(qq, k, v, cu=cu, most=40)
        graphs.append((g, out))
    for t in range(4):
        qq.copy_(rand(*qq.shape, seed=50 + t))
        want = K.cross_attend(qq, k, v, cu=cu, most=40)
        for g, out in graphs:
            g.replay()
        for g, out in graphs:
            assert torch.equal(out[:sum(new)], want[:sum(new)])


# ------------------------------------------------------------------------------------------------------- many workgroups, shared pages
@pytest.mark.parametrize('causal', [True, False])
@pytest.mark.parametrize('B', [9, 64, 70])
def test_more_tiles_than_fit_at_once(B, causal):
    """Calls of more than 512 workgroups, which are ordered by the keys that they see (up to 64 sequences): lengths of all kinds, sequences without rows,
    rows that see nothing."""
    from yanlongvla_amd import kernels as K
    Hq, H, D, T, dt = 16, 8, 64, 16, BF
    gen = torch.Generator().manual_seed(B)
    new = [0 if b % 7 == 3 else int(torch.randint(1, 700 if B < 64 else 150, (1,), generator=gen)) for b in range(B)]
    lens = [max(1, n - 40) if b % 5 == 1 else n + int(torch.randint(0, 200, (1,), generator=gen)) for b, n in enumerate(new)]
    pool = Pool(lens, H, D, T, dt, seed=B)
    q = rand(sum(new) + 2, Hq, D, seed=7, dt=dt, by=2.0)
    cu = ints([sum(new[:b]) for b in range(B + 1)])
    o = torch.full_like(q, 7.0)
    K.paged_attend(q, pool.pages, pool.table, pool.lens, o=o, causal=causal, cu=cu, most=700)
    assert (o[sum(new):] == 7).all()
    check(o, q, pool, lens, new, causal, dt)


def test_cross_attention_of_many_tiles():
    from yanlongvla_amd import kernels as K
    B, M, T, Hq, H, D = 5, 900, 150, 16, 16, 72
    k, v, q = rand(B, T, H, D, seed=1), rand(B, T, H, D, seed=2), rand(B * M, Hq, D, seed=3)
    lens = ints([150, 0, 77, 1, 128])
    cross_check(K.cross_attend(q, k, v, lens), q, k, v, lens, None, M, BF)
    mask = torch.rand(B, T, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV) < 0.5
    cross_check(K.cross_attend(q, k, v, lens, mask), q, k, v, lens, mask, M, BF)


def test_forks_attend_to_shared_pages_and_outputs_in_place():
    """Sequences that share pages give the same rows; an output may be the queries' own tensor; calls on two streams at once."""
    from yanlongvla_amd import kernels as K
    H, Hq, D, T, n = 2, 4, 128, 32, 3000
    pool, pt = K.kv_pages(110, H, D, DEV, T), K.page_table(3, 100, 110, DEV, T)
    k, v = rand(n, H, D, seed=1), rand(n, H, D, seed=2)
    start = K.pages_take(pt, pool, ints([n, 0, 0]))
    K.paged_append(pool, k, v, pt.table, pt.lens, start, ints([0, n, n, n]), n)
    K.pages_fork(pt, ints([0, 0]), ints([1, 2]))
    for m in (1, 40, 200):
        one = rand(m, Hq, D, seed=m)
        q = one.repeat(3, 1, 1)
        got = K.paged_attend(q, pool, pt.table, pt.lens)
        assert torch.equal(got[:m], got[m:2 * m]) and torch.equal(got[:m], got[2 * m:])
        streams = [torch.cuda.Stream() for _ in range(2)]
        outs = []
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                outs.append([K.paged_attend(q, pool, pt.table, pt.lens) for _ in range(5)])
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
        assert all(torch.equal(x, got) for x in outs[0] + outs[1])
        mine = q.clone()
        K.paged_attend(mine, pool, pt.table, pt.lens, o=mine)
        assert torch.equal(mine, got)
        wide = one[:1].expand(m, Hq, D)                                        # the same query in every row
        assert torch.equal(K.paged_attend(wide, pool, pt.table[:1], pt.lens[:1], causal=False)[0], K.paged_attend(wide.contiguous(), pool, pt.table[:1], pt.lens[:1], causal=False)[m - 1])
