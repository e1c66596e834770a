"""GPU tests of the 8-bit key / value cache: rows into it and out of it bit for bit against the definition, and attention over it against
64 bits. Sizes and masks where it can go wrong: no rows, one token, lengths at and around a block's end, more rows than a block, appends
that are taken back, ragged batches, grouped heads of every head size, rows that see nothing, long splits, offsets past 32 bits, values
that are not finite, views, other streams and graph replays.

Tolerance of attention, 2-norm of the difference over that of the result: half a step of the output type (2^-8 BF16, 2^-11 FP16), plus
2e-4 for what is held in 16-bit integers: a score is off by at most score_scale * (largest |q| / 32512) * sum |k|, and for the normal
inputs here (|q| <= 10, D = 256, 200 |k| of mean 0.8, scale 1 / 16) by less than 4e-3 in the worst case and 16 times less with random
signs; a probability by 1 / 65278 of its block's largest."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda'
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
T = 64


@pytest.fixture(scope='module', autouse=True)
def _lib():
    from yanlongvla_amd import _lib
    _lib.lib()
    torch.cuda.init()


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def rand(*shape, seed, dt=BF):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dt)


def values(x):
    """The values that a cache holding the rows x (n, H, D) of one sequence stands for: FP32, block by block."""
    out = torch.zeros(x.shape, dtype=FP, device=x.device)
    for j in range(0, x.shape[0], T):
        f = x[j:j + T].float()
        f = torch.where(f.isnan(), torch.zeros_like(f), f)
        big = torch.where(f.isinf(), torch.zeros_like(f), f).abs().amax((0, 2), keepdim=True)
        s = torch.where(big > 0, big / torch.full_like(big, 127), torch.ones_like(big))      # (by a number, torch multiplies by 1 / 127)
        code = 127 * torch.minimum(torch.maximum(f, -big), big).double() / torch.where(big > 0, big, torch.ones_like(big)).double()
        out[j:j + T] = code.round().float() * s
    return out


def fill(lens, H, D, dt=BF, seed=0, room=0, lead=None):
    """A cache of len(lens) sequences of these lengths, appended in one call, its rows and lengths."""
    from yanlongvla_amd import kernels as K
    k, v = (rand(sum(lens), H, D, seed=seed + i, dt=dt) for i in (1, 2))
    cache = K.kv8_cache(len(lens), H, D, max(max(lens), 1) + room, DEV, dt)
    cu = ints([sum(lens[:i]) for i in range(len(lens) + 1)])
    K.kv8_append(cache, k, v, ints([0] * len(lens)), cu, max(lens))
    return cache, k, v


def split(x, lens):
    return list(x.split(lens))


@pytest.mark.parametrize('H,D,dt', [(1, 256, BF), (8, 128, BF), (2, 64, HF), (3, 128, HF)])
@pytest.mark.parametrize('lens', [[1], [64], [65, 0, 63], [200, 128, 129, 1]])
def test_append_and_read_bit_for_bit(H, D, dt, lens):
    from yanlongvla_amd import kernels as K
    cache, k, v = fill(lens, H, D, dt, seed=D)
    n = max(lens) + 70
    got = K.kv8_read(cache, ints([0] * len(lens)), ints(lens), n, FP)
    for x, y in zip((k, v), got):
        for b, rows in enumerate(split(x, lens)):
            assert torch.equal(y[b, :lens[b]], values(rows))
            assert (y[b, lens[b]:] == 0).all()
    first = [min(5, x) for x in lens]
    for t in (BF, HF):
        part = K.kv8_read(cache, ints(first), ints(lens), 61, t)
        for x, y in zip(got, part):
            for b in range(len(lens)):
                assert torch.equal(y[b], x[b, first[b]:first[b] + 61].to(t))


@pytest.mark.parametrize('D', [64, 128, 256])
@pytest.mark.parametrize('steps', [[1] * 70, [63, 1, 1], [10, 60, 200], [64, 64, 5], [130, 1, 130], [7, 0, 300, 1]])
def test_codes_do_not_depend_on_how_the_rows_came(D, steps):
    from yanlongvla_amd import kernels as K
    n, H = sum(steps), 2
    k, v = rand(n, H, D, seed=3), rand(n, H, D, seed=4)
    one, many = (K.kv8_cache(1, H, D, n, DEV) for _ in range(2))
    K.kv8_append(one, k, v, ints([0]))
    at = 0
    for s in steps:
        K.kv8_append(many, k[at:at + s], v[at:at + s], ints([at]))
        at += s
    assert all(torch.equal(a, b) for a, b in zip(one[:3], many[:3]))
    # the newest two blocks' rows are kept
    j = (n - 1) // T
    for blk in range(max(0, j - 1), j + 1):
        rows = slice(blk * T, min(n, blk * T + T))
        for i, x in enumerate((k, v)):
            assert torch.equal(many.tail[0, :, blk % 2, i, :rows.stop - rows.start], x[rows].transpose(0, 1))


@pytest.mark.parametrize('P,M', [(850, 50), (128, 64), (127, 1), (100, 64), (64, 64), (0, 64)])
def test_rows_taken_back(P, M):
    """The same start again (a denoising step's action tokens): the cache is the one of the second rows alone."""
    from yanlongvla_amd import kernels as K
    H, D = 1, 256
    k, v = rand(P + 2 * M, H, D, seed=5), rand(P + 2 * M, H, D, seed=6)
    a, b = (K.kv8_cache(1, H, D, P + M, DEV) for _ in range(2))
    if P:
        K.kv8_append(a, k[:P], v[:P], ints([0]))
    for i in range(2):
        K.kv8_append(a, k[P + i * M:P + i * M + M], v[P + i * M:P + i * M + M], ints([P]))
    keep = [*range(P), *range(P + M, P + 2 * M)]
    K.kv8_append(b, k[keep], v[keep], ints([0]))
    assert all(torch.equal(x, y) for x, y in zip(a[:3], b[:3]))


@pytest.mark.parametrize('seed', range(6))
def test_appends_and_rows_taken_back_at_random(seed):
    """Starts as the documentation allows them, from the furthest position so far and new beginnings at multiples of 64: the cache is that
    of the surviving rows."""
    import random
    from yanlongvla_amd import kernels as K
    H, D, room, r = 2, 64, 1200, random.Random(seed)
    cache, one = (K.kv8_cache(1, H, D, room, DEV) for _ in range(2))
    k, v = (torch.zeros(room, H, D, dtype=BF, device=DEV) for _ in range(2))
    least = end = far = 0
    for i in range(60):
        low = max(least, far - T)
        if r.random() < 0.1 and end >= T:
            start = r.randrange(0, end // T + 1) * T
            if start < low:
                least = far = start
        else:
            start = end if r.random() < 0.4 else r.randint(min(low, end), end)
        n = r.choice((1, 1, 2, 7, 33, 64, 65, 130, 200))
        n = min(n, room - start)
        if n == 0:
            break
        k[start:start + n], v[start:start + n] = rand(n, H, D, seed=1000 * seed + 2 * i), rand(n, H, D, seed=1000 * seed + 2 * i + 1)
        K.kv8_append(cache, k[start:start + n], v[start:start + n], ints([start]))
        end = start + n
        far = max(far, end)
    K.kv8_append(one, k[:end], v[:end], ints([0]))
    got, want = ([x[0] for x in K.kv8_read(c, ints([0]), ints([end]), end, FP)] for c in (cache, one))
    assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize('dt', [BF, HF])
def test_half_of_the_largest_is_a_tie(dt):
    """Blocks of +-(largest, half of it), whatever the largest's rounded scale: code 127 and, half to even, 64. Largest values from the
    types' smallest to their greatest ones."""
    from yanlongvla_amd import kernels as K
    n, fi = 300, torch.finfo(dt)
    most = torch.logspace(math.log2(fi.smallest_normal), math.log2(fi.max), n, 2, dtype=torch.float64, device=DEV).clamp(max=fi.max).to(dt)
    most[:4] = torch.tensor([2.0, 4.0, 6.0, 254.0], device=DEV).to(dt) * fi.smallest_normal * fi.eps     # denormal ones
    half = most / 2
    x = torch.zeros(n * T, 1, 64, dtype=dt, device=DEV)
    x[::T, 0, 0], x[5::T, 0, 7], x[63::T, 0, 63] = 2 * half, half, -half
    cache = K.kv8_cache(1, 1, 64, n * T, DEV, dt)
    K.kv8_append(cache, x, x, ints([0]))
    codes = cache.k8[0, 0].permute(0, 1, 3, 2, 4).reshape(n, T, 64)
    assert (codes[:, 0, 0] == 127).all() and (codes[:, 5, 7] == 64).all() and (codes[:, 63, 63] == -64).all()
    got = K.kv8_read(cache, ints([0]), ints([n * T]), n * T, FP)
    assert all(torch.equal(y[0], values(x)) for y in got)


def test_views_other_sequences_and_the_capacity():
    """Rows as unaligned views of a wider row; a sequence without new rows and the blocks before the new ones stay; rows past the
    capacity, past `most` and past the tensor are dropped."""
    from yanlongvla_amd import kernels as K
    H, D = 2, 64
    for pad in (0, 1):
        row = rand(90, 3 * H * D + pad, seed=7)
        k, v = row[:, H * D:2 * H * D].unflatten(1, (H, D)), row[:, 2 * H * D:3 * H * D].unflatten(1, (H, D))
        cache = K.kv8_cache(3, H, D, 100, DEV)                       # 128 tokens
        for t in cache:
            t.fill_(3)
        before = [t.clone() for t in cache]
        K.kv8_append(cache, k, v, ints([64, 5, 120]), ints([0, 40, 40, 80]), 64)
        assert all(torch.equal(x[1], y[1]) and torch.equal(x[0, :, 0], y[0, :, 0]) for x, y in zip(cache[:3], before[:3]))
        assert torch.equal(cache.tail[1], before[3][1]) and torch.equal(cache.k8[2, :, 0], before[0][2, :, 0])
        got = K.kv8_read(cache, ints([64, 0, 120]), ints([104, 0, 160]), 40, FP)
        for x, y in zip((k, v), got):
            assert torch.equal(y[0], values(x[:40]))
            old = torch.full((56, H, D), 3.0, device=DEV)             # rows 64 .. 119 of the last sequence, from its tail
            assert torch.equal(y[2, :8], values(torch.cat([old.to(BF), x[40:48]]))[56:]) and (y[2, 8:] == 0).all()
    mark = [t.clone() for t in cache]
    K.kv8_append(cache, k, v, ints([128, 0, 500]), ints([0, 10, 10, 20]), 20)       # nothing fits
    K.kv8_append(cache, k, v, ints([0, 0, 0]), ints([90, 120, 130, 140]), 20)       # rows that the tensor does not have
    assert all(torch.equal(x, y) for x, y in zip(cache, mark))
    K.kv8_append(cache, k, v, ints([0, 0, 0]), ints([0, 50, 50, 50]), 20)           # most below the count: its first rows
    assert torch.equal(K.kv8_read(cache, ints([0] * 3), ints([20, 0, 0]), 20, FP)[0][0], values(k[:20]))


def test_not_finite_rows():
    """NaN becomes 0, an infinity the block's largest code; other rows keep theirs."""
    from yanlongvla_amd import kernels as K
    k, v = rand(70, 1, 128, seed=8), rand(70, 1, 128, seed=9)
    k[3, 0, 5], k[4, 0, 6], v[66, 0, 7], v[0, 0, 0] = float('nan'), float('-inf'), float('inf'), float('nan')
    k[64:] = float('nan')                                              # a block without a finite value
    cache = K.kv8_cache(1, 1, 128, 70, DEV)
    K.kv8_append(cache, k, v, ints([0]))
    got = K.kv8_read(cache, ints([0]), ints([70]), 70, FP)
    assert torch.equal(got[0][0], values(k)) and torch.equal(got[1][0], values(v))
    o = K.kv8_attend(rand(1, 1, 128, seed=1), cache, ints([70]))
    assert o.isfinite().all()


# ---------------------------------------------------------------------------------------------------------------- attention
def reference(q, k, v, lens, counts, G, causal, scale=None):
    """FP64 attention of packed rows q over k, v (B, n, H, D)."""
    out, at = torch.zeros(q.shape, dtype=torch.float64, device=q.device), 0
    for b, m in enumerate(counts):
        n = lens[b]
        for h in range(q.shape[1]):
            s = q[at:at + m, h].double() @ k[b, :n, h // G].double().t() * (scale or 1 / math.sqrt(q.shape[2]))
            if causal:
                s = s.masked_fill(torch.arange(n, device=q.device)[None] > torch.arange(m, device=q.device)[:, None] + n - m, -math.inf)
            p = torch.nan_to_num(torch.softmax(s, 1), nan=0.0) if n else s
            out[at:at + m, h] = p @ v[b, :n, h // G].double()
        at += m
    return out


def close(o, want, score=0.0):
    """score: the root mean square error of a score, for queries outside of what the 2e-4 covers: the probabilities' relative errors, and with
    values of mean zero the outputs' (sum p^2 |v|^2 enters both norms)."""
    tol = torch.finfo(o.dtype).eps / 2 + 2e-4 + score
    assert torch.isfinite(o).all()
    assert (o.double() - want).norm() <= tol * want.norm()
    assert (o.double() - want).abs().max() <= 8 * tol * want.abs().max()


@pytest.mark.parametrize('Hq,Hk,D,dt', [(8, 1, 256, BF), (16, 8, 128, BF), (4, 4, 64, HF), (6, 2, 64, BF), (16, 1, 128, HF), (7, 1, 256, HF)])
@pytest.mark.parametrize('lens,counts,causal', [
    ([1], [1], True), ([968], [1], True), ([64, 65, 63, 1], [1, 1, 1, 1], True), ([850, 70], [50, 50], False), ([300], [300], True),
    ([129, 500, 40], [1, 130, 40], True), ([2000, 64], [3, 0], True), ([5000], [2], False), ([64, 700], [0, 513], True)])
def test_attend_matches_fp64(Hq, Hk, D, dt, lens, counts, causal):
    from yanlongvla_amd import kernels as K
    cache, _, _ = fill(lens, Hk, D, dt, seed=11)
    k, v = K.kv8_read(cache, ints([0] * len(lens)), ints(lens), max(lens), FP)
    q = rand(sum(counts), Hq, D, seed=12, dt=dt) * 2
    cu = ints([sum(counts[:i]) for i in range(len(counts) + 1)])
    o = torch.full_like(q, float('nan'))
    K.kv8_attend(q, cache, ints(lens), o, causal=causal, cu=cu, most=max(counts))
    close(o, reference(q, k, v, lens, counts, Hq // Hk, causal))
    if len(set(counts)) == 1:
        p = K.kv8_attend(q, cache, ints(lens), causal=causal)
        assert torch.equal(o, p)


@pytest.mark.parametrize('D', [128, 64])
@pytest.mark.parametrize('dt', [BF, HF])
@pytest.mark.parametrize('lens,counts,causal', [([700, 420, 300, 64], [530, 420, 300, 1], True), ([333, 64], [1030, 1030], False)])
def test_attend_of_many_rows(lens, counts, causal, dt, D):
    """Enough rows for two tiles a wave: ragged ones, sequences shorter than their rows, rows that see nothing; blocks whose value scales
    differ by up to 2^40, the largest where nothing looks."""
    from yanlongvla_amd import kernels as K
    Hq, Hk = 16, 8
    cache, _, _ = fill(lens, Hk, D, dt, seed=31)
    q = rand(sum(counts), Hq, D, seed=32, dt=dt) * 2
    q[5, 3, 7] = float('nan')
    cu = ints([sum(counts[:i]) for i in range(len(counts) + 1)])
    k, v = K.kv8_read(cache, ints([0] * len(lens)), ints(lens), max(lens), FP)
    G = Hq // Hk

    def both(cache, k, v, q):
        o = torch.full_like(q, 9.0)
        K.kv8_attend(q, cache, ints(lens), o, causal=causal, cu=cu, most=max(counts))
        assert o[5, 3].isnan().all()
        want = reference(q, k, v, lens, counts, G, causal)
        o[5, 3], want[5, 3] = 0, 0
        return o, want

    close(*both(cache, k, v, q))
    # the second block's values 2^-40 of the others', then 2^30 of them but with keys that no query picks
    for e, pick in ((-40.0, False), (30.0, True)):
        scale, k2, v2 = cache.scale.clone(), k.clone(), v.clone()
        scale[:, :, 1, 1] *= 2.0 ** e
        v2[:, T:2 * T] *= 2.0 ** e
        qq = q.clone()
        if pick:                                                        # one dim decides: no query picks the keys of that block
            k8 = cache.k8.clone()
            k8[:, :, :, :, 0, :, 0] = 127
            k8[:, :, 1, :, 0, :, 0] = -127
            big = K.KV8(k8, cache.v8, scale, cache.tail)
            qq[..., 0] = 200.0
            k2, _ = K.kv8_read(big, ints([0] * len(lens)), ints(lens), max(lens), FP)
        else:
            big = cache._replace(scale=scale)
        # a digit of a query row whose largest value is 200 (2^E = 256) is off by at most half of 256 / 32512, 256 / 32512 / sqrt(12) =
        # 2.3e-3 root mean square; keys of D normal values, one of them 127 codes of 4 / 127: norm 12 (D = 128) or 9; scale 1 / sqrt(D):
        # 2.4e-3, 2.6e-3
        close(*both(big, k2, v2, qq), score=256 / 32512 / 12 ** 0.5 * (D + 16) ** 0.5 / D ** 0.5 if pick else 0.0)


@pytest.mark.parametrize('keys', [0, 64, 1000, 10 ** 6])
def test_hint_changes_the_split_only(keys):
    from yanlongvla_amd import kernels as K
    lens = [3000, 17]
    cache, _, _ = fill(lens, 2, 128, seed=13, room=3000)
    k, v = K.kv8_read(cache, ints([0, 0]), ints(lens), 3000, FP)
    q = rand(4, 8, 128, seed=14)
    close(K.kv8_attend(q, cache, ints(lens), keys=keys), reference(q, k, v, lens, [2, 2], 4, True))


@pytest.mark.parametrize('keys', [64, 10 ** 6])
def test_rows_that_see_nothing_are_zeros_and_others_untouched(keys):
    """Empty sequences, more causal rows than the sequence holds, rows of no sequence (left as they were)."""
    from yanlongvla_amd import kernels as K
    lens = [0, 2, 700]
    cache, _, _ = fill([1, 2, 700], 2, 64, seed=15)
    k, v = K.kv8_read(cache, ints([0] * 3), ints(lens), 700, FP)
    q = rand(30, 4, 64, seed=16)
    o = torch.full_like(q, 9.0)
    K.kv8_attend(q, cache, ints(lens), o, cu=ints([0, 5, 15, 25]), most=12, keys=keys)
    want = reference(q[:25], k, v, lens, [5, 10, 10], 2, True)
    assert (o[:13] == 0).all() and (o[25:] == 9).all() and (want[5:13] == 0).all()
    close(o[:25], want)
    o2 = torch.full_like(q, 9.0)
    K.kv8_attend(q, cache, ints(lens), o2, cu=ints([0, 5, 15, 25]), most=6, keys=keys)       # most below a count: its first rows
    assert torch.equal(o2[5:11], o[5:11]) and (o2[11:15] == 9).all() and torch.equal(o2[15:21], o[15:21])


def test_hidden_rows_do_not_count():
    """What the cache holds past a sequence's length, in its last block too, does not reach the result."""
    from yanlongvla_amd import kernels as K
    cache, _, _ = fill([200], 1, 256, seed=17)
    q = rand(3, 8, 256, seed=18)
    a = K.kv8_attend(q, cache, ints([131]))
    k8, v8 = cache.k8.clone(), cache.v8.clone()
    k8[0, 0, 2, 0, :, 3:], k8[0, 0, 2, 1:], k8[0, 0, 3] = 127, 127, 127
    for t in range(3, T):
        v8[0, 0, 2, :, t % 16 // 4, :, t // 16 * 4 + t % 4] = -127
    v8[0, 0, 3] = 127
    scale = cache.scale.clone()
    scale[0, 0, 3] = float('nan')
    assert torch.equal(a, K.kv8_attend(q, K.KV8(k8, v8, scale, cache.tail), ints([131])))


def test_not_finite_queries_and_extreme_sizes():
    """A row that is not finite is NaN, alone; rows of zeros are means; tiny and huge queries, keys and values keep their digits; a block of
    huge values does not cost another its own."""
    from yanlongvla_amd import kernels as K
    lens = [300]
    cache, _, _ = fill(lens, 1, 128, seed=19)
    k, v = K.kv8_read(cache, ints([0]), ints(lens), 300, FP)
    q = rand(16, 1, 128, seed=20)
    q[2, 0, 5], q[7, 0, 9], q[11] = float('nan'), float('inf'), 0
    for keys in (0, 10 ** 6):
        o = K.kv8_attend(q, cache, ints(lens), causal=False, keys=keys)
        ok = [i for i in range(16) if i not in (2, 7)]
        assert o[2].isnan().all() and o[7].isnan().all()
        close(o[ok], reference(q[ok], k, v, lens, [14], 1, False))
    for qe, ke, ve in ((1e-30, 1e30, 1.0), (1e30, 1e-30, 1e-30), (1.0, 1.0, 1e35), (1e-38, 1e37, 1e-35)):
        big = K.KV8(cache.k8, cache.v8, cache.scale * torch.tensor([ke, ve], device=DEV), cache.tail)
        qq = (rand(16, 1, 128, seed=21).float() * qe).to(BF)
        want = reference(qq, k.double() * ke, v.double() * ve, lens, [16], 1, False)
        o = K.kv8_attend(qq, big, ints(lens), causal=False)
        assert (o.double() - want).norm() <= (2.0 ** -8 + 2e-4) * want.norm()
    scale = cache.scale.clone()
    scale[0, 0, 0] *= torch.tensor([0.0, 1e6], device=DEV)              # huge values whose keys all score 0
    k2, v2 = k.clone(), v.clone()
    k2[:, :T] = 0
    v2[:, :T] *= 1e6
    qq = rand(16, 1, 128, seed=22) * 8
    close(K.kv8_attend(qq, K.KV8(cache.k8, cache.v8, scale, cache.tail), ints(lens), causal=False), reference(qq, k2, v2, lens, [16], 1, False))


def test_views_scale_and_streams():
    """q as an unpadded view of a q | k | v row; a score scale of its own; a stream of its own."""
    from yanlongvla_amd import kernels as K
    lens = [100, 333]
    cache, _, _ = fill(lens, 2, 64, seed=23)
    k, v = K.kv8_read(cache, ints([0, 0]), ints(lens), 333, FP)
    row = rand(6, 4 * 64 + 256, seed=24)
    q = row[:, 128:384].unflatten(1, (4, 64))
    want = reference(q, k, v, lens, [3, 3], 2, True, scale=0.3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o = K.kv8_attend(q, cache, ints(lens), scale=0.3)
    side.synchronize()
    close(o, want)


def test_offsets_past_32_bits():
    """The last of three sequences lies behind 2^31 bytes of keys; the cache of one long sequence has its last block there too."""
    from yanlongvla_amd import kernels as K
    tokens = (1 << 32) // 256 // 3
    cache = K.kv8_cache(3, 1, 256, tokens, DEV)
    assert cache.k8[2].data_ptr() - cache.k8.data_ptr() > 1 << 31
    k, v = rand(300, 1, 256, seed=25), rand(300, 1, 256, seed=26)
    K.kv8_append(cache, k, v, ints([0, 0, tokens // T * T - 200]), ints([0, 0, 0, 300]), 300)
    end = tokens // T * T + 100
    cap = cache.k8.shape[2] * T
    got = K.kv8_read(cache, ints([0, 0, end - 300]), ints([0, 0, end]), 300, FP)
    n = min(300, cap - (end - 300))
    # start at 64 i + 56: the first block also holds 56 rows of zeros, which change no scale
    pad = torch.zeros((end - 300) % T, 1, 256, device=DEV).to(BF)
    for x, y in zip((k, v), got):
        assert torch.equal(y[2, :n], values(torch.cat([pad, x[:n]]))[len(pad):])
    q = rand(3, 8, 256, seed=27)
    o = K.kv8_attend(q, cache, ints([0, 1, end]), causal=False)
    s = q[2].double() @ got[0][2, :n, 0].double().t() / 16
    s = torch.cat([s, torch.zeros(8, 1, dtype=torch.float64, device=DEV)], 1)       # the zeros before: exp(0) each
    m = s.amax(1, keepdim=True)
    e = (s - m).exp()
    want = e[:, :-1] @ got[1][2, :n, 0].double() / (e[:, :-1].sum(1, keepdim=True) + e[:, -1:] * (min(end, cap) - n))
    assert (o[2].double() - want).norm() <= (2.0 ** -8 + 2e-4) * want.norm() and (o[:2] == 0).all()


def test_decode_loop_as_one_graph():
    """A prompt, then steps of rotary positions, append and attention, captured once with the lengths on the device and replayed: every
    step equals the eager one on another cache and the FP64 attention over what that cache holds."""
    from yanlongvla_amd import kernels as K
    B, Hq, Hk, D, P = 2, 16, 8, 128, 61
    freq, axis = K.rope_frequencies(D, 10000.0, (24, 20, 20), True, device=DEV)
    caches = [K.kv8_cache(B, Hk, D, 200, DEV) for _ in range(2)]
    k, v = rand(2 * P, Hk, D, seed=28), rand(2 * P, Hk, D, seed=29)
    for c in caches:
        K.kv8_append(c, k, v, ints([0, 0]))
    row = rand(B, (Hq + 2 * Hk) * D, seed=30)
    qkv = [x.unflatten(1, (-1, D)) for x in row.split([Hq * D, Hk * D, Hk * D], 1)]
    pos, start = torch.full((3, B), P, dtype=torch.int32, device=DEV), ints([P, P])

    def step(cache, start, pos):
        q, k = (torch.empty(x.shape, dtype=x.dtype, device=DEV) for x in qkv[:2])
        K.rope_axes(qkv[0], qkv[1], pos, freq, axis, q, k)
        K.kv8_append(cache, k, qkv[2], start)
        return q, K.kv8_attend(q, cache, start + 1)

    first = [t.clone() for t in caches[0]]
    step(caches[0], start, pos)                                         # warm
    for t, s in zip(caches[0], first):
        t.copy_(s)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        _, o = step(caches[0], start, pos)
        start.add_(1)
        pos.add_(1)
    for t, s in zip(caches[0], first):
        t.copy_(s)
    at, pp = ints([P, P]), pos.clone()
    for i in range(8):
        row.copy_(rand(*row.shape, seed=40 + i))
        gr.replay()
        torch.cuda.synchronize()
        q, want = step(caches[1], at, pp)
        at.add_(1)
        pp.add_(1)
        assert torch.equal(o, want) and all(torch.equal(a, b) for a, b in zip(*caches))
        n = [P + i + 1] * B
        kk, vv = K.kv8_read(caches[1], ints([0, 0]), ints(n), n[0], FP)
        close(o, reference(q, kk, vv, n, [1, 1], 2, True))


FORMS = [([90, 400], 8, 1, 256, 2, 500), ([5000, 3000], 16, 8, 128, 1, 5000), ([5000, 100], 4, 1, 64, 3, 5000), ([9000], 8, 1, 256, 1, 9000),
         ([600, 900], 16, 8, 128, 520, 900), ([600, 900], 16, 8, 64, 520, 900), ([300, 200], 8, 2, 64, 70, 300)]


@pytest.mark.parametrize('lens,Hq,Hk,D,M,keys', FORMS)
def test_attend_replays_with_other_lengths(lens, Hq, Hk, D, M, keys):
    """One workgroup a tile, keys in few and in many parts, many rows: captured once, replayed with lengths and queries that change, eager
    calls in between; every replay is the eager call's result."""
    from yanlongvla_amd import kernels as K
    cache, _, _ = fill(lens, Hk, D, seed=51)
    B = len(lens)
    q, n = rand(B * M, Hq, D, seed=52), ints(lens)
    K.kv8_attend(q, cache, n, keys=keys)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        o = K.kv8_attend(q, cache, n, keys=keys)
    for i, cut in enumerate((0, 70, 1, 10 ** 6, 0)):
        q.copy_(rand(B * M, Hq, D, seed=60 + i))
        n.copy_(ints([max(0, x - cut) for x in lens]))
        gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, K.kv8_attend(q, cache, n, keys=keys))
        assert cut < 10 ** 6 or (o == 0).all()


def test_calls_on_two_streams_at_once():
    """Attention in parts of two caches on two streams, a third cache appended to beside them, the results those of one after the other."""
    from yanlongvla_amd import kernels as K
    jobs = []
    for i, (lens, Hq, Hk, D, M, keys) in enumerate(FORMS[1:4]):
        cache, _, _ = fill(lens, Hk, D, seed=70 + i)
        q = rand(len(lens) * M, Hq, D, seed=80 + i)
        jobs.append((cache, q, ints(lens), keys, K.kv8_attend(q, cache, ints(lens), keys=keys)))
    one, two = (K.kv8_cache(1, 8, 128, 3000, DEV) for _ in range(2))
    k, v = rand(3000, 8, 128, seed=90), rand(3000, 8, 128, seed=91)
    K.kv8_append(one, k, v, ints([0]))
    starts = [ints([a]) for a in range(0, 3000, 100)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = [[] for _ in jobs]
    for _ in range(10):
        for (cache, q, n, keys, _), st, g in zip(jobs, streams, got):
            with torch.cuda.stream(st):
                g.append(K.kv8_attend(q, cache, n, keys=keys))
        for a in starts[:3]:
            K.kv8_append(two, k[:100], v[:100], a)
    for i, a in enumerate(starts):
        K.kv8_append(two, k[100 * i:100 * i + 100], v[100 * i:100 * i + 100], a)
    torch.cuda.synchronize()
    for job, g in zip(jobs, got):
        assert all(torch.equal(x, job[4]) for x in g)
    assert all(torch.equal(x, y) for x, y in zip(one[:3], two[:3]))


def test_more_row_tiles_than_a_grid_axis_holds():
    """65600 rows of 16 heads on one KV head: 65600 tiles of 16 rows; the first, the last and those in between, causal and not."""
    from yanlongvla_amd import kernels as K
    rows, D, n = 65600, 64, 150
    cache, _, _ = fill([n], 1, D, seed=95)
    k, v = K.kv8_read(cache, ints([0]), ints([n]), n, FP)
    q = rand(rows, 16, D, seed=96)
    o = K.kv8_attend(q, cache, ints([n]), causal=False)
    for at in (0, 60, 90, 32000, 65500):
        close(o[at:at + 100], reference(q[at:at + 100], k, v, [n], [100], 16, False))
    o = K.kv8_attend(q, cache, ints([n]), torch.full_like(q, 9.0))
    assert (o[:rows - n] == 0).all()
    close(o[rows - n:], reference(q[rows - n:], k, v, [n], [n], 16, True))
