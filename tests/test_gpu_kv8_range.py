"""GPU tests of the attention over the 8-bit cache at the ends of its range, against 64 bits over the values that the cache stands for: large
scores, blocks of one large and many small probabilities, value scales far apart or denormal, lengths past the capacity.

Tolerance, 2-norm of the difference over that of the result: half a step of the output type (2^-8 BF16, 2^-11 FP16), plus 2e-4 for the
query's and the probabilities' 16-bit integers (a probability is off by 1 / 65278 of its block's largest; the queries' share is stated where it is
larger)."""
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


def rand(*shape, seed, dt=FP):
    return torch.randn(*shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV).to(dt)


def fill(B, n, H, D, dt=BF, seed=0):
    """A cache of B sequences of n normal rows each."""
    from yanlongvla_amd import kernels as K
    cache = K.kv8_cache(B, H, D, n, DEV, dt)
    K.kv8_append(cache, rand(B * n, H, D, seed=seed, dt=dt), rand(B * n, H, D, seed=seed + 1, dt=dt), ints([0] * B))
    return cache


def held(cache, n):
    """The values that a cache stands for, k and v (B, n, H, D) in 64 bits: codes times scales (in 32 bits the smallest ones would round)."""
    B, H, N, _, E = cache.k8.shape[:5]
    k = cache.k8.permute(0, 1, 2, 3, 5, 4, 6).reshape(B, H, N * T, E * 16)
    v = cache.v8.view(B, H, N, E, 4, 16, 4, 4).permute(0, 1, 2, 6, 4, 7, 3, 5).reshape(B, H, N * T, E * 16)
    s = cache.scale.double().repeat_interleave(T, 2)
    return [(x.double() * s[..., i:i + 1]).transpose(1, 2)[:, :n] for i, x in enumerate((k, v))]


def reference(q, k, v, lens, G, causal=False, scale=None):
    """FP64 attention of len(lens) equal shares of the rows q over k, v (B, n, H, D); a row that sees nothing is zeros."""
    m, out = q.shape[0] // len(lens), torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for b, n in enumerate(lens):
        rows = slice(b * m, b * m + m)
        for h in range(q.shape[1]):
            s = q[rows, h].double() @ k[b, :n, h // G].t() * (scale or 1 / math.sqrt(q.shape[2]))
            if causal:
                s = s.masked_fill(torch.arange(n, device=q.device)[None] > torch.arange(m, device=q.device)[:, None] + n - m, -math.inf)
            out[rows, h] = torch.nan_to_num(torch.softmax(s, 1), nan=0.0) @ v[b, :n, h // G]
    return out


def close(o, want, more=0.0):
    tol = torch.finfo(o.dtype).eps / 2 + 2e-4 + more
    assert torch.isfinite(o).all()
    assert (o.double() - want).norm() <= tol * want.norm()


def each_row_close(o, want, more=0.0):
    """The same for every row and head alone."""
    tol = torch.finfo(o.dtype).eps / 2 + 2e-4 + more
    assert torch.isfinite(o).all()
    assert ((o.double() - want).norm(dim=-1) <= tol * want.norm(dim=-1)).all()


# one launch of eight waves, four waves in parts, four waves with 64 dims, two row tiles a wave with 128 and 64 dims
FORMS = [(2, 16, 8, 1, 256, 300), (2, 16, 8, 1, 256, 3000), (1, 40, 4, 2, 64, 1500), (2, 600, 16, 8, 128, 700), (4, 600, 16, 8, 64, 300)]


@pytest.mark.parametrize('dt', [BF, HF])
@pytest.mark.parametrize('logit', [100.0, 400.0, 700.0, 1500.0, 5000.0, 1e5, 1e7])
@pytest.mark.parametrize('B,M,Hq,Hk,D,n', FORMS)
def test_large_scores_pick_their_key(B, M, Hq, Hk, D, n, logit, dt):
    """Every query row is a multiple of one key, whose score is `logit`, several standard deviations above the others': the
    output is that key's value."""
    from yanlongvla_amd import kernels as K
    logit = min(logit, 1e7 if dt == BF else 1e4)                       # (FP16 queries end at 65504)
    cache = fill(B, n, Hk, D, dt, seed=11)
    k, v = held(cache, n)
    pick = torch.randint(0, n, (B, M, Hq), generator=torch.Generator(device=DEV).manual_seed(3), device=DEV)
    b, h = torch.arange(B, device=DEV)[:, None, None], torch.arange(Hq, device=DEV) // (Hq // Hk)
    key = k[b, pick, h]                                                # (B, M, Hq, D)
    q = (key * (logit * D ** 0.5 / key.square().sum(-1, keepdim=True))).to(dt).view(B * M, Hq, D)
    each_row_close(K.kv8_attend(q, cache, ints([n] * B), causal=False), v[b, pick, h].view(B * M, Hq, D))


def test_weights_of_a_block_add_up_to_one():
    """One key of a block ahead of 63 whose probabilities are 0.489 of a digit each, values that are all 1: the output is 1, whatever the small
    probabilities are rounded to. Numerator and denominator are the same whole numbers times powers of two and the value's 127 / 127: three
    FP32 roundings, then the type's half step."""
    from yanlongvla_amd import kernels as K
    for D, n in ((64, 64), (256, 64), (128, 128)):
        k = torch.zeros(n, 1, D, dtype=HF, device=DEV)
        k[::T, 0, 0] = 1                                               # the only key that counts, one in every block
        cache = K.kv8_cache(1, 1, D, n, DEV, HF)
        K.kv8_append(cache, k, torch.ones_like(k), ints([0]))
        q = torch.zeros(3, 1, D, dtype=HF, device=DEV)
        q[:, 0, 0] = 11.109 * D ** 0.5                                 # exp(-11.109) = 0.489 / 32639
        o = K.kv8_attend(q, cache, ints([n]), causal=False)
        assert ((o.double() - 1).abs() <= 2.0 ** -11 + 4 * 2.0 ** -24).all()


ROWS = [(2, 600, 16, 8, 128, 700), (4, 600, 16, 8, 64, 300)]           # two row tiles a wave


@pytest.mark.parametrize('B,M,Hq,Hk,D,n', ROWS)
@pytest.mark.parametrize('causal', [False, True])
def test_denormal_value_scales_of_many_rows(B, M, Hq, Hk, D, n, causal):
    """BF16 values whose scale is denormal in FP32 in some blocks, in all of them, or in none of those that a row sees."""
    from yanlongvla_amd import kernels as K
    cache = fill(B, n, Hk, D, seed=21)
    q = rand(B * M, Hq, D, seed=22, dt=BF) * 2
    for blocks in (slice(1, 2), slice(0, 1), slice(None)):
        scale = cache.scale.clone()
        scale[:, :, blocks, 1] *= 2.0 ** -122                          # about 2^-127 to 2^-128
        assert (scale[:, :, blocks, 1] < torch.finfo(FP).smallest_normal).all() and (scale > 0).all()
        big = cache._replace(scale=scale)
        o = K.kv8_attend(q, big, ints([n] * B), causal=causal)
        want = reference(q, *held(big, n), [n] * B, Hq // Hk, causal)
        if blocks == slice(None):                                      # a result of 2^-122 to 2^-127 rounds to whole multiples of 2^-133
            assert ((o.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2e-4 * want.abs().max() + 2.0 ** -134).all()
        else:
            close(o, want)


@pytest.mark.parametrize('dt', [BF, HF])
@pytest.mark.parametrize('Hq,Hk,D', [(16, 8, 128), (16, 16, 64)])
def test_many_small_probabilities_behind_large_values(Hq, Hk, D, dt):
    """32768 keys of one small probability each (2^-17.4 of the four keys' that are picked) behind blocks whose value scale is 50 times
    theirs, values of opposite sign: together they are 4 % of the weight. As FP16 numbers in units of the larger scale they are 190 steps
    of the smallest FP16 number, off by half of one: 2.6e-3 of 4 %, twice (both signs), 2.3e-4 in all."""
    from yanlongvla_amd import kernels as K
    M, n = 1024, 32768
    k, v = (torch.zeros(n, Hk, D, dtype=dt, device=DEV) for _ in range(2))
    v -= 1
    k[:4 * T:T, :, 0] = 1
    v[:4 * T:T] = 1
    v[1:4 * T:T] = 50
    cache = K.kv8_cache(1, Hk, D, n, DEV, dt)
    K.kv8_append(cache, k, v, ints([0]))
    q = torch.zeros(M, Hq, D, dtype=dt, device=DEV)
    q[..., 0] = 12.086 * D ** 0.5
    o = K.kv8_attend(q, cache, ints([n]), causal=False)
    each_row_close(o, reference(q[:1], *held(cache, n), [n], Hq // Hk).expand(M, Hq, D), more=2.3e-4)


@pytest.mark.parametrize('order', [(0, 1), (1, 0), (0, 0, 1), (1, 1, 1, 1, 1, 0)])
@pytest.mark.parametrize('e', [(0, -100), (100, 0), (60, -60), (0, -120), (3, -12)])
@pytest.mark.parametrize('B,M,Hq,Hk,D,n', [*ROWS, (2, 16, 16, 8, 128, 700)])
def test_value_scales_far_apart(B, M, Hq, Hk, D, n, e, order):
    """Two kinds of blocks in turn whose value scales differ by up to 2^120; every other row (token and head) looks at the one kind alone, the rest at
    the other (the scores lie 170 apart): each row for itself is held to 64 bits, whatever the other rows of its tile look at.
    The queries' largest value is 32: a digit is off by 32 / 32512 / sqrt(12) root mean square, keys of norm sqrt(D + 8 * 16), scale 1 / sqrt(D):
    4e-4, taken twice for single rows."""
    from yanlongvla_amd import kernels as K
    cache = fill(B, n, Hk, D, seed=31)
    k8, scale = cache.k8.clone(), cache.scale.clone()
    for j in range(k8.shape[2]):
        kind = order[j % len(order)]
        k8[:, :, j, :, 0, :, :8] = 127 if kind else -127
        scale[:, :, j, 1] *= 2.0 ** e[kind]
    big = K.KV8(k8, cache.v8, scale, cache.tail)
    q = rand(B * M, Hq, D, seed=32)
    sign = 1 - 2 * ((torch.arange(B * M, device=DEV)[:, None] + torch.arange(Hq, device=DEV)) % 2)
    q[..., :8] = 30.0 * sign[..., None]
    q = q.to(BF)
    o = K.kv8_attend(q, big, ints([n] * B), causal=False)
    each_row_close(o, reference(q, *held(big, n), [n] * B, Hq // Hk), more=2 * 32 / 32512 / 12 ** 0.5 * ((D + 128) / D) ** 0.5)


@pytest.mark.parametrize('B,M,Hq,Hk,D,n', ROWS)
@pytest.mark.parametrize('causal', [False, True])
def test_blocks_of_zeros_among_small_values(B, M, Hq, Hk, D, n, causal):
    """A block of zero values has scale 1, others 2^-100 of a usual one; and a scale of zero, which counts as zeros."""
    from yanlongvla_amd import kernels as K
    cache = fill(B, n, Hk, D, seed=41)
    q = rand(B * M, Hq, D, seed=42, dt=BF)
    for zero in (1.0, 0.0):
        v8, scale = cache.v8.clone(), cache.scale.clone()
        scale[..., 1] *= 2.0 ** -100
        v8[:, :, 1::3] = 0
        scale[:, :, 1::3, 1] = zero
        big = K.KV8(cache.k8, v8, scale, cache.tail)
        close(K.kv8_attend(q, big, ints([n] * B), causal=causal), reference(q, *held(big, n), [n] * B, Hq // Hk, causal))


@pytest.mark.parametrize('B,M,Hq,Hk,D', [(1, 20, 8, 1, 256), (1, 20, 4, 2, 64), (2, 1200, 8, 8, 64)])
@pytest.mark.parametrize('past', [0, 1, 12, 64, 1000])
def test_causal_rows_past_the_capacity(B, M, Hq, Hk, D, past):
    """Lengths past the capacity: rows that no longer fit are dropped, row i of n still sees positions j <= lens - n + i of what is held."""
    from yanlongvla_amd import kernels as K
    n = 1280 if M > 20 else 128
    cache = fill(B, n, Hk, D, seed=51)
    k, v = held(cache, n)
    q = rand(B * M, Hq, D, seed=52, dt=BF)
    lens = [n + past, n - 7][:B]
    o = K.kv8_attend(q, cache, ints(lens))
    want = torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    for b, x in enumerate(lens):
        for h in range(Hq):
            s = q[b * M:b * M + M, h].double() @ k[b, :, h // (Hq // Hk)].t() / D ** 0.5
            hidden = torch.arange(n, device=DEV)[None] > torch.arange(M, device=DEV)[:, None] + x - M
            s = s.masked_fill(hidden | (torch.arange(n, device=DEV) >= x), -math.inf)
            want[b * M:b * M + M, h] = torch.nan_to_num(torch.softmax(s, 1), nan=0.0) @ v[b, :, h // (Hq // Hk)]
    close(o, want)
    both = K.kv8_attend(q, cache, ints(lens), causal=False)              # every row sees what is held
    close(both, reference(q, k, v, [min(x, n) for x in lens], Hq // Hk))


@pytest.mark.parametrize('B,M,Hq,Hk,D,n', FORMS)
@pytest.mark.parametrize('qe,ke', [(1e34, 1e-36), (1e36, 1e-37), (1e-36, 1e34), (1e-10, 1e10)])
def test_huge_queries_of_tiny_keys(B, M, Hq, Hk, D, n, qe, ke):
    """Scores of usual size from a product of very large and very small numbers."""
    from yanlongvla_amd import kernels as K
    cache = fill(B, n, Hk, D, seed=61)
    scale = cache.scale.clone()
    scale[..., 0] *= ke
    big = cache._replace(scale=scale)
    q = (rand(B * M, Hq, D, seed=62) * 2 * qe).to(BF)
    close(K.kv8_attend(q, big, ints([n] * B), causal=False), reference(q, *held(big, n), [n] * B, Hq // Hk))


@pytest.mark.parametrize('B,M,Hq,Hk,D,n', FORMS)
@pytest.mark.parametrize('causal', [False, True])
def test_a_score_scale_of_zero_gives_means(B, M, Hq, Hk, D, n, causal):
    from yanlongvla_amd import kernels as K
    cache = fill(B, n, Hk, D, seed=71)
    q = rand(B * M, Hq, D, seed=72, dt=BF)
    zero = reference(q * 0, *held(cache, n), [n] * B, Hq // Hk, causal)
    close(K.kv8_attend(q, cache, ints([n] * B), causal=causal, scale=0.0), zero)
    close(K.kv8_attend(q * 0, cache, ints([n] * B), causal=causal), zero)
