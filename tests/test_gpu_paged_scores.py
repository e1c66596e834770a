"""GPU tests of the attentions over pages and states with scores far out, the same by every plan: few rows or many, the keys whole or in parts.

Scores here are sums that FP32 holds exactly, in any order: 56 products of A^2 and some of `unit`, where unit is at least the step of FP32 at 56 A^2 to
64 A^2. So the weights follow from their differences (S - m) times a scale that is rounded twice (2^-23), rounded once more (2^-24): of keys up to 128 bits
below the reference a weight is off by 128 * 1.5 * 2^-23 ln 2 = 1.6e-5 of itself. The rest as in test_gpu_paged.py."""
import math

import pytest
import torch

from test_gpu_paged import BF, DEV, HF, Pool, close, formula, rand

pytestmark = pytest.mark.gpu
# new rows, rows held, the plan's keys: few rows whole, in parts; many rows whole, in parts (of one KV head)
PLANS = [(1, 300, 64), (1, 300, 6000), (5500, 300, 64), (200, 300, 6000)]


@pytest.fixture(scope='module', autouse=True)
def _lib():
    from yanlongvla_amd import _lib
    _lib.lib()
    torch.cuda.init()


def both(q, pool, k, v, scale, keys):
    """The attention over the pages, and over the same rows as states."""
    from yanlongvla_amd import kernels as K
    yield K.paged_attend(q, pool.pages, pool.table, pool.lens, causal=False, scale=scale, keys=keys)
    yield K.cross_attend(q, k[None], v[None], scale=scale)


@pytest.mark.parametrize('scale', [None, 1.0, 30.0])
@pytest.mark.parametrize('M,n,keys', PLANS)
@pytest.mark.parametrize('dt', [BF, HF])
def test_every_score_minus_infinity(M, n, keys, scale, dt):
    """A row all of whose scores are -inf has no weights: NaN, not the zeros of a row that sees nothing. One key in a late tile that is finite has them all."""
    pool = Pool([n], 1, 64, 64, dt, seed=5)
    q = rand(M, 1, 64, seed=6, dt=dt).abs() + 0.1
    pool.pages.k.fill_(-math.inf)
    pool.k[0].fill_(-math.inf)
    for got in both(q, pool, pool.k[0], pool.v[0], scale, keys):
        assert got.isnan().all()
    j = n - 3
    pool.pages.k[int(pool.table[0, j // 64]), :, j % 64] = 1.0
    pool.k[0][j] = 1.0
    for got in both(q, pool, pool.k[0], pool.v[0], scale, keys):
        assert torch.equal(got, pool.v[0][j].expand_as(got))


def far_out(M, n, dt, A, unit, seed):
    """q (M, 1, 64) and k (n, 1, 64) with scores 56 A^2 + unit c[j], and c: integers that rise over the tiles in steps, the largest of them several times."""
    g = torch.Generator().manual_seed(seed)
    j = torch.arange(n)
    c = torch.randint(0, 40, (n,), generator=g) + 30 * (j // 64).clamp(max=3)
    c[[n // 2, n // 2 + 1, n - 2]] = 130
    root = 2.0 ** math.floor(math.log2(unit) / 2)
    q = torch.full((M, 1, 64), A)
    k = torch.full((n, 1, 64), A)
    q[:, :, 56:], k[:, :, 56:] = 0, 0
    q[:, :, 60], k[:, 0, 60] = root, c * (unit / root)
    return q.to(DEV, dt), k.to(DEV, dt), c


# A, unit, scale: differences of one unit are half a nat (the first three), or so much that keys with the same score alone count; the last ones past FP16
FAR = [(2.0 ** 5, 2.0 ** 0, 0.5), (2.0 ** 10, 4.0, 0.125), (2.0 ** 14, 2.0 ** 10, 2.0 ** -11), (2.0 ** 10, 4.0, 64.0), (2.0 ** 10, 4.0, 1e12)]
PAST = [(2.0 ** 60, 2.0 ** 102, 2.0 ** -103), (2.0 ** 60, 2.0 ** 102, 1.0), (2.0 ** 60, 2.0 ** 102, 3e38)]


@pytest.mark.parametrize('dt,A,unit,scale', [(dt, *x) for dt in (BF, HF) for x in FAR] + [(BF, *x) for x in PAST])
@pytest.mark.parametrize('M,n,keys', PLANS)
def test_scores_far_out(M, n, keys, A, unit, scale, dt):
    q, k, c = far_out(M, n, dt, A, unit, seed=3)
    assert torch.equal((q[0, 0].double() @ k[:, 0].double().t()).cpu(), 56 * A * A + unit * c.double())
    pool = Pool([n], 1, 64, 64, dt, seed=5)
    for j in range(0, n, 64):
        pool.pages.k[int(pool.table[0, j // 64]), 0, :min(64, n - j)] = k[j:j + 64, 0]
    v = pool.v[0]
    o, a, _ = formula(q[:1, 0], k[:, 0], v[:, 0], torch.ones(1, n, dtype=torch.bool, device=DEV), scale)
    for got in both(q, pool, k, v, scale, keys):
        assert got.isfinite().all() and (got == got[:1]).all()
        close(got[:1, 0], o, a, 1.6e-5, dt)
