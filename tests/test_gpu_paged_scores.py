"""GPU tests of the attentions over pages and states with scores far out, the same by every plan: few rows or many, the keys whole or in parts. Tolerances as in test_gpu_paged.py."""
import math

import pytest
import torch

from test_gpu_paged import BF, HF, Pool, rand

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
