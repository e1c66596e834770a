"""CPU checks of what the cache in pages, its attention and cross attention refuse: the C entries before any launch (status codes, pointers that are
never read), the Python helpers on host tensors."""
import ctypes
from pathlib import Path

import pytest
import torch

from yanlongvla_amd import kernels as K
from yanlongvla_amd._lib import SIGNATURES, TcqError

LIB = Path(__file__).resolve().parents[1] / 'yanlongvla_amd' / 'libtcq.so'
pytestmark = pytest.mark.skipif(not LIB.exists(), reason='libtcq.so not built')
P = 256                                            # an aligned address
ARG, SHAPE, DTYPE, UNSUPPORTED, ALIGN = -1, -2, -3, -4, -5
BF16, I8 = 1, 4


def entry(name):
    f = getattr(ctypes.CDLL(str(LIB)), name)
    f.argtypes, f.restype = SIGNATURES[name], ctypes.c_int
    return f


BOOK = dict(table=P, lens=P, refs=P, free=P, lack=P, B=2, N=4, pages=8, rows=16)
POOL = dict(k=P, v=P, layers=1, size=512)
BAD_BOOK = [(dict(table=None), ARG), (dict(lens=None), ARG), (dict(refs=None), ARG), (dict(free=None), ARG), (dict(lack=None), ARG), (dict(B=0), ARG),
            (dict(N=0), ARG), (dict(pages=0), ARG), (dict(rows=0), ARG), (dict(B=4097), UNSUPPORTED), (dict(N=1 << 27), UNSUPPORTED),
            (dict(pages=1 << 29), UNSUPPORTED), (dict(lens=P + 2), ALIGN)]
BAD_POOL = [(dict(k=None), ARG), (dict(v=None), ARG), (dict(layers=0), ARG), (dict(size=0), ARG), (dict(size=24), ALIGN), (dict(k=P + 8), ALIGN)]
ATTEND = dict(q=P, qt=64, qh=64, dtype=BF16, cu=P, lens=P, rows=4, most=2, B=2, Hq=2, Hk=1, D=64, k=P, kp=64, kh=64, kt=64, v=P, vp=64, vh=64, vt=64, pages=8,
              T=16, table=P, N=400, causal=1, scale=0.1, keys=6400, part=P, o=P, stream=None)
CROSS = dict(q=P, qt=64, qh=64, dtype=BF16, cu=P, rows=4, most=2, B=2, Hq=2, Hk=1, D=64, k=P, kb=64, kh=64, kt=64, v=P, vb=64, vh=64, vt=64, keys=6400,
             lens=P, mask=None, mb=0, scale=0.1, part=P, o=P, stream=None)
BAD_ATTEND = [(dict(q=None), ARG), (dict(k=None), ARG), (dict(v=None), ARG), (dict(o=None), ARG), (dict(part=None), ARG), (dict(rows=0), ARG),
              (dict(most=0), ARG), (dict(B=0), ARG), (dict(Hk=0), ARG), (dict(D=0), ARG), (dict(keys=-1), ARG), (dict(scale=-1.0), ARG),
              (dict(scale=float('nan')), ARG), (dict(scale=float('inf')), ARG), (dict(dtype=0), DTYPE), (dict(dtype=I8), DTYPE), (dict(Hk=3), SHAPE),
              (dict(cu=None, most=3), SHAPE), (dict(D=68), UNSUPPORTED), (dict(D=264), UNSUPPORTED), (dict(B=70000), UNSUPPORTED),
              (dict(kt=1 << 25), UNSUPPORTED), (dict(vh=-64), UNSUPPORTED), (dict(vt=56), UNSUPPORTED), (dict(qt=65), ALIGN), (dict(kt=68), ALIGN), (dict(q=P + 2), ALIGN),
              (dict(k=P + 8), ALIGN), (dict(o=P + 8), ALIGN), (dict(part=P + 4), ALIGN)]


@pytest.mark.parametrize('name,good,bad', [
    ('tcq_pages_take', dict(**BOOK, take=P, start=P, **POOL, moves=P, stream=None),
     BAD_BOOK + BAD_POOL + [(dict(take=None), ARG), (dict(start=None), ARG), (dict(moves=None), ARG)]),
    ('tcq_pages_fork', dict(**BOOK, src=P, dst=P, n=1, stream=None), BAD_BOOK + [(dict(src=None), ARG), (dict(dst=None), ARG), (dict(n=0), ARG), (dict(n=65536), UNSUPPORTED)]),
    ('tcq_pages_trim', dict(**BOOK, keep=P, stream=None), BAD_BOOK + [(dict(keep=None), ARG)]),
    ('tcq_pages_compact', dict(**BOOK, **POOL, moves=P, stream=None), BAD_BOOK + BAD_POOL + [(dict(moves=None), ARG)]),
    ('tcq_pages_copy', dict(k=P, v=P, layers=1, pages=8, size=512, src=P, dst=P, n=1, stream=None),
     BAD_POOL + [(dict(pages=0), ARG), (dict(src=None), ARG), (dict(dst=None), ARG), (dict(n=0), ARG)]),
    ('tcq_paged_append', dict(k=P, kt=64, kh=64, v=P, vt=64, vh=64, cu=P, rows=4, most=2, B=2, H=1, D=64, pk=P, pkp=64, pkh=64, pkt=64, pv=P, pvp=64,
                              pvh=64, pvt=64, pages=8, T=16, table=P, N=4, lens=P, start=P, stream=None),
     [(dict(k=None), ARG), (dict(pv=None), ARG), (dict(table=None), ARG), (dict(lens=None), ARG), (dict(start=None), ARG), (dict(rows=0), ARG),
      (dict(most=0), ARG), (dict(H=0), ARG), (dict(cu=None, most=3), SHAPE), (dict(T=24), UNSUPPORTED), (dict(T=8), UNSUPPORTED),
      (dict(B=70000), UNSUPPORTED), (dict(k=P + 1), ALIGN), (dict(start=P + 2), ALIGN)]),
    ('tcq_paged_attend', ATTEND, BAD_ATTEND + [(dict(lens=None), ARG), (dict(table=None), ARG), (dict(pages=0), ARG), (dict(N=0), ARG),
                                               (dict(T=24), UNSUPPORTED), (dict(T=8), UNSUPPORTED), (dict(N=1 << 27), UNSUPPORTED)]),
    ('tcq_cross_attend', CROSS, BAD_ATTEND + [(dict(keys=0), ARG)]),
])
def test_entries_refuse_before_launching(name, good, bad):
    f = entry(name)
    for change, status in bad:
        assert f(*{**good, **change}.values()) == status, change


@pytest.mark.parametrize('name', ['tcq_paged_attend_floats', 'tcq_cross_attend_floats'])
def test_workspace_size(name):
    f = entry(name)
    f.restype = ctypes.c_int64
    assert f(1, 1, 1, 8, 1, 256, 64) == 0                                # one tile: no split
    n = f(1, 1, 1, 8, 1, 256, 64000)
    assert n % (8 * 258) == 0 and n > 0
    assert f(0, 1, 1, 8, 1, 256, 64) == 0 and f(1, 1, 1, 8, 3, 256, 6400) == 0 and f(1, 1, 1, 8, 1, 100, 6400) == 0


def ints(*v):
    return torch.tensor(v, dtype=torch.int32)


def bf(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


def book(B=2, N=4, pages=8, rows=16):
    return K.page_table(B, N, pages, 'cpu', rows)


def test_tables_and_pools():
    pt = book(3, 5, 40)
    assert pt.table.shape == (3, 5) and (pt.table == -1).all() and pt.lens.tolist() == [0, 0, 0] and pt.refs.tolist() == [0] * 40
    assert pt.free.tolist() == [-1, 255] and pt.lack.tolist() == [0] and pt.rows == 16
    assert book(1, 1, 64).free.tolist() == [-1, -1]
    pool = K.kv_pages(8, 2, 64, 'cpu', 32, torch.float16, 3)
    assert pool.k.shape == pool.v.shape == (3, 8, 2, 32, 64)
    for bad in (dict(rows=24), dict(rows=8), dict(D=68), dict(D=264), dict(pages=0), dict(H=0), dict(dtype=torch.float32)):
        with pytest.raises(ValueError):
            K.kv_pages(**{**dict(pages=8, H=2, D=64, device='cpu'), **bad})
    for bad in ((0, 1, 1), (4097, 1, 1), (1, 0, 1), (1, 1, 0)):
        with pytest.raises(ValueError):
            K.page_table(*bad, 'cpu')
    with pytest.raises(ValueError):
        K.page_table(1, 1, 1, 'cpu', 48)


def test_helpers_refuse():
    pt, pool = book(), K.kv_pages(8, 2, 64, 'cpu', 16)
    layer, q = pool, bf(4, 4, 64)
    V, Y = ValueError, TypeError
    cases = [
        (V, lambda: K.pages_take(pt._replace(lens=ints(0)), pool, ints(1, 1))), (V, lambda: K.pages_take(pt, pool, ints(1))),
        (V, lambda: K.pages_take(pt, pool, ints(1, 1).long())), (V, lambda: K.pages_take(pt, K.kv_pages(9, 2, 64, 'cpu', 16), ints(1, 1))),
        (V, lambda: K.pages_take(pt, K.kv_pages(8, 2, 64, 'cpu', 32), ints(1, 1))), (V, lambda: K.pages_take(pt, pool, ints(1, 1), start=ints(1))), (V, lambda: K.pages_take(pt, pool, ints(1, 1), start=pt.lens)),
        (V, lambda: K.pages_take(pt._replace(free=ints(0, 0)), pool, ints(1, 1))), (V, lambda: K.pages_fork(pt, ints(0, 1), ints(1))),
        (V, lambda: K.pages_trim(pt, ints(0))), (V, lambda: K.pages_compact(pt, K.Pages(pool.k.transpose(0, 1), pool.v.transpose(0, 1)))),
        (V, lambda: K.pages_copy(K.Pages(pool.k[0, 0], pool.v[0, 0]), ints(0), ints(1))), (V, lambda: K.pages_copy(pool, ints(0), ints(1, 2))),
        (V, lambda: K.paged_append(layer, bf(2, 2, 64), bf(2, 1, 64), pt.table, pt.lens, ints(0, 0))),
        (V, lambda: K.paged_append(layer, bf(2, 3, 64), bf(2, 3, 64), pt.table, pt.lens, ints(0, 0))),
        (V, lambda: K.paged_append(layer, bf(2, 2, 64).half(), bf(2, 2, 64).half(), pt.table, pt.lens, ints(0, 0))),
        (V, lambda: K.paged_append(layer, bf(3, 2, 64), bf(3, 2, 64), pt.table, pt.lens, ints(0, 0))),
        (V, lambda: K.paged_append(layer, bf(2, 2, 64), bf(2, 2, 64), pt.table.long(), pt.lens, ints(0, 0))),
        (V, lambda: K.paged_append(layer, bf(2, 2, 64), bf(2, 2, 64), pt.table, pt.lens, ints(0))),
        (V, lambda: K.paged_append(K.Pages(*(t[:1].expand(8, -1, -1, -1) for t in pool)), bf(2, 2, 64), bf(2, 2, 64), pt.table, pt.lens, ints(0, 0))),
        (V, lambda: K.paged_attend(bf(4, 3, 64), layer, pt.table, pt.lens)), (V, lambda: K.paged_attend(bf(4, 4, 32), layer, pt.table, pt.lens)),
        (Y, lambda: K.paged_attend(q.half(), layer, pt.table, pt.lens)), (V, lambda: K.paged_attend(bf(5, 4, 64), layer, pt.table, pt.lens)),
        (V, lambda: K.paged_attend(q, layer, pt.table, pt.lens, o=bf(4, 4, 32))), (V, lambda: K.paged_attend(q, layer, pt.table, pt.lens, cu=ints(0, 1, 2))),
        (V, lambda: K.paged_attend(q, layer, pt.table[0], pt.lens)), (V, lambda: K.paged_attend(q, K.Pages(pool.k[:, :, :12], pool.v[:, :, :12]), pt.table, pt.lens)),
        (V, lambda: K.cross_attend(q, bf(2, 9, 2, 64), bf(2, 8, 2, 64))), (Y, lambda: K.cross_attend(q, bf(2, 9, 2, 64).half(), bf(2, 9, 2, 64).half())),
        (Y, lambda: K.cross_attend(q.float(), bf(2, 9, 2, 64).float(), bf(2, 9, 2, 64).float())),
        (V, lambda: K.cross_attend(q, bf(2, 9, 2, 64), bf(2, 9, 2, 64), lens=ints(1))), (V, lambda: K.cross_attend(q, bf(2, 9, 3, 64), bf(2, 9, 3, 64))),
        (V, lambda: K.cross_attend(q, bf(2, 9, 2, 64), bf(2, 9, 2, 64), mask=torch.ones(2, 9))),
        (V, lambda: K.cross_attend(q, bf(2, 9, 2, 64), bf(2, 9, 2, 64), mask=torch.ones(9, 2, dtype=torch.bool).t())),
    ]
    for i, (kind, call) in enumerate(cases):
        with pytest.raises(kind):
            call()
            pytest.fail(f'case {i} was taken')
    for call in (lambda: K.pages_take(pt, pool, ints(1, 1)), lambda: K.pages_fork(pt, ints(0), ints(1)), lambda: K.pages_trim(pt, ints(0, 0)),
                 lambda: K.pages_compact(pt, pool), lambda: K.pages_copy(pool, ints(0), ints(1)),
                 lambda: K.paged_append(layer, bf(2, 2, 64), bf(2, 2, 64), pt.table, pt.lens, ints(0, 0)),
                 lambda: K.paged_attend(q, layer, pt.table, pt.lens), lambda: K.cross_attend(q, bf(2, 9, 2, 64), bf(2, 9, 2, 64))):
        with pytest.raises(TcqError):                                        # host tensors
            call()
