"""CPU checks of what the rotary positions, the 8-bit cache, its attention and the norm to INT8 rows refuse: the C entries before any
launch (status codes, pointers that are never read), the Python helpers on host tensors."""
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
BF16, F16, I8 = 1, 2, 4


def entry(name):
    f = getattr(ctypes.CDLL(str(LIB)), name)
    f.argtypes, f.restype = SIGNATURES[name], ctypes.c_int
    return f


NORM = dict(x=P, ldx=64, r=P, ldr=64, w=P, eps=1e-6, offset=1.0, dtype=BF16, xout=P, ldo=64, q=P, q4=None, ldq=0, scale=P, M=2, K=64, stream=None)
ROPE = dict(q=P, qt=64, qh=64, qo=P, qot=64, qoh=64, Hq=2, k=P, kt=64, kh=64, ko=P, kot=64, koh=64, Hk=1, dtype=BF16, pos=P, pos64=0, pa=1, pt=1,
            freq=P, axis=P, A=1, M=1, D=64, R=64, adjacent=0, inverse=0, stream=None)
APPEND = dict(k=P, kt=64, kh=64, v=P, vt=64, vh=64, dtype=BF16, cu=P, start=P, rows=4, most=2, B=2, H=1, D=64, nblk=1, k8=P, v8=P, scale=P, tail=P,
              stream=None)
READ = dict(k8=P, v8=P, scale=P, first=P, lens=P, n=4, B=1, H=1, D=64, nblk=1, k=P, v=P, dtype=BF16, stream=None)
ATTEND = dict(q=P, qt=64, qh=64, dtype=BF16, cu=P, lens=P, rows=4, most=2, B=2, Hq=2, Hk=1, D=64, nblk=100, k8=P, v8=P, scale=P, causal=1, ss=0.1,
              keys=6400, part=P, o=P, stream=None)


@pytest.mark.parametrize('name,good,bad', [
    ('tcq_add_norm_quantize', NORM, [(dict(x=None), ARG), (dict(w=None), ARG), (dict(scale=None), ARG), (dict(q=None), ARG), (dict(M=0), ARG),
                                     (dict(K=0), ARG), (dict(K=40000), SHAPE), (dict(dtype=I8), DTYPE), (dict(q4=P, ldq=1), ARG),
                                     (dict(q4=P, ldq=-16, K=72), SHAPE), (dict(q4=P + 4, ldq=-16), ALIGN), (dict(x=P + 1), ALIGN),
                                     (dict(q4=P, ldq=2, K=62), SHAPE)]),
    ('tcq_rope_axes', ROPE, [(dict(q=None), ARG), (dict(qo=None), ARG), (dict(k=None), ARG), (dict(pos=None), ARG), (dict(freq=None), ARG),
                             (dict(A=0), ARG), (dict(M=0), ARG), (dict(Hq=0), ARG), (dict(Hk=-1), ARG), (dict(R=65), SHAPE), (dict(R=66), SHAPE),
                             (dict(R=0), SHAPE), (dict(dtype=I8), DTYPE), (dict(q=P + 1), ALIGN), (dict(pos=P + 4, pos64=1), ALIGN),
                             (dict(freq=P + 4), ALIGN), (dict(axis=P + 2), ALIGN)]),
    ('tcq_kv8_append', APPEND, [(dict(k=None), ARG), (dict(start=None), ARG), (dict(tail=None), ARG), (dict(rows=0), ARG), (dict(most=0), ARG),
                                (dict(B=0), ARG), (dict(nblk=0), ARG), (dict(dtype=0), DTYPE), (dict(D=96), UNSUPPORTED), (dict(B=70000), UNSUPPORTED),
                                (dict(cu=None, most=3), SHAPE), (dict(k8=P + 8), ALIGN), (dict(k=P + 1), ALIGN), (dict(scale=P + 4), ALIGN)]),
    ('tcq_kv8_read', READ, [(dict(k8=None), ARG), (dict(lens=None), ARG), (dict(v=None), ARG), (dict(n=0), ARG), (dict(dtype=I8), DTYPE),
                            (dict(D=32), UNSUPPORTED), (dict(k=P + 8), ALIGN)]),
    ('tcq_kv8_attend', ATTEND, [(dict(q=None), ARG), (dict(lens=None), ARG), (dict(o=None), ARG), (dict(part=None), ARG), (dict(rows=0), ARG),
                                (dict(keys=-1), ARG), (dict(ss=-1.0), ARG), (dict(ss=float('nan')), ARG), (dict(ss=float('inf')), ARG),
                                (dict(dtype=0), DTYPE), (dict(Hk=3), SHAPE), (dict(cu=None, most=3), SHAPE), (dict(D=80), UNSUPPORTED),
                                (dict(qt=65), ALIGN), (dict(q=P + 2), ALIGN), (dict(o=P + 8), ALIGN)]),
])
def test_entries_refuse_before_launching(name, good, bad):
    f = entry(name)
    for change, status in bad:
        assert f(*{**good, **change}.values()) == status, change


def test_workspace_size():
    f = entry('tcq_kv8_attend_floats')
    f.restype = ctypes.c_int64
    assert f(1, 1, 1, 8, 1, 256, 64) == 0                                # one block: no split
    n = f(1, 1, 1, 8, 1, 256, 6400)
    assert n % (8 * 258) == 0 and n > 0
    assert f(0, 1, 1, 8, 1, 256, 64) == 0 and f(1, 1, 1, 8, 3, 256, 6400) == 0 and f(1, 1, 1, 8, 1, 100, 6400) == 0


def ints(*v):
    return torch.tensor(v, dtype=torch.int32)


def test_norm_helper_refuses():
    x, w = torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(64, dtype=torch.bfloat16)
    q, s = torch.zeros(2, 64, dtype=torch.int8), torch.zeros(2)
    for change in (dict(r=x[:1]), dict(r=x.half()), dict(w=w[:32]), dict(w=w.float()), dict(scale=s[:1]), dict(scale=None), dict(q=None), dict(q=q[:, :32]),
                   dict(xout=x.t().contiguous().t()), dict(q4=torch.zeros(1, 4, 16, 16, dtype=torch.int32)), dict(q4=torch.zeros(16, 1, dtype=torch.int32)),
                   dict(q4=torch.zeros(1, 3, 16, 16, dtype=torch.int8))):
        with pytest.raises(ValueError):
            K.add_norm_quantize(**{**dict(x=x, r=x, w=w, eps=1e-6, q=q, scale=s), **change})
    with pytest.raises(TypeError):
        K.add_norm_quantize(x.int(), None, w.int(), 1e-6, q, s)
    with pytest.raises(TcqError):
        K.add_norm_quantize(x, x, w, 1e-6, q, s)                         # host tensors


def test_rope_helper_refuses():
    q, k, pos = torch.zeros(3, 4, 64), torch.zeros(3, 2, 64), torch.zeros(2, 3, dtype=torch.int32)
    freq, axis = K.rope_frequencies(64, sections=(20, 12))
    for change in (dict(q=q[0]), dict(k=k[:2]), dict(k=k.half()), dict(k=k[..., :32]), dict(pos=pos[:, :2]), dict(pos=pos.float()), dict(freq=freq.float()),
                   dict(freq=torch.cat([freq, freq])), dict(axis=axis[:3]), dict(axis=axis.long()), dict(q_out=q[:2]), dict(k_out=q), dict(k=None, k_out=k),
                   dict(q=q.transpose(0, 2))):
        with pytest.raises(ValueError):
            K.rope_axes(**{**dict(q=q, k=k, pos=pos, freq=freq, axis=axis), **change})
    with pytest.raises(TcqError):
        K.rope_axes(q, k, pos, freq, axis)
    for sections in ((20, 11), (33,)):
        with pytest.raises(ValueError):
            K.rope_frequencies(64, sections=sections)


def test_frequencies_and_axes():
    freq, axis = K.rope_frequencies(16, 100.0, (3, 3, 2), True)
    assert axis.tolist() == [0, 1, 2, 0, 1, 2, 0, 1] and freq.tolist() == [100.0 ** (-i / 8) for i in range(8)]
    assert K.rope_frequencies(16, 100.0, (3, 3, 2))[1].tolist() == [0, 0, 0, 1, 1, 1, 2, 2]
    assert K.rope_frequencies(128, sections=(24, 20, 20), interleaved=True)[1].tolist() == [0, 1, 2] * 20 + [0] * 4


def test_cache_helpers_refuse():
    c = K.kv8_cache(2, 1, 64, 100, 'cpu')
    assert c.k8.shape == (2, 1, 2, 4, 4, 16, 16) and c.v8.shape == (2, 1, 2, 4, 4, 16, 16)
    for bad in (dict(D=96), dict(dtype=torch.float32), dict(tokens=0), dict(B=0)):
        with pytest.raises(ValueError):
            K.kv8_cache(**{**dict(B=1, H=1, D=64, tokens=64, device='cpu'), **bad})
    k = torch.zeros(4, 1, 64, dtype=torch.bfloat16)
    for change in (dict(k=k.half(), v=k.half()), dict(v=k[:3]), dict(k=k[..., :32]), dict(start=ints(0)), dict(start=torch.zeros(2, dtype=torch.int64)),
                   dict(cu=ints(0, 1)), dict(cu=ints(0, 2, 4)), dict(most=3), dict(k=k[:3], v=k[:3]), dict(cache=c._replace(v8=c.v8[:1])),
                   dict(cache=c._replace(scale=c.scale.double())), dict(cu=ints(0, 2, 4), most=-1)):
        with pytest.raises(ValueError):
            K.kv8_append(**{**dict(cache=c, k=k, v=k, start=ints(0, 0)), **change})
    q = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    for change in (dict(q=q[0]), dict(q=q[:, :, :32]), dict(lens=ints(0)), dict(o=q[:2]), dict(o=q.half()), dict(q=q[:3]), dict(q=q[:, :0]),
                   dict(cache=K.kv8_cache(2, 3, 64, 64, 'cpu')), dict(cu=ints(0, 2, 4))):
        with pytest.raises(ValueError):
            K.kv8_attend(**{**dict(q=q, cache=c, lens=ints(1, 1)), **change})
    with pytest.raises(TypeError):
        K.kv8_attend(q.float(), c, ints(1, 1))
    with pytest.raises(ValueError):
        K.kv8_read(c, ints(0), ints(1, 1), 4)
    for call in (lambda: K.kv8_append(c, k, k, ints(0, 0)), lambda: K.kv8_attend(q, c, ints(1, 1)), lambda: K.kv8_read(c, ints(0, 0), ints(1, 1), 4)):
        with pytest.raises(TcqError):
            call()
