"""GPU tests of the rotary positions (kernels.rope_axes) against the rotation in 64 bits: types, head layouts, strides, one to three
axes, both pairings, partial rotation, in place, far and negative positions, the inverse as the gradient, and graph replays.

Tolerance of one value y = x1 c - x2 s: half a step of the output type, plus FP32 arithmetic: c and s within 2^-22 (the angle is exact to
far below that, the library's sine and cosine within two units of 2^-24 of numbers up to 1) and two roundings of 2^-24 of terms up to
|x1| + |x2|; together below 2^-21 (|x1| + |x2|). FP16 adds its smallest step."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda'
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope='module', autouse=True)
def _lib():
    from yanlongvla_amd import _lib
    _lib.lib()
    torch.cuda.init()


def reference(x, pos, freq, axis, adjacent, inverse):
    """The rotation and the sum of the magnitudes that enter each value, FP64 on the host."""
    x, pos, freq, axis = x.double().cpu(), pos.double().cpu(), freq.cpu(), axis.cpu().long()
    a = (pos[axis] * freq[:, None]).t()[:, None] * (-1 if inverse else 1)
    h = freq.numel()
    i, j = (torch.arange(0, 2 * h, 2), torch.arange(1, 2 * h, 2)) if adjacent else (torch.arange(h), torch.arange(h, 2 * h))
    y, mag = x.clone(), torch.zeros_like(x)
    y[..., i] = x[..., i] * a.cos() - x[..., j] * a.sin()
    y[..., j] = x[..., j] * a.cos() + x[..., i] * a.sin()
    mag[..., i] = mag[..., j] = x[..., i].abs() + x[..., j].abs()
    return y, mag


def check(got, want, mag):
    step = torch.finfo(got.dtype).eps / 2
    tol = step * want.abs() + 2.0 ** -21 * mag + (2.0 ** -25 if got.dtype == HF else 0.0)
    assert ((got.double().cpu() - want).abs() <= tol).all()


def make(M, Hq, Hk, D, R, A, dt, seed, far=5000, low=0, sections=None, interleaved=False):
    from yanlongvla_amd import kernels as K
    g = torch.Generator(device=DEV).manual_seed(seed)
    q = torch.randn(M, Hq, D, generator=g, device=DEV).to(dt)
    k = torch.randn(M, Hk, D, generator=g, device=DEV).to(dt) if Hk else None
    pos = torch.randint(low, far + 1, (A, M), generator=g, device=DEV, dtype=torch.int64)
    if sections is None and A > 1:
        sections = [R // 2 // A + (R // 2 % A if a == 0 else 0) for a in range(A)]
    freq, axis = K.rope_frequencies(R, 10000.0, sections, interleaved, device=DEV)
    return q, k, pos, freq, axis


@pytest.mark.parametrize('M,Hq,Hk,D,R,A,dt,adjacent', [
    (1, 8, 1, 256, 256, 1, BF, False), (1, 16, 8, 128, 128, 3, BF, False), (700, 16, 8, 128, 128, 3, HF, True),
    (4761, 16, 16, 64, 64, 2, FP, False), (33, 5, 0, 80, 64, 2, BF, False), (7, 3, 1, 40, 20, 3, HF, False), (9, 2, 2, 64, 6, 1, FP, True),
    (2500, 1, 1, 72, 72, 2, BF, False), (3, 1, 1, 4096, 2048, 1, BF, False), (257, 4, 2, 96, 32, 2, FP, True)])
@pytest.mark.parametrize('inverse', [False, True])
def test_rope_matches_fp64(M, Hq, Hk, D, R, A, dt, adjacent, inverse):
    from yanlongvla_amd import kernels as K
    q, k, pos, freq, axis = make(M, Hq, Hk, D, R, A, dt, M + D)
    qo, ko = torch.empty_like(q), None if k is None else torch.empty_like(k)
    K.rope_axes(q, k, pos, freq, axis, qo, ko, adjacent=adjacent, inverse=inverse)
    for x, y in ((q, qo), (k, ko)):
        if x is not None:
            check(y, *reference(x, pos, freq, axis, adjacent, inverse))


def test_positions_far_negative_and_of_both_types():
    from yanlongvla_amd import kernels as K
    q, k, pos, freq, axis = make(64, 2, 1, 128, 128, 3, FP, 5, far=2 ** 31 - 1, low=-2 ** 31)
    out = [torch.empty_like(q) for _ in range(2)]
    K.rope_axes(q, None, pos, freq, axis, out[0])
    K.rope_axes(q, None, pos.int(), freq, axis, out[1])
    # at 2^31 an FP64 angle in turns is within 2^-24: 2^-21 rad more than at near positions
    want, mag = reference(q, pos, freq, axis, False, False)
    assert ((out[0].double().cpu() - want).abs() <= 2.0 ** -24 * want.abs() + 2.0 ** -19 * mag).all()
    assert torch.equal(out[0], out[1])


@pytest.mark.parametrize('interleaved', [False, True])
def test_sections_give_each_pair_its_axis(interleaved):
    from yanlongvla_amd import kernels as K
    freq, axis = K.rope_frequencies(128, 10000.0, (24, 20, 20), interleaved, device=DEV)
    assert [int((axis == a).sum()) for a in range(3)] == [24, 20, 20]
    assert axis.tolist()[:4] == ([0, 1, 2, 0] if interleaved else [0, 0, 0, 0])
    assert freq[0] == 1 and math.isclose(freq[63], 10000 ** (-63 / 64), rel_tol=1e-15)


@pytest.mark.parametrize('dt,pad', [(BF, 0), (BF, 3), (FP, 2)])
def test_strided_views_in_place_leave_the_rest(dt, pad):
    """q and k as parts of one q | k | v row (aligned or not), turned in place: only they change."""
    from yanlongvla_amd import kernels as K
    M, Hq, Hk, D = 37, 4, 2, 64
    row = torch.randn(M, (Hq + 2 * Hk) * D + pad, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).to(dt)
    before = row.clone()
    q, k = row[:, :Hq * D].unflatten(1, (Hq, D)), row[:, Hq * D:(Hq + Hk) * D].unflatten(1, (Hk, D))
    _, _, pos, freq, axis = make(M, 1, 1, D, D, 2, dt, 3)
    want = [reference(x, pos, freq, axis, False, False) for x in (q, k)]
    K.rope_axes(q, k, pos, freq, axis)
    check(q, *want[0]), check(k, *want[1])
    assert torch.equal(row[:, (Hq + Hk) * D:], before[:, (Hq + Hk) * D:])


def test_pair_without_axis_stays_and_copies_elsewhere():
    from yanlongvla_amd import kernels as K
    q, _, pos, freq, axis = make(5, 2, 0, 64, 32, 1, BF, 9)
    axis[3:7] = 9
    axis[8] = -1
    o = torch.full_like(q, float('nan'))
    K.rope_axes(q, None, pos, freq, axis, o)
    still = [*range(3, 7), 8, *range(19, 23), 24, *range(32, 64)]
    assert torch.equal(o[..., still], q[..., still]) and not torch.equal(o, q)


@pytest.mark.parametrize('adjacent', [False, True])
def test_inverse_is_the_gradient(adjacent):
    """<g, d/dx rope(x) dx> = <rope^T g, dx>: the inverse of the gradient equals the adjoint in FP64, and central differences of a
    linear map are its own values: rope(x + d) - rope(x - d) = 2 rope(d) up to roundings of the three calls."""
    from yanlongvla_amd import kernels as K
    x, _, pos, freq, axis = make(50, 3, 0, 64, 64, 2, FP, 2)
    g = torch.randn(x.shape, generator=torch.Generator(device=DEV).manual_seed(8), device=DEV)
    xd = x.double().cpu().requires_grad_()
    y, _ = reference(xd, pos, freq, axis, adjacent, False)
    y.backward(g.double().cpu())
    o = torch.empty_like(g)
    K.rope_axes(g, None, pos, freq, axis, o, adjacent=adjacent, inverse=True)
    check(o, xd.grad, reference(g, pos, freq, axis, adjacent, True)[1])
    d = torch.randn_like(x) * 0.25
    call = lambda t: K.rope_axes(t, None, pos, freq, axis, torch.empty_like(t), adjacent=adjacent)[0].double()   # noqa: E731
    diff, lin = call(x + d) - call(x - d), 2 * call(d)
    mag = reference(x.abs() + d.abs(), pos, freq, axis, adjacent, False)[1].to(DEV)
    assert ((diff - lin).abs() <= 4 * 2.0 ** -21 * mag).all()


def test_not_finite_values_stay_in_their_pair():
    from yanlongvla_amd import kernels as K
    q, _, pos, freq, axis = make(4, 2, 0, 64, 64, 1, BF, 4)
    clean = torch.empty_like(q)
    K.rope_axes(q, None, pos, freq, axis, clean)
    q[1, 0, 5], q[2, 1, 40] = float('nan'), float('inf')
    o = torch.empty_like(q)
    K.rope_axes(q, None, pos, freq, axis, o)
    hit = torch.zeros_like(q, dtype=torch.bool)
    hit[1, 0, [5, 37]] = hit[2, 1, [8, 40]] = True
    assert torch.equal(o[~hit], clean[~hit]) and o[1, 0, [5, 37]].isnan().all() and not o[2, 1, [8, 40]].isfinite().all()


def test_no_tokens_and_graph_replays():
    from yanlongvla_amd import kernels as K
    q, k, pos, freq, axis = make(20, 4, 2, 128, 128, 3, BF, 6)
    K.rope_axes(q[:0], k[:0], pos[:, :0], freq, axis)
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    K.rope_axes(q, k, pos, freq, axis, qo, ko)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        K.rope_axes(q, k, pos, freq, axis, qo, ko)
    for i in range(3):
        pos.add_(17 + i)
        gr.replay()
        torch.cuda.synchronize()
        got = qo.clone(), ko.clone()
        K.rope_axes(q, k, pos, freq, axis, qo, ko)
        assert torch.equal(got[0], qo) and torch.equal(got[1], ko)
