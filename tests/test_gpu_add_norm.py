"""GPU tests of kernels.add_norm_quantize against its definition in 64 bits: types, widths (vector and scalar path), strides, in place,
both forms of the weight, INT8 layouts, rows of zeros, rows that overflow or are not finite, the product that takes its rows.

Tolerances: h is one FP32 sum rounded to the type (exact comparison with the same two roundings). scale: FP32 sums of squares over at
most 32 values a lane and 10 further additions, so within 42 * 2^-24 / 2 of the root, plus five roundings: 2e-6 relative. A code is the
whole number next to n / scale, off by at most half plus 127 times three FP32 roundings: 0.50003."""
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


def inputs(M, K, dt, seed, offset=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    wide = torch.randn(K, generator=g, device=DEV).exp()
    return (torch.randn(M, K, generator=g, device=DEV).to(dt), (torch.randn(M, K, generator=g, device=DEV) * wide).to(dt),
            (torch.randn(K, generator=g, device=DEV) * 0.2 + 1 - offset).to(dt))


def outputs(M, K, dt):
    return (torch.full((M, K), -128, dtype=torch.int8, device=DEV), torch.full((M,), -1.0, device=DEV), torch.full((M, K), float('nan'), device=DEV).to(dt))


def check(x, r, w, eps, offset, q, scale, h):
    want = (x.float() + r.float()).to(x.dtype) if r is not None else x
    if h is not None:
        assert torch.equal(h, want)
    f = want.double()
    n = f / (f.square().mean(1, keepdim=True) + eps).sqrt() * (w.double() + offset)
    s = n.abs().amax(1) / 127
    assert ((scale.double() - s).abs() <= 2e-6 * s).all()
    assert ((q.double() - n / s[:, None]).abs() <= 0.50003).all() and (q.abs() <= 127).all()


@pytest.mark.parametrize('M,K', [(1, 1), (1, 2048), (3, 17), (2, 1152), (50, 1024), (968, 2048), (5, 4304), (700, 4304), (2, 16384), (520, 16384),
                                 (1, 32768), (600, 64), (513, 1000), (7, 2044)])
@pytest.mark.parametrize('dt', [BF, HF, FP])
def test_add_norm_quantize_matches_fp64(M, K, dt):
    from yanlongvla_amd import kernels as Kn
    for offset, add in ((1.0, True), (0.0, False)):
        x, r, w = inputs(M, K, dt, M + K, offset)
        q, s, h = outputs(M, K, dt)
        r = r if add else None
        Kn.add_norm_quantize(x, r, w, 1e-6, q, s, h if add else None, offset=offset)
        check(x, r, w, 1e-6, offset, q, s, h if add else None)


@pytest.mark.parametrize('K,pad', [(2048, 8), (2048, 3), (1152, 1)])
def test_strides_in_place_and_neighbours(K, pad):
    """Rows inside wider ones (aligned or not), the residual updated in place: the columns between the rows stay."""
    from yanlongvla_amd import kernels as Kn
    M = 9
    x0, r0, w = inputs(M, K, BF, 3)
    wide = torch.full((2, M, K + pad), 7.0, device=DEV).to(BF)
    x, r = wide[0, :, :K], wide[1, :, :K]
    x.copy_(x0), r.copy_(r0)
    q, s, _ = outputs(M, K, BF)
    Kn.add_norm_quantize(x, r, w, 1e-5, q, s, r)
    check(x0, r0, w, 1e-5, 1.0, q, s, r)
    assert (wide[:, :, K:] == 7).all() and torch.equal(x, x0)
    q2, s2, _ = outputs(M, K, BF)
    x1 = x0.clone()                                # the sum over the other input
    Kn.add_norm_quantize(x1, r0, w, 1e-5, q2, s2, x1)
    check(x0, r0, w, 1e-5, 1.0, q2, s2, x1)        # (another path sums in another order: its scale may differ in the last bit)


@pytest.mark.parametrize('M,K', [(5, 2048), (33, 1152), (16, 2064), (3, 48)])
def test_token_blocks_and_words_hold_the_same_codes(M, K):
    from yanlongvla_amd import kernels as Kn
    x, r, w = inputs(M, K, BF, 1)
    q, s, h = outputs(M, K, BF)
    tb = Kn.token_blocks(M, K, DEV).zero_()
    Kn.add_norm_quantize(x, r, w, 1e-6, q, s, h, q4=tb)
    assert torch.equal(Kn.rows_of_token_blocks(tb, M), q)
    words = torch.zeros(K // 4, M + 2, dtype=torch.int32, device=DEV)
    Kn.add_norm_quantize(x, r, w, 1e-6, None, s, h, q4=words)
    assert torch.equal(words[:, :M].t().contiguous().view(torch.int8).view(M, K), q) and (words[:, M:] == 0).all()


@pytest.mark.parametrize('K', [1024, 1021])
def test_rows_of_zeros_overflow_and_not_finite(K):
    from yanlongvla_amd import kernels as Kn
    x, r, w = inputs(8, K, FP, 2)
    x[0], r[0] = 0, 0                              # zeros
    x[1, 3] = float('nan')
    r[2, K - 1] = float('inf')
    x[3] = 1e30                                    # finite, its square is not: the FP32 norm is zero
    x[4, 0], r[4, 0] = float('inf'), float('-inf')
    q, s, h = outputs(8, K, FP)
    Kn.add_norm_quantize(x, r, w, 1e-6, q, s, h)
    assert s[0] == 1 and (q[0] == 0).all()
    assert s[1].isnan() and s[2].isnan() and s[4].isnan()
    assert s[3] == 1 and (q[3] == 0).all()
    check(x[5:], r[5:], w, 1e-6, 1.0, q[5:], s[5:], h[5:])


def test_feeds_the_int8_product_and_replays():
    """The rows go into gemm_i8 as they are; a captured pair of calls gives the eager result on every replay, on a stream of its own."""
    from yanlongvla_amd import kernels as Kn
    M, K, N = 70, 1024, 256
    x, r, w = inputs(M, K, BF, 4)
    q, s, h = outputs(M, K, BF)
    W = torch.randint(-127, 128, (N, K), generator=torch.Generator(device=DEV).manual_seed(5), device=DEV).to(torch.int8)
    sw = torch.full((N,), 0.01, device=DEV)
    y = torch.empty(M, N, dtype=BF, device=DEV)

    def both():
        Kn.add_norm_quantize(x, r, w, 1e-6, q, s, h)
        Kn.gemm_i8(q, W, y, sa=s, sw=sw)

    both()
    want = ((q.double() @ W.double().t()) * s.double()[:, None] * sw.double())
    assert ((y.double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-6 * want.abs().max()).all()
    st, gr = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(gr, stream=st):
        both()
    for _ in range(3):
        x.mul_(1.25)
        gr.replay()
        torch.cuda.synchronize()
        got = q.clone(), s.clone(), y.clone()
        both()
        assert all(torch.equal(a, b) for a, b in zip(got, (q, s, y)))
    Kn.add_norm_quantize(x[:0], None, w, 1e-6, q[:0], s[:0])
