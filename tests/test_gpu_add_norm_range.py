"""GPU tests of kernels.add_norm_quantize at the ends of its range: rows of zeros without an eps, rows whose squares leave FP32."""
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


@pytest.mark.parametrize('dt', [BF, HF, FP])
@pytest.mark.parametrize('K', [1024, 1021, 8])
@pytest.mark.parametrize('eps', [0.0, 1e-6])
def test_rows_of_zeros_have_scale_one(K, dt, eps):
    """Also without an eps, where a row of zeros is divided by zero: scale 1, codes 0; the rows beside it are as ever, to the FP32
    roundings of 2e-6 (scale) and 0.50003 (codes)."""
    from yanlongvla_amd import kernels as Kn
    x = torch.randn(6, K, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).to(dt)
    w = torch.randn(K, generator=torch.Generator(device=DEV).manual_seed(2), device=DEV).mul(0.2).to(dt)
    r = -x
    r[2:] = x[2:]
    x[1] = r[1] = 0
    q, s, h = torch.full((6, K), 9, dtype=torch.int8, device=DEV), torch.zeros(6, device=DEV), torch.empty_like(x)
    Kn.add_norm_quantize(x, r, w, eps, q, s, h)
    assert (s[:2] == 1).all() and (q[:2] == 0).all() and (h[:2] == 0).all()
    f = h[2:].double()
    n = f / (f.square().mean(1, keepdim=True) + eps).sqrt() * (w.double() + 1)
    want = n.abs().amax(1) / 127
    assert ((s[2:].double() - want).abs() <= 2e-6 * want).all() and ((q[2:].double() - n / want[:, None]).abs() <= 0.50003).all()
