"""CPU checks of what the rotary positions, the 8-bit cache behind the decoder layers and the norm to INT8 rows refuse, beside
test_layer8_refusals.py."""
import pytest
import torch

from yanlongvla_amd import _lib
from yanlongvla_amd import kernels as K


@pytest.mark.parametrize('rows', [65, 100, 968])
@pytest.mark.parametrize('causal', [False, True])
def test_rows_that_replace_each_other_are_a_block_at_most(rows, causal):
    cache = K.kv8_cache(1, 1, 64, 2000, 'cpu')
    before = [t.clone() for t in cache]
    q, k = torch.zeros(rows, 4 * 64, dtype=torch.bfloat16), torch.zeros(rows, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match='64'):
        K.KV8Rows(cache, torch.zeros(1, dtype=torch.int32)).core(q, k, k, 4, causal)
    assert all(torch.equal(a, b) for a, b in zip(cache, before))
    with pytest.raises(_lib.TcqError):                                 # 64 are taken (and end at the host tensors)
        K.KV8Rows(cache, torch.zeros(1, dtype=torch.int32)).core(q[:64], k[:64], k[:64], 4, causal)
