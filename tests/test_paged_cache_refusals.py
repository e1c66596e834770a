"""CPU test of what a cache in pages refuses before it takes a page: sequences that it does not have."""
import pytest
import torch

from yanlongvla_amd import gemma
from yanlongvla_amd._lib import TcqError


@pytest.mark.parametrize('sequence', [-1, -3, 3, 1000])
def test_sequences_that_are_not_there(sequence):
    cache = gemma.PagedKVCache(2, 3, 8, 64, 'cpu', rows=16)
    rows = [torch.zeros(5, 64, dtype=torch.bfloat16)] * 2
    model = gemma.BackbonePolicy(layers=2, width=64, hidden=64, heads=1, head_dim=64, vocab=8)
    for call in (lambda: cache.extend(rows, rows, sequence), lambda: cache.chunk(sequence, 5),
                 lambda: model.prefill_chunk(torch.zeros(5, 64), cache, sequence)):
        with pytest.raises(IndexError):
            call()
    for there in (0, 2):
        with pytest.raises(TcqError):                                        # host tensors
            cache.extend(rows, rows, there)
