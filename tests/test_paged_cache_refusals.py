"""CPU tests of what a cache in pages refuses before it takes a page: sequences that it does not have, a start that
is another operand, rows of other layers or sizes."""
import pytest
import torch

from yanlongvla_amd import gemma, kernels
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


def test_a_start_of_its_own():
    """Where it is take the rows to take would be gone after the call, and a replay take as many as there are."""
    pt, pool = kernels.page_table(2, 4, 8, 'cpu', 16), kernels.kv_pages(8, 1, 64, 'cpu', 16)
    take = torch.ones(2, dtype=torch.int32)
    for start in (take, take.view(2), pt.lens):
        with pytest.raises(ValueError, match='of its own'):
            kernels.pages_take(pt, pool, take, start)
    with pytest.raises(TcqError):                                            # host tensors
        kernels.pages_take(pt, pool, take, torch.zeros_like(take))


def test_rows_of_other_layers_or_sizes():
    cache = gemma.PagedKVCache(2, 3, 8, 64, 'cpu', rows=16, heads=2)
    one = torch.zeros(5, 128, dtype=torch.bfloat16)
    good = [one, one]
    for bad in ([], [one], [one] * 3, [one, one[:4]], [one, one[:, :64]], [one, one.half()], [one, one.float()]):
        for ks, vs in ((bad, bad), (good, bad), (bad, good)):
            with pytest.raises(ValueError):
                cache.extend(ks, vs, 0)
    with pytest.raises(TcqError):                                            # host tensors
        cache.extend(good, good, 0)
    model = gemma.BackbonePolicy(layers=3, width=64, hidden=64, heads=1, head_dim=64, vocab=8)
    with pytest.raises(ValueError):
        model.prefill_chunk(torch.zeros(5, 64), cache, 0)
