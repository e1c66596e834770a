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


def test_outputs_whose_rows_overlap_are_refused():
    """In place on heads or tokens that are one and the same memory (an expanded tensor, windows of a row) every row would be turned several
    times at once; as inputs with an output of their own they are taken (and end at the host tensors here)."""
    M, D = 3, 64
    pos = torch.zeros(1, M, dtype=torch.int32)
    freq, axis = K.rope_frequencies(D)
    q, k = torch.zeros(M, 4, D), torch.zeros(M, 1, D)
    row = torch.zeros(M * 4 * D)
    overlapping = [k.expand(M, 4, D), torch.zeros(1, 4, D).expand(M, 4, D), torch.zeros(1, 1, D).expand(M, 4, D),
                   row.as_strided((M, 4, D), (4 * D, D // 2, 1)), row.as_strided((M, 4, D), (D, D, 1)), row.as_strided((M, 4, D), (3 * D, D, 1))]
    for t in overlapping:
        with pytest.raises(ValueError):
            K.rope_axes(t, None, pos, freq, axis)
        with pytest.raises(ValueError):
            K.rope_axes(q, t, pos, freq, axis)
        with pytest.raises(ValueError):
            K.rope_axes(q, q, pos, freq, axis, t, q)
        with pytest.raises(ValueError):
            K.rope_axes(q, q, pos, freq, axis, q, t)
        with pytest.raises(_lib.TcqError):
            K.rope_axes(t, t, pos, freq, axis, torch.empty_like(q), torch.empty_like(q))
    for t in (q, k, q.transpose(0, 1).contiguous().transpose(0, 1), torch.zeros(M, 4, 2 * D)[..., :D], torch.zeros(M, 12, D)[:, 4:8],
              torch.zeros(4, 1, M * D).as_strided((M, 4, D), (D, M * D, 1)), torch.zeros(1, 4, D).expand(1, 4, D)):
        with pytest.raises(_lib.TcqError):
            K.rope_axes(t, None, pos[:, :t.shape[0]], freq, axis)
    x, w, codes, s = torch.zeros(2, D), torch.zeros(D), torch.zeros(2, D, dtype=torch.int8), torch.zeros(2)
    for t in (torch.zeros(1, D).expand(2, D), torch.zeros(2 * D).as_strided((2, D), (D // 2, 1))):
        with pytest.raises(ValueError):
            K.add_norm_quantize(x, t, w, 1e-6, codes, s, t)
        with pytest.raises(_lib.TcqError):
            K.add_norm_quantize(t, t, w, 1e-6, codes, s, x)
    with pytest.raises(_lib.TcqError):
        K.add_norm_quantize(x[:1], x[:1], w, 1e-6, codes[:1], s[:1], torch.zeros(1, D).expand(1, D))


def test_frequencies_of_no_whole_pairs_or_other_sections_are_refused():
    for R in (65, 1, 0, -2):
        with pytest.raises(ValueError):
            K.rope_frequencies(R)
    for sections in ((10, 27, 27), (1, 2, 29), (0, 32)):              # interleaved, an axis would come out with other than its pairs
        with pytest.raises(ValueError):
            K.rope_frequencies(2 * sum(sections), sections=sections, interleaved=True)
        assert K.rope_frequencies(2 * sum(sections), sections=sections)[1].bincount(minlength=3).tolist()[:len(sections)] == list(sections)
    for sections in ((24, 20, 20), (32, 32), (3, 3, 2), (22, 21, 21), (8,)):
        axis = K.rope_frequencies(2 * sum(sections), sections=sections, interleaved=True)[1]
        assert [int((axis == a).sum()) for a in range(len(sections))] == list(sections)
