"""CPU test: pages that are written may not share their rows; every other layout goes on to the device check (host tensors end there)."""
import pytest
import torch

from yanlongvla_amd import kernels as K
from yanlongvla_amd._lib import TcqError

P, H, T, D = 4, 2, 16, 64


def append(k, v):
    rows, ints = torch.zeros(2, H, D, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int32)
    K.paged_append((k, v), rows, rows, torch.zeros(2, 1, dtype=torch.int32), ints, ints)


def view(strides):
    return torch.zeros(200000, dtype=torch.bfloat16).as_strided((P, H, T, D), (*strides, 1))


@pytest.mark.parametrize('strides', [
    (T * D, T * D, D), (H * T * D, 0, D), (0, T * D, D), (H * T * D, T * D, 0),      # pages and heads that are the same, expanded axes
    (H * T * D, T * D, D - 8), (H * T * D, (T - 1) * D, D), (T * D, T * D + 8, D),   # windows: of rows, heads, pages
    (H * T * D - 64, T * D, D), (T * H * D, D // 2, H * D), (T * H * D, D, H * D - 8), (D, P * D, (H - 1) * P * D),
])
def test_rows_that_overlap(strides):
    for pages in ((view(strides), view((H * T * D, T * D, D))), (view((H * T * D, T * D, D)), view(strides))):
        with pytest.raises(ValueError, match='overlap'):
            append(*pages)


@pytest.mark.parametrize('strides', [
    (H * T * D, T * D, D), (2 * H * T * D + 8, T * D + 8, D), (H * T * 72, T * 72, 72), (T * H * D, D, H * D), (D, P * D, H * P * D), (T * D, P * T * D, D),
])
def test_rows_apart(strides):
    with pytest.raises(TcqError):
        append(view(strides), view(strides))


def test_keys_and_values_in_one_place():
    same = view((H * T * D, T * D, D))
    with pytest.raises(ValueError, match='overlap'):
        append(same, same)
    assert K._rows_apart((1, 1, 1, D), (0, 0, 0, 1)) and not K._rows_apart((2, 1, 16, D), (D, 5, D, 1))
