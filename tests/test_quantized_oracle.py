"""CPU checks of the definitions of the 8-bit paged cache against torch's own conversions and by hand."""

import math

import numpy as np
import pytest
import torch

from oracle import quantized_reference as qr


def test_rounding_of_codes():
    gen = torch.Generator().manual_seed(0)
    x = torch.cat([torch.randn(100000, generator=gen) * 100, torch.randn(10000, generator=gen) * 0.01,
                   torch.tensor([0.0, -0.0, 448, 449, 464, 1e9, -1e9, 2.0 ** -10, 3 * 2.0 ** -10, 17, 19, 18, math.nan])])
    e4m3 = x.clamp(-448, 448).to(torch.float8_e4m3fn).float().double().numpy()
    assert np.array_equal(qr.nearest(x.double().numpy(), torch.float8_e4m3fn), e4m3, equal_nan=True)
    int8 = x.nan_to_num(0.0).clamp(-127, 127).round().double().numpy()
    assert np.array_equal(qr.nearest(x.double().numpy(), torch.int8), int8)


@pytest.mark.parametrize("top,dtype,scale", [
    (448.0, torch.float8_e4m3fn, 1.0), (448.5, torch.float8_e4m3fn, 2.0), (224.0, torch.float8_e4m3fn, 0.5), (0.0, torch.int8, 2.0 ** -80),
    (127.0, torch.int8, 1.0), (128.0, torch.int8, 2.0), (63.5, torch.int8, 0.5), (1e-30, torch.int8, 2.0 ** -80),
])
def test_scale_of_a_block(top, dtype, scale):
    rows = np.array([[0.0, -top, math.inf, math.nan]])
    assert qr.needed_scale(rows, dtype) == scale


def test_a_block_rounded_anew():
    codes = np.zeros((1, 16, 1, 2))
    codes[0, 0, 0] = 100, -3
    scale = np.ones((1, 1, 1))
    qr.append(torch.tensor([[[1016.0, -12.0]]]), (codes, torch.int8), scale, torch.tensor([[0]]), [0, 1], [2])
    assert scale[0, 0, 0] == 8 and codes[0, 0, 0].tolist() == [12, 0] and codes[0, 1, 0].tolist() == [127, -2]


def test_fork_by_hand():
    # Two beams of 20 tokens on pages of 16: beam 1 dies, beam 0 goes on twice.
    rows, counts, source, destination, missing = qr.fork([[0, 1], [0, 2]], [2, 1, 1, 0], [0, 0], [20, 20], 16, 0)
    assert rows == [[0, 1], [0, 2]] and counts == [2, 1, 1, 0] and source == [-1, 1] and destination == [-1, 2] and missing == 0


def test_compaction_by_hand():
    assert qr.compact([[5, 0, -1]], [1, 0, 0, 0, 0, 2]) == ([[1, 0, -1]], [1, 2, 0, 0, 0, 0], [(5, 1)])
