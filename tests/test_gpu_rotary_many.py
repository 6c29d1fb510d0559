"""More tokens than a launch has workgroups along one dimension."""

import torch
import pytest

from ascendflow_amd.sparse_attention import append_paged_kv, apply_rotary, rotary_frequencies

pytestmark = pytest.mark.gpu
T = (1 << 27) + 21  # over 2^24 workgroups of 8 tokens


def test_rotary(device):
    """A quarter turn a position: (1, 0) goes to (1, 0), (0, 1), (-1, 0), (0, -1)."""
    x = torch.zeros((T, 1, 2), dtype=torch.bfloat16, device=device)
    x[:, 0, 0] = 1
    frequencies = torch.full((1,), torch.pi / 2, dtype=torch.float64, device=device)
    positions = torch.arange(T, dtype=torch.int32, device=device)
    apply_rotary(x, positions, frequencies, out=x)
    quarter = positions % 4
    # The angle is exact to 2^-25 turns at these positions: cosines and sines of 0 within 2^-20.
    for column, want in ((0, [1, 0, -1, 0]), (1, [0, 1, 0, -1])):
        want = torch.tensor(want, device=device, dtype=torch.float32)[quarter.long()]
        assert (x[:, 0, column].float() - want).abs().max() <= 2.0 ** -20


def test_append(device):
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=device)
    page = 1 << 20
    pages = T // page + 1
    rows = torch.randint(-128, 128, (T, 1, 1), dtype=torch.int8, device=device).to(torch.bfloat16)
    cache = torch.full((pages, page, 1, 1), 200.0, dtype=torch.bfloat16, device=device)
    append_paged_kv(rows, cache, torch.arange(pages, dtype=torch.int32, device=device)[None], i32(0, T), i32(T))
    assert torch.equal(cache.view(-1)[:T], rows.view(-1)) and (cache.view(-1)[T:] == 200).all()
