"""In place through another view of the same rows, whose one-entry dimensions have other strides."""

import pytest
import torch

from ascendflow_amd.sparse_attention import apply_rotary, rotary_frequencies

pytestmark = pytest.mark.gpu


def test_one_token_of_heads_first_rows(device):
    q = torch.randn((5, 1, 64), device=device).bfloat16()
    positions, frequencies = torch.tensor([77], device=device), rotary_frequencies(64, device=device)
    x, out = q.transpose(0, 1), q.view(1, 5, 64)
    assert x.stride() != out.stride()
    want = apply_rotary(x, positions, frequencies)
    assert apply_rotary(x, positions, frequencies, out=out) is out
    assert torch.equal(out, want)


def test_two_tokens_are_not_the_same_rows(device):
    q = torch.randn((5, 2, 64), device=device).bfloat16()
    positions, frequencies = torch.tensor([77, 78], device=device), rotary_frequencies(64, device=device)
    with pytest.raises(ValueError, match="overlap"):
        apply_rotary(q.transpose(0, 1), positions, frequencies, out=q.view(2, 5, 64))
