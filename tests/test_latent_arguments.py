"""CPU checks: operands that are no tensors are refused by name, whatever else the call has."""

import pytest
import torch

from ascendflow_amd.sparse_attention import apply_rotary, rotary_frequencies


@pytest.mark.parametrize("name", ["x", "positions", "frequencies", "out"])
@pytest.mark.parametrize("value", [[1.0], 3, None])
def test_rotary_operands(name, value):
    x = torch.zeros((3, 2, 64), dtype=torch.bfloat16)
    operands = dict(x=x, positions=torch.zeros(3, dtype=torch.int32), frequencies=rotary_frequencies(32, device="cpu"), out=x.clone())
    for leaf in (x, x.clone().requires_grad_(True)):
        with pytest.raises(ValueError, match="ROCm" if name == "out" and value is None else f"{name} must be a torch.Tensor"):
            apply_rotary(**{**operands, "x": leaf, name: value})
