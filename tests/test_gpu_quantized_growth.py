"""Blocks of an 8-bit cache filled token by token while their scales grow: how far codes may be from the values appended."""

import pytest
import torch

from ascendflow_amd.sparse_attention import append_quantized_kv
from tests.quantized_helpers import CODES

pytestmark = pytest.mark.gpu


def append(device, x, codes, step):
    """Tokens x [T, 1, D] into one page of 64, ``step`` tokens a call; (codes, scale)."""
    T, _, D = x.shape
    caches = [torch.zeros((1, 64, 1, D), dtype=CODES[codes], device=device) for _ in range(2)]
    scales = [torch.zeros((1, 1, 1), device=device) for _ in range(2)]
    table = torch.zeros((1, 1), dtype=torch.int32, device=device)
    for i in range(0, T, step):
        n = min(step, T - i)
        cu, used = (torch.tensor(v, dtype=torch.int32, device=device) for v in ([0, n], [i + n]))
        append_quantized_kv(x[i:i + n], -x[i:i + n], *caches, *scales, table, cu, used)
    assert torch.equal(caches[0].float(), -caches[1].float()) and torch.equal(*scales)
    return caches[0][0, :T, 0].double(), scales[0].item()


def test_int8_codes_depend_on_how_a_block_was_filled(device):
    """5.40625 is code 5 at a scale of 1 and then, of 2.5, code 2 at a scale of 2; in one call it is code 3."""
    x = torch.zeros((2, 1, 16), dtype=torch.bfloat16, device=device)
    x[0, 0, :2] = torch.tensor([100.0, 5.40625])
    x[1, 0, 0] = 250.0
    whole, by_token = append(device, x, "int8", 2), append(device, x, "int8", 1)
    assert whole[1] == by_token[1] == 2 and whole[0][0, 1] == 3 and by_token[0][0, 1] == 2


@pytest.mark.parametrize("codes", ["int8", "e4m3"])
@pytest.mark.parametrize("step", [1, 3, 64])
@pytest.mark.parametrize("growth", [1.0, 1.3, 2.0, 3.7])
def test_distance_after_any_number_of_growths(device, codes, step, growth):
    """A scale grows by powers of two, and each time a code is rounded by half a step of int8, or of e4m3's subnormals (2^-9),
    in units of the scale of then: over all times less than twice the last one's, s or 2^-9 s. e4m3's first rounding is half
    a step of 2^-3 of the value besides."""
    gen = torch.Generator().manual_seed(7)
    x = torch.randn((64, 1, 64), generator=gen) * growth ** (torch.arange(64.0) / 4)[:, None, None]
    x = x.bfloat16().to(device)
    got, scale = append(device, x, codes, step)
    off, exact = (got * scale - x[:, 0].double()).abs(), x[:, 0].double().abs()
    assert (off <= (scale if codes == "int8" else exact * 2 ** -4 + scale * 2 ** -9)).all()
    if step == 64:  # once
        assert (off <= (scale / 2 if codes == "int8" else exact * 2 ** -4 + scale * 2 ** -10)).all()
