"""bf16 rows of two keys, the later one the larger by less than the 2^8 that a lagging running maximum would let a weight
grow to: the largest weight is exactly 1, so what it multiplies reaches the output without a rounding of its own."""

import torch
import pytest

from tests import test_gpu_latent_expanded as expanded
from tests.latent_helpers import call, paged
from tests.test_gpu_latent_forms import expanded_form, form_of

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def leads(rows):
    """Lead of the later key over the earlier one in each row, up to e^5.4 < 2^8: bf16 values."""
    return torch.linspace(0.05, 5.4, rows, dtype=torch.float64).to(BF16).double()


def check(got, lead):
    """The later key's values are 1, the earlier one's 0. The smaller weight times 0 is 0, the larger one is exactly 1 and
    the rest float32: the output is its value in [1/2, 1) rounded once, to a multiple of 2^-8."""
    want = 1 / (1 + (-lead).exp())
    bound = 2.0 ** -9 + 2.0 ** -16
    weight = lead.exp().float().to(BF16).double()  # as a weight of a lagging maximum
    lagging = (weight / (1 + lead.exp())).to(BF16).double()
    assert ((lagging - want).abs() > 1.2 * bound).sum() >= 5, "the rows could not tell a rounded largest weight"
    off = (got.cpu().double() - want).abs()
    assert off.max() <= bound, off.max().item()


@pytest.mark.parametrize("H", [64, 128])
@pytest.mark.parametrize("L", [128, 256, 512])
def test_absorbed(device, H, L):
    t = paged(device, [1], [200], H=H, L=L, R=64, page=64)
    assert form_of(t)[0] == H
    t["kv_cache"].zero_()
    t["kv_cache"][..., 1] = -1  # every other key: a score of -64
    rows = t["block_table"][0].long()
    for at, columns in ((5, {1: 0.0}), (150, {0: 1.0, 1: 0.0, 2: 1.0})):
        for column, value in columns.items():
            t["kv_cache"][rows[at // 64], at % 64, 0, column] = value
    lead = leads(H)
    t["q"].zero_()
    t["q"][0, :, 0] = lead.to(device)
    t["q"][0, :, 1] = 64
    t["q_rope"].zero_()
    check(call(t, 1.0)[0, :, 2], lead)


@pytest.mark.parametrize("nq,nk,H,form", [([64], [200], 1, [64, 1]), ([1000, 770], [1000, 900], 64, [128, 1]),
                                          ([1900], [1901], 64, [256, 1]), ([90], [1700], 3, [64, None])])
def test_expanded(device, nq, nk, H, form):
    causal = len(nq) > 1
    got_form = expanded_form(nq, nk, H, causal)
    assert got_form[0] == form[0] and (got_form[1] > 1 if form[1] is None else got_form[1] == form[1])
    t = expanded.inputs(device, nq, nk, H=H)
    for name in ("q", "k_nope", "k_rope", "v"):
        t[name].zero_()
    t["k_nope"][..., 1] = -1
    t["q"][..., 1] = 64
    start = 0
    for n in nk:
        t["k_nope"][start + 5, :, 1] = 0
        t["k_nope"][start + 150, :, 1] = 0
        t["k_nope"][start + 150, :, 0] = 1
        t["v"][start + 150] = 1
        start += n
    lead = leads(sum(nq))
    t["q"][..., 0] = lead.to(device)[:, None]
    out = expanded.call(t, causal, scale=1.0)
    start = 0
    for q, k in zip(nq, nk):
        first = max(0, 151 - (k - q)) if causal else 0  # queries that see both keys
        rows = slice(start + first, start + q)
        for h in {0, H - 1}:
            for column in (0, 127):
                check(out[rows, h, column], lead[rows])
        start += q
