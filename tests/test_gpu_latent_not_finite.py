"""Queries whose scores are not numbers or overflow: NaN in output and softmax_lse, never the -inf of a query that sees no
key, and nothing in any other row."""

import math

import pytest
import torch

from tests import test_gpu_latent_expanded as expanded
from tests.latent_helpers import call, paged

pytestmark = pytest.mark.gpu

# bf16 reaches 3e38: against keys of 2^60 the products overflow.
POISON = {"nan": math.nan, "inf": math.inf, "overflow": 2.0 ** 100}


def check(run, q, tokens, value):
    """``run(q)`` is (out, lse); the rows ``tokens`` (token, head) of q get ``value`` in their first column."""
    out, lse = run(q)
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()
    poisoned = q.clone()
    bad = torch.zeros(lse.shape, dtype=torch.bool, device=q.device)
    for t, h in tokens:
        poisoned[t, h, 0] = value
        bad[t, h] = True
    got, got_lse = run(poisoned)
    assert torch.isnan(got[bad]).all() and torch.isnan(got_lse[bad]).all()
    assert torch.equal(got[~bad], out[~bad]) and torch.equal(got_lse[~bad], lse[~bad])


@pytest.mark.parametrize("value", POISON)
@pytest.mark.parametrize("counts,lengths,H,L", [
    ([1], [4000], 16, 512),               # parts of one tile, joined by 16 waves
    ([1, 2], [700, 65], 128, 256),        # 128-row tiles
    ([1] * 20 + [4] * 20, [300] * 40, 64, 512),  # joined by one wave, or whole
    ([230], [260], 128, 128),             # a tile a workgroup
])
def test_absorbed(device, counts, lengths, H, L, value):
    t = paged(device, counts, lengths, H=H, L=L, page=64)
    t["kv_cache"][..., 0] = 2.0 ** 60 if value == "overflow" else 1.0
    t["q"][..., 0] = 0.0

    def run(q):
        out, lse = torch.empty_like(q), torch.empty(q.shape[:2], device=device)
        call(dict(t, q=q), 0.05, True, out, lse)
        return out, lse

    rows = [(0, 0), (0, H - 1), (sum(counts) - 1, H // 2)]
    check(run, t["q"], rows, POISON[value])


@pytest.mark.parametrize("value", POISON)
@pytest.mark.parametrize("nq,nk,H", [([300, 45], [300, 333], 20), ([1, 20], [2500, 900], 3), ([600], [600], 128)])
def test_expanded(device, nq, nk, H, value):
    t = expanded.inputs(device, nq, nk, H=H)
    t["k_nope"][..., 0] = 2.0 ** 60 if value == "overflow" else 1.0
    t["q"][..., 0] = 0.0

    def run(q):
        out, lse = torch.empty(q.shape[0], H, 128, dtype=q.dtype, device=device), torch.empty(q.shape[:2], device=device)
        expanded.call(dict(t, q=q), out=out, softmax_lse=lse)
        return out, lse

    check(run, t["q"], [(0, 0), (sum(nq) - 1, H - 1), (sum(nq) // 2, H // 2)], POISON[value])
