"""Tensors that a call writes count a new version: a backward pass that saved one of them raises, as after torch's own
operations in place, and does not go on with the new values."""

import pytest
import torch

from ascendflow_amd.sparse_attention import append_paged_kv, apply_rotary, rotary_frequencies
from tests import test_gpu_latent_expanded as expanded
from tests.latent_helpers import call, paged

pytestmark = pytest.mark.gpu


def check(written, run):
    weight = torch.ones_like(written).requires_grad_(True)
    saved = (weight * written).sum()
    before = written._version
    run()
    assert written._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        saved.backward()
    with torch.inference_mode():
        run()


@pytest.mark.parametrize("place", ["in place", "apart", "a part"])
def test_rotary(device, place):
    x = torch.randn((5, 2, 64), device=device).bfloat16()
    positions, frequencies = torch.arange(5, device=device), rotary_frequencies(32, device=device)
    out = x if place == "in place" else torch.zeros_like(x)
    part = out[..., :32] if place == "a part" else out
    given = x[..., :32] if place == "a part" else x
    check(out, lambda: apply_rotary(given, positions, frequencies, out=part))


def test_nothing_is_counted_where_nothing_is_written(device):
    x = torch.randn((5, 2, 64), device=device).bfloat16()
    positions, frequencies = torch.arange(5, device=device), rotary_frequencies(32, device=device)
    apply_rotary(x, positions, frequencies)
    apply_rotary(x[:0], positions[:0], frequencies, out=x[:0])
    assert x._version == 0 and positions._version == 0


@pytest.mark.parametrize("which", ["k_cache", "v_cache"])
def test_append(device, which):
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=device)
    rows = torch.randn((3, 2, 64), device=device).bfloat16()
    caches = dict(k_cache=torch.zeros((2, 16, 2, 64), dtype=torch.bfloat16, device=device),
                  v_cache=torch.zeros((2, 16, 2, 64), dtype=torch.bfloat16, device=device))
    check(caches[which], lambda: append_paged_kv(rows, block_table=i32(1, 0)[None], cu_seqlens_q=i32(0, 3), seqused_kv=i32(20),
                                                 v=rows, **caches))


@pytest.mark.parametrize("form", ["absorbed", "expanded"])
def test_attention(device, form):
    if form == "absorbed":
        t = paged(device, [1, 2], [40, 70], H=8, page=64)
        run = lambda out, lse: call(t, 0.1, True, out, lse)
        out = torch.zeros_like(t["q"])
    else:
        t = expanded.inputs(device, [5, 3], [40, 30], H=8)
        run = lambda out, lse: expanded.call(t, out=out, softmax_lse=lse)
        out = torch.zeros((8, 8, 128), dtype=torch.bfloat16, device=device)
    lse = torch.zeros(out.shape[:2], device=device)
    check(out, lambda: run(out, None))
    check(lse, lambda: run(None, lse))
