"""Expanded latent attention of ragged prompts against its float64 definition."""

import math

import pytest
import torch

from ascendflow_amd.flash_attention import latent_attention_expanded
from oracle import latent_reference as lr
from tests.latent_helpers import B16, compare

pytestmark = pytest.mark.gpu
SCALE = 192 ** -0.5


def inputs(device, nq, nk, H=3, dtype="bf16", seed=0, spare=0):
    gen = torch.Generator().manual_seed(seed)
    b16 = B16[dtype]
    offsets = lambda n: torch.tensor([0] + [sum(n[:i + 1]) for i in range(len(n))], dtype=torch.int32).to(device)
    Tq, Tk = sum(nq) + spare, sum(nk) + spare
    normal = lambda *shape: torch.randn(shape, generator=gen).to(b16).to(device)
    both = normal(Tk, H, 256)
    t = dict(q=normal(Tq, H, 192), k_nope=both[..., :128], k_rope=normal(Tk, 64), v=both[..., 128:], cu_q=offsets(nq),
             cu_k=offsets(nk))
    if spare:  # keys and values behind the last request are not read
        both[sum(nk):] = math.nan
        t["k_rope"][sum(nk):] = math.nan
    return t


def call(t, causal=True, scale=SCALE, **kw):
    return latent_attention_expanded(t["q"], t["k_nope"], t["k_rope"], t["v"], t["cu_q"], t["cu_k"], SCALE=scale,
                                     CAUSAL=causal, **kw)


def check(device, nq, nk, causal=True, scale=SCALE, tensors=None, **kw):
    t = inputs(device, nq, nk, **kw) if tensors is None else tensors
    dtype = t["q"].dtype
    Tq, H = t["q"].shape[:2]
    out = torch.full((Tq, H, 128), 7.0, dtype=dtype, device=device)
    lse = torch.full((Tq, H), 7.0, device=device)
    assert call(t, causal, scale, out=out, softmax_lse=lse) is out
    cpu = {k: v.cpu() for k, v in t.items()}
    expected = lr.latent_attention_expanded(*(cpu[k] for k in ("q", "k_nope", "k_rope", "v", "cu_q", "cu_k")), scale, causal)
    values = cpu["v"][torch.isfinite(cpu["v"])].abs().max().item() if sum(nk) else 0.0
    compare(out.cpu(), lse.cpu(), expected, dtype, max(1, *nk, 1), values)
    assert (out[sum(nq):] == 7).all() and (lse[sum(nq):] == 7).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 129, 255, 256, 257, 600])
def test_prompts(device, n, causal, dtype):
    check(device, [n], [n], causal, H=2, dtype=dtype)


@pytest.mark.parametrize("causal", [True, False])
def test_ragged_chunks_behind_context(device, causal):
    check(device, [70, 1, 0, 300, 5], [200, 130, 40, 300, 64], causal, H=5, spare=9)


def test_queries_that_see_nothing(device):
    """More queries than keys, no keys at all, and all of it at once."""
    check(device, [90, 3, 8], [20, 0, 8], H=2)
    check(device, [4], [0], H=2)
    check(device, [4], [0], causal=False, H=2)


@pytest.mark.parametrize("H", [1, 8, 17])
def test_head_counts(device, H):
    check(device, [33, 20], [40, 90], H=H)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_sharp_and_flat_scores(device, dtype):
    t = inputs(device, [130], [400], dtype=dtype, seed=4)
    t["k_nope"] *= torch.linspace(0.01, 4, 400, device=device)[:, None, None].to(t["q"].dtype)
    for scale in (1.0, 1e-4):
        check(device, [130], [400], tensors=t, scale=scale)


def test_strides(device):
    t = inputs(device, [40], [70], H=4)
    dense = call({k: v.contiguous() for k, v in t.items()})
    assert torch.equal(call(t), dense)
    first = lambda x: x.transpose(0, 1).contiguous().transpose(0, 1)
    out = torch.empty((4, 40, 128), dtype=torch.bfloat16, device=device).transpose(0, 1)
    assert torch.equal(call(dict(t, q=first(t["q"]), k_nope=first(t["k_nope"]), v=first(t["v"])), out=out), dense)
    wide = torch.zeros((70, 576), dtype=torch.bfloat16, device=device)
    wide[:, 512:] = t["k_rope"]
    assert torch.equal(call(dict(t, k_rope=wide[:, 512:])), dense)


def test_captured_call_follows_its_inputs(device):
    t = inputs(device, [300, 20], [300, 90], H=4)
    call(t)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(t)
    for _ in range(3):
        t["q"].normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call(t))


def test_custom_op(device):
    t = inputs(device, [10], [30])
    lse = torch.empty((10, 3), device=device)
    want = call(t, softmax_lse=lse)
    out, got = torch.ops.ascendflow_amd.latent_attention_expanded(t["q"], t["k_nope"], t["k_rope"], t["v"], t["cu_q"],
                                                                 t["cu_k"], SCALE)
    assert torch.equal(out, want) and torch.equal(got, lse)


@pytest.mark.parametrize("name,change", [
    ("q", lambda t: t["q"][..., :128]),
    ("q", lambda t: t["q"].float()),
    ("k_nope", lambda t: t["k_nope"][:, :2]),
    ("k_rope", lambda t: t["k_rope"][:5]),
    ("k_rope", lambda t: t["k_rope"].cpu()),
    ("v", lambda t: t["v"].half()),
    ("v", lambda t: t["v"].transpose(1, 2).contiguous().transpose(1, 2)),
    ("cu_k", lambda t: t["cu_k"][:-1]),
    ("cu_q", lambda t: t["cu_q"].long()),
])
def test_refusals(device, name, change):
    t = inputs(device, [10], [30])
    with pytest.raises(ValueError):
        call(dict(t, **{name: change(t)}))


def test_refused_outputs(device):
    t = inputs(device, [10], [30])
    with pytest.raises(ValueError):
        call(t, scale=0.0)
    with pytest.raises(ValueError, match="overlap"):
        call(t, out=t["q"][..., :128])
    with pytest.raises(ValueError, match="16-byte"):
        call(t, out=torch.empty(10 * 3 * 128 + 1, dtype=torch.bfloat16, device=device)[1:].view(10, 3, 128))
