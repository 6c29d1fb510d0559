"""Absorbed latent attention over a paged cache against its float64 definition: lengths, pages, head counts, widths,
masks that leave rows empty, strides and refusals."""

import pytest
import torch

from tests.latent_helpers import B16, call, check, paged

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("L,R", [(128, 0), (128, 64), (256, 0), (256, 64), (512, 0), (512, 64)])
@pytest.mark.parametrize("H", [3, 64])
def test_widths_and_types(device, L, R, dtype, H):
    check(device, [1, 2], [45, 130], H=H, L=L, R=R, dtype=dtype, page=32)


@pytest.mark.parametrize("length", [1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 97, 128, 129, 500])
def test_lengths_of_one_token(device, length):
    check(device, [1], [length], H=16, L=512, R=64, page=16)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 1024])
def test_pages_that_end_inside_a_chunk(device, page):
    check(device, [1, 3, 1], [3 * page + 5, page, 70], H=8, L=256, R=64, page=page)


@pytest.mark.parametrize("H", [1, 5, 16, 20, 48, 63, 65, 128, 130])
def test_head_counts(device, H):
    check(device, [1, 4, 2], [50, 77, 33], H=H, L=128, R=64, page=16)


@pytest.mark.parametrize("causal", [True, False])
def test_chunks_of_prompts(device, causal):
    check(device, [70, 1, 33], [200, 40, 33], H=12, L=128, R=64, page=64, causal=causal)


def test_rows_that_see_nothing(device):
    """More tokens than rows: the first ones see none; a request without rows, one without tokens, and padding."""
    check(device, [5, 0, 3, 4], [2, 20, 0, 9], H=7, L=128, R=0, page=16, spare_tokens=6)


def test_every_row_empty(device):
    check(device, [2, 1], [0, 0], H=4, L=512, R=64, page=16)


@pytest.mark.parametrize("causal", [True, False])
def test_pages_outside_the_cache_hold_no_keys(device, causal):
    t = paged(device, [2, 1, 1], [150, 90, 40], H=6, L=256, R=64, page=16, seed=3)
    blocks = t["kv_cache"].shape[0]
    t["block_table"][0, 0] = -1
    t["block_table"][0, 4:6] = blocks
    t["block_table"][0, 9] = 2**31 - 1
    t["block_table"][1, 5] = -(2**31)
    t["block_table"][2] = blocks + 5  # nothing left of the third
    check(device, [2, 1, 1], [150, 90, 40], tensors=t, causal=causal)


def test_lengths_beyond_the_table_are_cut(device):
    t = paged(device, [1, 2], [64, 64], H=4, L=128, R=64, page=16)
    t["seqused_kv"][0] = 64
    longer = dict(t, seqused_kv=torch.tensor([1000, 64], dtype=torch.int32, device=device))
    check(device, [1, 2], [64, 64], tensors=t)
    a, b = call(t, 0.1, causal=False), call(longer, 0.1, causal=False)
    assert torch.equal(a, b)


def test_strided_heads_first_queries_and_output(device):
    t = paged(device, [3, 2], [60, 41], H=10, L=256, R=64, page=16, heads_first=True)
    check(device, [3, 2], [60, 41], tensors=t)
    dense = call(dict(t, q=t["q"].contiguous(), q_rope=t["q_rope"].contiguous()), 0.05)
    out = torch.empty((10, 5, 256), dtype=torch.bfloat16, device=device).transpose(0, 1)
    assert torch.equal(call(t, 0.05, out=out), dense)
    both = torch.cat([t["q"], t["q_rope"]], dim=-1)  # one projection, its two parts as views
    assert torch.equal(call(dict(t, q=both[..., :256], q_rope=both[..., 256:]), 0.05), dense)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_sharp_and_flat_scores(device, dtype):
    """Scores of some hundreds (one key takes all) and of nearly zero; the running maximum grows along the keys."""
    t = paged(device, [2], [300], H=16, L=128, R=64, page=16, dtype=dtype, seed=5)
    ramp = torch.linspace(0.01, 4, 300, device=device)
    rows = t["block_table"][0].long()
    cache = t["kv_cache"][rows].view(-1, 192)
    cache[:300] *= ramp[:, None].to(cache.dtype)
    t["kv_cache"][rows] = cache.view(rows.numel(), 16, 1, 192)
    for scale in (1.0, 1e-4):
        check(device, [2], [300], tensors=t, scale=scale, dtype=dtype)


def test_long_context_beyond_32_bit_offsets(device):
    """Pages past 2^32 bytes and 2^31 elements of the cache."""
    L, R, page = 512, 64, 128
    blocks = (2**32 // (page * (L + R))) + 40
    cache = torch.empty((blocks, page, 1, L + R), dtype=torch.bfloat16, device=device)
    small = paged(device, [1, 3], [700, 260], H=16, L=L, R=R, page=page, spare_pages=0)
    used = small["kv_cache"].shape[0]
    far = blocks - 1 - torch.arange(used, device=device)
    cache[far] = small["kv_cache"]
    table = small["block_table"].long()
    moved = torch.where(table >= 0, far[table.clamp(min=0)], table).to(torch.int32)
    assert torch.equal(call(small, 0.05), call(dict(small, kv_cache=cache, block_table=moved), 0.05))


def test_calls_repeat_bit_for_bit_on_another_stream(device):
    t = paged(device, [1, 6, 2], [900, 300, 40], H=32, L=512, R=64, page=64)
    first = call(t, 0.07)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        second = call(t, 0.07)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(first, second) and torch.equal(first, call(t, 0.07))


def test_two_captured_calls_follow_their_inputs(device):
    """Two graphs of different sizes, replayed in turn with eager work between; lengths change between replays."""
    a = paged(device, [1, 1, 1], [700, 90, 33], H=16, L=512, R=64, page=64, seed=1)
    b = paged(device, [4, 2], [500, 120], H=64, L=512, R=64, page=64, seed=2)
    graphs, outs = [], []
    for t in (a, b):
        call(t, 0.06)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(call(t, 0.06))
        graphs.append(graph)
    for step in range(3):
        for t, graph, out in zip((a, b), graphs, outs):
            t["q"].normal_()
            t["seqused_kv"] -= step
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, call(t, 0.06)), step


def test_custom_op(device):
    import ascendflow_amd.sparse_attention  # noqa: F401

    t = paged(device, [1, 2], [40, 70], H=8, L=128, R=64, page=16)
    args = (t["q"], t["q_rope"], t["kv_cache"], t["block_table"], t["cu_seqlens_q"], t["seqused_kv"], 0.1)
    out, lse = torch.ops.ascendflow_amd.latent_attention(*args)
    want = torch.empty_like(lse)
    assert torch.equal(out, call(t, 0.1, lse=want)) and torch.equal(lse, want)


def test_no_tokens(device):
    t = paged(device, [0], [10], H=8, L=128, R=64, page=16)
    assert call(t, 0.1).shape == (0, 8, 128)


@pytest.mark.parametrize("name,change", [
    ("q", lambda t: t["q"].float()),
    ("q", lambda t: t["q"][..., :100]),
    ("q", lambda t: t["q"].transpose(1, 2).contiguous().transpose(1, 2)),
    ("q", lambda t: t["q"].cpu()),
    ("q_rope", lambda t: t["q_rope"][:, :3]),
    ("q_rope", lambda t: None),
    ("q_rope", lambda t: t["q_rope"].to(torch.float16)),
    ("kv_cache", lambda t: t["kv_cache"][:, :10].contiguous()),
    ("kv_cache", lambda t: t["kv_cache"][:, ::2]),
    ("kv_cache", lambda t: t["kv_cache"].half()),
    ("block_table", lambda t: t["block_table"].long()),
    ("block_table", lambda t: t["block_table"][:, :0]),
    ("cu_seqlens_q", lambda t: t["cu_seqlens_q"][:-1]),
    ("seqused_kv", lambda t: t["seqused_kv"].cpu()),
])
def test_refusals(device, name, change):
    t = paged(device, [1, 2], [40, 70], H=8, L=128, R=64, page=16)
    with pytest.raises(ValueError):
        call(dict(t, **{name: change(t)}), 0.1)


def test_refused_outputs_and_scales(device):
    t = paged(device, [1, 2], [40, 70], H=8, L=128, R=64, page=16)
    for scale in (0.0, -1.0):
        with pytest.raises(ValueError):
            call(t, scale)
    with pytest.raises(ValueError, match="overlap"):
        call(t, 0.1, out=t["q"])
    with pytest.raises(ValueError, match="overlap"):
        call(t, 0.1, out=torch.empty((3, 1, 128), dtype=torch.bfloat16, device=device).expand(3, 8, 128))
    with pytest.raises(ValueError):
        call(t, 0.1, out=torch.empty((3, 8, 64), dtype=torch.bfloat16, device=device))
    with pytest.raises(ValueError):
        call(t, 0.1, lse=torch.empty((3, 8), dtype=torch.float64, device=device))
    odd = torch.empty(3 * 8 * 128 + 1, dtype=torch.bfloat16, device=device)[1:].view(3, 8, 128)
    with pytest.raises(ValueError, match="16-byte"):
        call(t, 0.1, out=odd)
    assert B16["bf16"] is torch.bfloat16
