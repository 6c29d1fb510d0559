"""Attention over an 8-bit paged cache against its float64 definition: lengths, pages, blocks of scales, head layouts, widths,
types, masks that leave rows empty, strides and refusals."""

import math

import pytest
import torch

from oracle import quantized_reference as qr
from tests.quantized_helpers import call, check, paged

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("codes", ["e4m3", "int8"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("HQ,HKV", [(3, 3), (8, 2), (40, 2)])
def test_widths_and_types(device, D, codes, dtype, HQ, HKV):
    check(device, [1, 2], [45, 330], HQ=HQ, HKV=HKV, D=D, codes=codes, dtype=dtype)


@pytest.mark.parametrize("length", [1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 1000])
def test_lengths_of_one_token(device, length):
    check(device, [1], [length], page=16)


@pytest.mark.parametrize("page,group", [(16, 16), (32, 16), (32, 32), (64, 16), (64, 64), (128, 32), (1024, 16), (1024, 1024)])
def test_pages_and_blocks_that_end_inside_a_chunk(device, page, group):
    check(device, [1, 3, 1], [3 * page + 5, page, 70], page=page, group=group)


@pytest.mark.parametrize("HQ,HKV", [(1, 1), (5, 1), (16, 1), (17, 1), (63, 1), (130, 1), (7, 7), (24, 8), (65, 13)])
def test_head_layouts(device, HQ, HKV):
    check(device, [1, 4, 2], [50, 177, 33], HQ=HQ, HKV=HKV, D=64, page=16)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_chunks_of_prompts(device, causal, D):
    check(device, [70, 1, 133], [300, 40, 133], HQ=6, HKV=2, D=D, page=64, causal=causal)


@pytest.mark.parametrize("counts,lengths", [([300], [300]), ([513], [1100]), ([40, 200, 3], [700, 200, 900])])
@pytest.mark.parametrize("codes", ["e4m3", "int8"])
def test_longer_chunks(device, counts, lengths, codes):
    check(device, counts, lengths, HQ=8, HKV=2, codes=codes, page=64, group=16)


def test_rows_that_see_nothing(device):
    """More tokens than rows: the first ones see none; a request without rows, one without tokens, and padding."""
    check(device, [5, 0, 3, 4], [2, 20, 0, 9], HQ=7, HKV=1, page=16, spare_tokens=6)
    check(device, [60, 0, 30, 40], [20, 20, 0, 9], HQ=8, HKV=2, page=16, spare_tokens=6)


def test_every_row_empty(device):
    check(device, [2, 1], [0, 0], page=16)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("n", [1, 40])
def test_pages_outside_the_cache_hold_no_keys(device, causal, n):
    t = paged(device, [n + 1, n, n], [250, 190, 40], page=16, seed=3)
    blocks = t["k_cache"].shape[0]
    t["block_table"][0, 0] = -1
    t["block_table"][0, 4:6] = blocks
    t["block_table"][0, 9] = 2**31 - 1
    t["block_table"][1, 5] = -(2**31)
    t["block_table"][2] = blocks + 5  # nothing left of the third
    check(device, [n + 1, n, n], [250, 190, 40], tensors=t, causal=causal)


@pytest.mark.parametrize("counts,over", [([4], [2]), ([5, 3, 0, 2], [4, 1, 3, 2**31 - 1 - 64]), ([70], [66]), ([150, 9], [40, 0])])
def test_lengths_beyond_the_table(device, counts, over):
    lengths = [64] * len(counts)
    t = paged(device, counts, lengths, page=16, spare_tokens=2)
    t["seqused_kv"] = torch.tensor([n + o for n, o in zip(lengths, over)], dtype=torch.int32, device=device)
    check(device, counts, lengths, tensors=t)
    check(device, counts, lengths, tensors=t, causal=False)


def test_strided_heads_first_queries_and_output(device):
    t = paged(device, [3, 2], [60, 41], HQ=10, HKV=5, page=16, heads_first=True)
    check(device, [3, 2], [60, 41], tensors=t)
    dense = call(dict(t, q=t["q"].contiguous()), 0.05)
    out = torch.empty((10, 5, 128), dtype=torch.bfloat16, device=device).transpose(0, 1)
    assert torch.equal(call(t, 0.05, out=out), dense)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("n", [2, 60])
def test_sharp_and_flat_scores(device, dtype, n):
    """Scores of some hundreds (one key takes all) and of nearly zero; the running maximum grows along the keys."""
    t = paged(device, [n], [300], HQ=16, HKV=2, page=16, dtype=dtype, seed=5)
    ramp = torch.linspace(-6, 4, 19, device=device).exp2()
    t["k_scale"][t["block_table"][0].long()] *= ramp[:, None, None]
    for scale in (2.0, 1e-4):
        check(device, [n], [300], tensors=t, scale=scale, dtype=dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("n", [1, 60])
def test_value_scales_far_apart(device, dtype, n):
    """Blocks whose value scales lie up to 2^60 apart, zeros and the least scale among them: what the small ones hold is
    lost next to the large ones, their weights are not."""
    t = paged(device, [n], [320], HQ=16, HKV=2, page=16, dtype=dtype, seed=6)
    rows = t["block_table"][0].long()
    t["v_scale"][rows[0::4]] *= 2.0 ** -30
    t["v_scale"][rows[1::4]] = 2.0 ** -80
    t["v_cache"][rows[1::4]] = 0
    t["v_scale"][rows[3]] = 0.0  # counts as 2^-80
    t["v_cache"][rows[3]] = 0
    check(device, [n], [320], tensors=t, dtype=dtype)


@pytest.mark.parametrize("n", [1, 60])
def test_largest_weight_is_exact(device, n):
    """One key of a large score: the output is its values in bf16, rounded once, whatever the scale."""
    t = paged(device, [n], [200], HQ=16, HKV=2, page=16, seed=7)
    rows = t["block_table"][0].long()
    t["q"].fill_(1.0)
    t["k_cache"].view(torch.uint8).zero_()
    t["k_cache"][rows[2], 5] = 1.0
    t["k_scale"][rows] = 1.0
    out = call(t, 1.0)
    want = t["v_cache"][rows[2], 5].double() * t["v_scale"][rows[2], 0].double()[:, None]  # [HKV, D]
    lead = 199 * math.exp(-128.0)
    assert lead < 2.0 ** -100
    assert torch.equal(out[-1].double(), want.to(torch.bfloat16).double().repeat_interleave(8, dim=0))


@pytest.mark.parametrize("what", ["nan query", "infinite query", "nan scale"])
@pytest.mark.parametrize("n", [1, 60])
def test_scores_that_are_not_finite(device, what, n):
    t = paged(device, [n, 2], [200, 90], HQ=4, HKV=2, page=16, seed=8)
    clean = call(t, 0.1)
    if what == "nan query":
        t["q"][n - 1, 3, 5] = math.nan
    elif what == "infinite query":
        t["q"][n - 1, 3].zero_()
        t["q"][n - 1, 3, 5] = math.inf
        t["k_cache"][t["block_table"][0].long(), :, 1, 5] = 2.0
    else:
        t["k_scale"][t["block_table"][0].long(), :, 1] = math.nan
    lse = torch.empty((n + 2, 4), device=device)
    out = call(t, 0.1, lse=lse)
    assert torch.isnan(out[n - 1, 3]).all() and torch.isnan(lse[n - 1, 3])
    others = torch.ones((n + 2, 4), dtype=torch.bool, device=device)
    others[:n, 2:] = False  # the heads that share the keys of the one that was changed
    assert torch.isfinite(out[others]).all() and torch.isfinite(lse[others]).all()
    if what != "infinite query":
        assert torch.equal(out[others], clean[others])


def test_long_context_beyond_32_bit_offsets(device):
    """Pages past 2^32 bytes of each cache."""
    page, HKV, D = 128, 8, 128
    blocks = 2**32 // (page * HKV * D) + 40
    small = paged(device, [1, 3], [700, 260], HQ=16, HKV=HKV, D=D, page=page, spare_pages=0)
    used = small["k_cache"].shape[0]
    far = blocks - 1 - torch.arange(used, device=device)
    moved = dict(small)
    for w in ("k", "v"):
        cache = torch.empty((blocks, page, HKV, D), dtype=torch.uint8, device=device)
        cache[far] = small[w + "_cache"].view(torch.uint8)
        moved[w + "_cache"] = cache.view(torch.float8_e4m3fn)
        scale = torch.empty((blocks, 1, HKV), device=device)
        scale[far] = small[w + "_scale"]
        moved[w + "_scale"] = scale
    table = small["block_table"].long()
    moved["block_table"] = torch.where(table >= 0, far[table.clamp(min=0)], table).to(torch.int32)
    assert torch.equal(call(small, 0.05), call(moved, 0.05))


@pytest.mark.parametrize("n", [1, 80])
def test_calls_repeat_bit_for_bit_on_another_stream(device, n):
    t = paged(device, [n, 6, 2], [900, 300, 40], HQ=32, HKV=4, page=64)
    first = call(t, 0.07)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        second = call(t, 0.07)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(first, second) and torch.equal(first, call(t, 0.07))


def test_two_captured_calls_follow_their_inputs(device):
    """Two graphs of different sizes, replayed in turn with eager work between; lengths change between replays."""
    a = paged(device, [1, 1, 1], [700, 90, 33], HQ=16, page=64, seed=1)
    b = paged(device, [40, 2], [500, 120], HQ=8, page=64, seed=2)
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
    t = paged(device, [1, 2], [40, 70])
    args = (t["q"], t["k_cache"], t["v_cache"], t["k_scale"], t["v_scale"], t["block_table"], t["cu_seqlens_q"],
            t["seqused_kv"], 0.1)
    out, lse = torch.ops.ascendflow_amd.quantized_attention(*args)
    want = torch.empty_like(lse)
    assert torch.equal(out, call(t, 0.1, lse=want)) and torch.equal(lse, want)


def test_no_tokens(device):
    assert call(paged(device, [0], [10]), 0.1).shape == (0, 8, 128)


@pytest.mark.parametrize("counts,lengths", [([1, 1], [300, 37]), ([40], [200]), ([450], [1700])])
@pytest.mark.parametrize("dtype,codes", [("bf16", "e4m3"), ("f16", "int8")])
@pytest.mark.parametrize("negative", [False, True])
@pytest.mark.parametrize("exponent", [16, 24, 30, 60, 110])
def test_scores_far_from_zero(device, counts, lengths, dtype, codes, negative, exponent):
    far_scores(device, counts, lengths, dtype, codes, negative, exponent)


@pytest.mark.parametrize("counts,lengths", [([1, 1], [9000, 3000]), ([40], [5000]), ([450], [5000]), ([300, 400], [900, 9000])])
@pytest.mark.parametrize("exponent", [24, 60])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_scores_far_from_zero_in_some_pages(device, counts, lengths, exponent, D):
    far_scores(device, counts, lengths, "bf16", "int8", False, exponent, D, some=True)


def far_scores(device, counts, lengths, dtype, codes, negative, exponent, D=128, some=False):
    """Scores whose float32 steps are many units (`some`: of each request's last twentieth of the pages that all its
    tokens see): a row is its best key's where the next is clearly behind."""
    t = paged(device, counts, lengths, HQ=4, HKV=2, D=D, page=32, codes=codes, dtype=dtype, seed=exponent)
    factor = torch.full((t["k_scale"].shape[0], 1, 1), 1.0 if some else 2.0 ** exponent)
    if some:
        for b, (n, s) in enumerate(zip(counts, lengths)):
            pages = (s - n) // 32
            factor[t["block_table"][b, pages - pages // 20 - 1:pages].long().cpu()] = 2.0 ** exponent
    t["k_scale"] = t["k_scale"] * factor.to(device)
    if negative:
        t["q"] = -t["q"].abs()
        t["k_cache"] = (t["k_cache"].view(torch.uint8) & 0x7f).view(t["k_cache"].dtype)
    T, HQ, D = t["q"].shape
    lse = torch.empty((T, HQ), device=device)
    out = call(t, D ** -0.5, lse=lse).cpu().double()
    lse = lse.cpu().double()
    cpu = {n: x.cpu() for n, x in t.items()}
    caches = [qr.values(cpu[w + "_cache"], cpu[w + "_scale"]).double() for w in "kv"]
    eps, told, at = torch.finfo(t["q"].dtype).eps / 2, 0, 0
    for b, (n, s) in enumerate(zip(counts, lengths)):
        pages = cpu["block_table"][b, :-(-s // 32)].long()
        k, v = [c[pages].reshape(-1, 2, D)[:s].repeat_interleave(2, 1).transpose(0, 1) for c in caches]
        q = cpu["q"][at:at + n].double().transpose(0, 1)
        scores, reach = q @ k.transpose(1, 2) * D ** -0.5, (q.abs() @ k.abs().transpose(1, 2)).amax(-1) * D ** -0.5
        hidden = torch.arange(s) > s - n + torch.arange(n)[:, None]
        top = scores.masked_fill(hidden, -torch.inf).topk(min(s, 2), dim=-1)
        # A product of D terms in float32 is off by D 2^-24 of their magnitudes; 60 are what no weight is seen behind.
        clear = top.values[..., 0] - top.values[..., -1] > 60 + 4 * D * 2.0 ** -24 * reach
        want = v.gather(1, top.indices[..., :1].expand(-1, -1, D))
        # The weight is rounded where it meets the value but not in the sum, and then the result is.
        off = (out[at:at + n].transpose(0, 1) - want).abs() - want.abs() * (2 * eps + 2.0 ** -16)
        assert off[clear].max() <= 1e-30
        assert ((lse[at:at + n].T - top.values[..., 0]).abs() <= 60 + (D + 8) * 2.0 ** -24 * reach)[clear].all()
        told += clear.sum().item()
        at += n
    assert told > 0.8 * T * HQ


@pytest.mark.parametrize("name", ["k_cache", "v_cache", "k_scale", "v_scale"])
def test_a_gradient_of_the_cache_alone_is_refused_in_backward(device, name):
    t = paged(device, [1, 2], [40, 70])
    t[name].requires_grad_(True)
    out = call(t, 0.1)
    assert out.requires_grad
    with pytest.raises(RuntimeError, match="forward only"):
        out.sum().backward()


def test_forward_only(device):
    t = paged(device, [1, 2], [40, 70])
    t["q"].requires_grad_(True)
    out = call(t, 0.1)
    with pytest.raises(RuntimeError, match="forward only"):
        out.sum().backward()
    with pytest.raises(ValueError, match="gradient"):
        call(t, 0.1, out=torch.empty_like(out))
    with torch.no_grad():
        assert not call(t, 0.1).requires_grad
    import torch.autograd.forward_ad as fwd

    with fwd.dual_level(), pytest.raises(NotImplementedError):
        call(dict(t, q=fwd.make_dual(t["q"].detach(), torch.ones_like(t["q"]))), 0.1)


def test_written_tensors_count_a_version(device):
    t = paged(device, [1, 2], [40, 70])
    out, lse = torch.empty_like(t["q"]), torch.empty((3, 8), device=device)
    call(t, 0.1, out=out, lse=lse)
    assert out._version == 1 and lse._version == 1 and t["q"]._version == 0


@pytest.mark.parametrize("name,change", [
    ("q", lambda t: t["q"].float()),
    ("q", lambda t: t["q"][..., :100]),
    ("q", lambda t: t["q"][:, :7]),
    ("q", lambda t: t["q"].transpose(1, 2).contiguous().transpose(1, 2)),
    ("q", lambda t: t["q"].cpu()),
    ("q", lambda t: t["q"].tolist()),
    ("k_cache", lambda t: t["k_cache"][:, :10].contiguous()),
    ("k_cache", lambda t: t["k_cache"][:, ::2]),
    ("k_cache", lambda t: t["k_cache"].view(torch.uint8)),
    ("k_cache", lambda t: t["k_cache"].view(torch.float8_e5m2)),
    ("v_cache", lambda t: t["v_cache"].view(torch.int8)),
    ("v_cache", lambda t: t["v_cache"][..., :64].contiguous()),
    ("k_scale", lambda t: t["k_scale"].double()),
    ("k_scale", lambda t: t["k_scale"][:, :0]),
    ("v_scale", lambda t: t["v_scale"][:-1]),
    ("v_scale", lambda t: t["v_scale"].expand(-1, 2, -1).contiguous()),
    ("block_table", lambda t: t["block_table"].long()),
    ("block_table", lambda t: t["block_table"][:, :0]),
    ("cu_seqlens_q", lambda t: t["cu_seqlens_q"][:-1]),
    ("seqused_kv", lambda t: t["seqused_kv"].cpu()),
])
def test_refusals(device, name, change):
    t = paged(device, [1, 2], [40, 70])
    with pytest.raises(ValueError):
        call(dict(t, **{name: change(t)}), 0.1)


def test_refused_outputs_and_scales(device):
    t = paged(device, [1, 2], [40, 70])
    for scale in (0.0, -1.0, math.inf, math.nan):
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
