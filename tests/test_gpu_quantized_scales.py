"""Attention over an 8-bit cache whose value scales lie up to 2^206 apart, against the float64 definition: a key whose values
are too small to show next to others' still has its whole weight in the denominator and in softmax_lse."""

import math

import pytest
import torch

from oracle import latent_reference as lr
from oracle import quantized_reference as qr
from tests.quantized_helpers import call, compare, expected, paged
from tests.test_gpu_quantized_forms import form_of, tiles

pytestmark = pytest.mark.gpu

# Exponents of the value scales of a request's pages: a block of zeros (2^-80) next to large values, the largest scales that
# an append writes, and the largest that are read.
PAIRS = [(-80, 50), (-80, 110), (-30, 100), (-80, 122), (-80, 126)]
ORDERS = ["rising", "falling", "mixed"]


def spread_scales(t, low, high, order):
    """Value scales 2^low and 2^high over the pages of every request; codes of 1 and -1 where others would overflow."""
    table, blocks = t["block_table"].cpu(), t["k_cache"].shape[0]
    for b in range(table.shape[0]):
        ids = table[b][(table[b] >= 0) & (table[b] < blocks)].long()
        for i, page in enumerate(ids.tolist()):
            large = {"rising": 2 * i >= len(ids), "falling": 2 * i < len(ids), "mixed": i % 3 == 1}[order]
            t["v_scale"][page] = torch.where(torch.isnan(t["v_scale"][page]), math.nan, 2.0 ** (high if large else low))
    if high > 110:
        e4m3, codes = t["v_cache"].dtype == torch.float8_e4m3fn, t["v_cache"].view(torch.uint8)
        one, minus = (0x38, 0xb8) if e4m3 else (0x01, 0xff)
        signs = torch.where(codes >= 0x80, minus, one).to(torch.uint8)
        t["v_cache"] = torch.where((codes == 0x7f) & e4m3, codes, signs).view(t["v_cache"].dtype)  # rows behind the last stay no numbers
    return t


def check(device, counts, lengths, tensors, causal=True, scale=None):
    """One call against the definition, by its derived bound and what float32 cannot hold: with a weight times its value scale
    as p, the largest of a row 1, a p below 2^-126 is 0. The denominator, in the same units, is at least 1 over the value
    scale of that largest, so what `keys` lost products p v, |v| <= C, take from a result is at most
    keys 2^-126 C (the largest value scale), ``lost``; ``spread`` enters the bound times half a step of the type."""
    t, T, HQ, D = tensors, *tensors["q"].shape
    scale = D ** -0.5 if scale is None else scale
    out, lse = torch.full((T, HQ, D), 7.0, dtype=t["q"].dtype, device=device), torch.full((T, HQ), 7.0, device=device)
    call(t, scale, causal, out, lse)
    torch.cuda.synchronize()
    (want, want_lse, spread, reach), largest, exponents = expected(t, scale, causal)
    lost = max(lengths) * 2.0 ** -126 * largest
    spread = spread + lost / (torch.finfo(t["q"].dtype).eps / 2)
    compare(out.cpu(), lse.cpu(), ((want, want_lse, spread, reach), largest, exponents), t["q"].dtype, max(lengths))
    padding = int(t["cu_seqlens_q"][-1])
    assert (out[padding:] == 7).all() and (lse[padding:] == 7).all()


@pytest.mark.parametrize("low,high", PAIRS)
@pytest.mark.parametrize("order", ORDERS)
@pytest.mark.parametrize("D,codes", [(64, "int8"), (128, "e4m3"), (128, "int8"), (256, "e4m3")])
@pytest.mark.parametrize("counts,lengths,rows", [([1, 2, 0, 3], [300, 170, 40, 3], 16), ([6, 9, 4], [330, 170, 0], 32)])
def test_few_rows(device, counts, lengths, rows, D, codes, order, low, high):
    t = spread_scales(paged(device, counts, lengths, D=D, codes=codes, group=16, spare_tokens=2), low, high, order)
    assert form_of(t)[0] == rows
    check(device, counts, lengths, tensors=t)


@pytest.mark.parametrize("low,high", PAIRS)
@pytest.mark.parametrize("order", ORDERS)
@pytest.mark.parametrize("D,codes", [(64, "int8"), (128, "e4m3"), (128, "int8"), (256, "e4m3")])
def test_tiles(device, D, codes, order, low, high):
    """The last request's first tokens see one page, or none."""
    counts, lengths = [130, 3, 200], [430, 90, 190]
    t = spread_scales(tiles(device, counts, lengths, D=D, codes=codes, group=16), low, high, order)
    check(device, counts, lengths, tensors=t)


@pytest.mark.parametrize("low,high", [(-80, 50), (-80, 122)])
@pytest.mark.parametrize("order", ORDERS)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n", [1, 6, 700])
def test_many_parts(device, n, D, order, low, high):
    """Of parts on either side of the step, and of such that hold both scales; every key weighs about the same."""
    t = spread_scales(paged(device, [n], [9000], HQ=4, HKV=1, D=D, page=64, seed=9), low, high, order)
    assert form_of(t)[0] == (16 if n == 1 else 32 if n == 6 else 128 if D == 256 else 256)
    check(device, [n], [9000], tensors=t, scale=1e-3)


@pytest.mark.parametrize("n", [1, 6, 300])
def test_one_key_of_large_values_among_many(device, n):
    """Equal scores: a page of 16 rows at 2^60 and thousands at 2^-80, each of which weighs as much."""
    t = paged(device, [n], [4000], HQ=4, HKV=1, page=16, seed=2)
    t["q"].zero_()
    t["v_scale"][t["block_table"][0].long()] = 2.0 ** -80
    t["v_scale"][t["block_table"][0, 3].long()] = 2.0 ** 60
    check(device, [n], [4000], tensors=t)


@pytest.mark.parametrize("order", ORDERS)
@pytest.mark.parametrize("n", [1, 60, 300])
def test_sharp_scores(device, n, order):
    """Scores some hundreds apart: small values may outweigh large ones, or not."""
    t = spread_scales(paged(device, [n], [500], HQ=16, HKV=2, page=16, seed=5, width=96), -80, 50, order)
    ramp = torch.linspace(-6, 4, 32, device=device).exp2()
    t["k_scale"][t["block_table"][0, :32].long()] *= ramp[:, None, None]
    check(device, [n], [500], tensors=t, scale=1.0)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("n", [1, 40, 300])
def test_pages_outside_the_cache(device, n, causal):
    counts, lengths = [n + 1, n, n], [450, 390, 340]
    t = spread_scales(paged(device, counts, lengths, page=16, seed=3, width=96), -80, 90, "mixed")
    blocks = t["k_cache"].shape[0]
    t["block_table"][0, 0] = -1
    t["block_table"][0, 4:9] = blocks
    t["block_table"][0, 11] = 2**31 - 1
    t["block_table"][1, 5] = -(2**31)
    t["block_table"][2] = blocks + 5  # nothing left of the third
    check(device, counts, lengths, tensors=t, causal=causal)


@pytest.mark.parametrize("codes", ["e4m3", "int8"])
@pytest.mark.parametrize("n", [1, 6, 400])
def test_lse_of_float16_queries(device, n, codes):
    """Such values overflow a float16 output; the weights' sum does not."""
    t = spread_scales(paged(device, [n], [900], HQ=8, HKV=2, page=16, codes=codes, dtype="f16", seed=4, width=96), -80, 60, "mixed")
    lse = torch.empty((n, 8), device=device)
    call(t, 0.09, lse=lse)
    (_, want, _, reach), _, exponents = expected(t, 0.09, True)
    bound = lr.lse_bound(want, reach, 900) + 8 * 2.0 ** -24 * (reach + exponents)
    assert ((lse.cpu().double() - want).abs() <= bound).all()


@pytest.mark.parametrize("what", ["nan query", "infinite query"])
@pytest.mark.parametrize("n", [1, 60, 300])
def test_scores_that_are_not_finite(device, what, n):
    t = spread_scales(paged(device, [n, 2], [500, 90], HQ=4, HKV=2, page=16, seed=8, width=96), -80, 60, "mixed")
    t["q"][n - 1, 3].zero_()
    t["q"][n - 1, 3, 5] = math.nan if what == "nan query" else math.inf
    t["k_cache"][t["block_table"][0, :32].long(), :, 1, 5] = 2.0
    lse = torch.empty((n + 2, 4), device=device)
    out = call(t, 0.1, lse=lse)
    assert torch.isnan(out[n - 1, 3]).all() and torch.isnan(lse[n - 1, 3])
    others = torch.ones((n + 2, 4), dtype=torch.bool, device=device)
    others[n - 1, 3] = False
    assert torch.isfinite(out[others]).all() and torch.isfinite(lse[others]).all()


@pytest.mark.parametrize("order", ORDERS)
@pytest.mark.parametrize("n", [1, 40, 450])
@pytest.mark.parametrize("exponent", [24, 60])
def test_scores_far_from_zero(device, n, order, exponent):
    """Scores whose float32 steps are many units: a row is its best key's where the next is clearly behind."""
    D, s = 128, 1700
    t = spread_scales(paged(device, [n], [s], HQ=4, HKV=2, D=D, page=32, codes="int8", seed=exponent), -80, 50, order)
    t["k_scale"] = t["k_scale"] * 2.0 ** exponent
    lse = torch.empty((n, 4), device=device)
    out = call(t, D ** -0.5, lse=lse).cpu().double().transpose(0, 1)
    cpu = {name: x.cpu() for name, x in t.items()}
    pages = cpu["block_table"][0, :-(-s // 32)].long()
    k, v = [qr.values(cpu[w + "_cache"], cpu[w + "_scale"])[pages].reshape(-1, 2, D)[:s].repeat_interleave(2, 1).transpose(0, 1) for w in "kv"]
    q = cpu["q"].double().transpose(0, 1)
    scores, reach = q @ k.transpose(1, 2) * D ** -0.5, (q.abs() @ k.abs().transpose(1, 2)).amax(-1) * D ** -0.5
    top = scores.masked_fill(torch.arange(s) > s - n + torch.arange(n)[:, None], -torch.inf).topk(2, dim=-1)
    # 60 units are what no weight is seen behind, and 130 ln 2 what a value scale makes up for.
    clear = top.values[..., 0] - top.values[..., 1] > 60 + 130 * math.log(2) + 4 * D * 2.0 ** -24 * reach
    want = v.gather(1, top.indices[..., :1].expand(-1, -1, D))
    # The weight is rounded where it meets the value but not in the sum, and then the result is; the exponent of the sum is
    # off by 2^-15 at most (float32 numbers up to 2^9), that of the weight by as much.
    off = (out - want).abs() - want.abs() * (2 * 2.0 ** -9 * (1 + 2.0 ** -9) + 2 * 2.0 ** -15)
    assert off[clear].max() <= 1e-30
    assert ((lse.cpu().double().T - top.values[..., 0]).abs() <= 60 + (D + 8) * 2.0 ** -24 * reach)[clear].all()
    assert clear.sum().item() > 0.5 * n * 4


@pytest.mark.parametrize("n", [1, 6, 300])
def test_past_32_bit_offsets(device, n):
    """The second reading of the keys too: pages past 2^32 bytes of each cache."""
    page, HKV, D = 128, 8, 128
    blocks = 2**32 // (page * HKV * D) + 40
    small = spread_scales(paged(device, [n], [1600], HQ=16, HKV=HKV, D=D, page=page, group=32, spare_pages=0), -80, 60, "mixed")
    far = blocks - 1 - torch.arange(small["k_cache"].shape[0], device=device)
    moved = dict(small)
    for w in ("k", "v"):
        cache = torch.empty((blocks, page, HKV, D), dtype=torch.uint8, device=device)
        cache[far] = small[w + "_cache"].view(torch.uint8)
        moved[w + "_cache"] = cache.view(torch.float8_e4m3fn)
        scale = torch.empty((blocks, 4, HKV), device=device)
        scale[far] = small[w + "_scale"]
        moved[w + "_scale"] = scale
    moved["block_table"] = far[small["block_table"].long()].to(torch.int32)
    check(device, [n], [1600], small)
    assert torch.equal(call(small, 0.05), call(moved, 0.05))


@pytest.mark.parametrize("page,group", [(16, 16), (128, 16), (1024, 1024)])
@pytest.mark.parametrize("HQ,HKV", [(5, 5), (24, 8), (13, 1)])
def test_pages_and_heads(device, page, group, HQ, HKV):
    counts, lengths = [3, 1, 280], [2 * page + 5, 1500, 1700]
    t = paged(device, counts, lengths, HQ=HQ, HKV=HKV, D=64, page=page, group=group, codes="int8", seed=HQ)
    check(device, counts, lengths, spread_scales(t, -80, 55, "mixed"))


def test_in_a_graph_and_on_another_stream(device):
    calls = [spread_scales(paged(device, c, s, HQ=8, page=64, seed=2), -80, 70, "falling") for c, s in (([1, 2], [900, 120]), ([400], [1700]))]
    for t in calls:
        first = call(t, 0.06)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            second = call(t, 0.06)
        torch.cuda.current_stream().wait_stream(stream)
        assert torch.equal(first, second) and torch.equal(first, call(t, 0.06))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        outs = [call(t, 0.06) for t in calls]
    for step in range(3):
        for t in calls:
            t["q"].normal_()
            t["seqused_kv"] -= step
            t["v_scale"] *= 2.0 ** step
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out, call(t, 0.06)) for out, t in zip(outs, calls)), step
