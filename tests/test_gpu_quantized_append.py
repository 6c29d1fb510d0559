"""Append to an 8-bit paged cache against its definition, code for code: blocks begun and blocks that hold rows, scales that
grow and that stay, types, odd widths, strides, values that are not finite, tokens without a place, refusals."""

import math

import numpy as np
import pytest
import torch

from oracle import quantized_reference as qr
from tests.quantized_helpers import B16, CODES

pytestmark = pytest.mark.gpu


def inputs(device, counts, lengths, *, HKV=2, D=64, page=32, group=None, codes="e4m3", dtype="bf16", seed=0, spare_tokens=0,
           earlier=1.0, new=1.0):
    """New tokens, and a cache whose rows before them were written with values of size ``earlier`` and some scale."""
    gen = torch.Generator().manual_seed(seed)
    group = page if group is None else group
    need = [max(1, -(-s // page)) for s in lengths]
    blocks = sum(need) + 2
    order = torch.randperm(blocks, generator=gen).to(torch.int32)
    table = torch.full((len(counts), max(need) + 1), -1, dtype=torch.int32)
    at = 0
    for b, pages in enumerate(need):
        table[b, :pages] = order[at:at + pages]
        at += pages
    T = sum(counts) + spare_tokens
    t = {}
    for which in ("k", "v"):
        t[which] = (new * torch.randn((T, HKV, D), generator=gen) * torch.exp(torch.randn((T, HKV, 1), generator=gen))).to(B16[dtype])
        scale = torch.exp2(torch.randint(-8, -4, (blocks, page // group, HKV), generator=gen).float()) * earlier
        x = torch.randn((blocks, page, HKV, D), generator=gen) * (60 if codes == "e4m3" else 40)
        t[which + "_cache"] = torch.from_numpy(qr.nearest(x.double().numpy(), CODES[codes])).to(CODES[codes])
        t[which + "_scale"] = scale
    t.update(block_table=table, cu_seqlens_q=torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32),
             seqused_kv=torch.tensor(lengths, dtype=torch.int32))
    return {k: v.to(device) for k, v in t.items()}


def call(t):
    from ascendflow_amd.sparse_attention import append_quantized_kv

    return append_quantized_kv(t["k"], t["v"], t["k_cache"], t["v_cache"], t["k_scale"], t["v_scale"], t["block_table"],
                               t["cu_seqlens_q"], t["seqused_kv"])


def same(got, want):
    """Equal values, zeros of either sign and NaN alike."""
    return np.array_equal(got, want, equal_nan=True)


def check(t):
    before = {k: v.clone() for k, v in t.items()}
    k_cache, v_cache = call(t)
    assert k_cache is t["k_cache"] and v_cache is t["v_cache"]
    torch.cuda.synchronize()
    for which in ("k", "v"):
        codes = before[which + "_cache"].cpu()
        values, scale = codes.float().double().numpy(), before[which + "_scale"].cpu().double().numpy()
        qr.append(before[which].cpu(), (values, codes.dtype), scale, before["block_table"].cpu(), before["cu_seqlens_q"].cpu(),
                  before["seqused_kv"].cpu())
        assert same(t[which + "_scale"].cpu().double().numpy(), scale)
        assert same(t[which + "_cache"].cpu().float().double().numpy(), values)
    return before


@pytest.mark.parametrize("codes", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("page,group", [(16, 16), (64, 16), (64, 64), (128, 32)])
def test_types_and_blocks(device, codes, dtype, page, group):
    check(inputs(device, [1, 5, 100], [40, 70, 150], codes=codes, dtype=dtype, page=page, group=group))


@pytest.mark.parametrize("codes", ["e4m3", "int8"])
@pytest.mark.parametrize("earlier", [2.0 ** -12, 2.0 ** -3, 1.0, 2.0 ** 6])
def test_scales_that_grow_and_that_stay(device, codes, earlier):
    check(inputs(device, [1, 1, 3, 1], [17, 32, 50, 33], codes=codes, earlier=earlier, seed=1))


@pytest.mark.parametrize("codes", ["e4m3", "int8"])
def test_earlier_scales_that_are_no_powers_of_two(device, codes):
    t = inputs(device, [1, 2, 3], [20, 30, 50], codes=codes, seed=2)
    for which in ("k", "v"):
        t[which + "_scale"] *= 1.37
    before = {k: v.clone() for k, v in t.items()}
    call(t)
    for which in ("k", "v"):
        was, now = before[which + "_scale"].cpu(), t[which + "_scale"].cpu()
        assert (torch.frexp(now[now != was])[0] == 0.5).all()  # powers of two
        # Codes of the new rows are x times the float32 reciprocal of the scale.
        block = before["block_table"][0, 0].long()
        inverse = (1.0 / t[which + "_scale"][block, 0]).cpu()
        want = qr.nearest((before[which][0].float().cpu() * inverse[:, None]).double().numpy(), t[which + "_cache"].dtype)
        assert same(t[which + "_cache"][block, 19].cpu().float().double().numpy(), want)


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 32, 33, 64, 65, 200])
@pytest.mark.parametrize("ahead", [0, 1, 16, 31])
def test_numbers_of_tokens(device, n, ahead):
    check(inputs(device, [n], [ahead + n], seed=n))


@pytest.mark.parametrize("D", [1, 7, 24, 100, 128, 256, 1024])
def test_widths(device, D):
    check(inputs(device, [3, 20], [30, 40], D=D, HKV=3))


@pytest.mark.parametrize("HKV", [1, 5, 8, 33])
def test_heads(device, HKV):
    check(inputs(device, [3, 20], [30, 40], HKV=HKV))


def test_many_requests(device):
    B = 300
    gen = torch.Generator().manual_seed(3)
    counts = torch.randint(0, 4, (B,), generator=gen).tolist()
    lengths = [c + x for c, x in zip(counts, torch.randint(0, 40, (B,), generator=gen).tolist())]
    check(inputs(device, counts, lengths, HKV=1, D=16, page=16, spare_tokens=5))


@pytest.mark.parametrize("codes", ["e4m3", "int8"])
def test_values_at_the_edges(device, codes):
    """Zeros, the largest code times powers of two and its neighbours, subnormals, infinities and NaN."""
    t = inputs(device, [6], [22], codes=codes, dtype="bf16", HKV=2, D=64)
    k = t["k"].float()
    k[:, 0] = 0.0
    k[1, 1] = 3.0e38
    k[2, 1, 5] = math.inf
    k[2, 1, 6] = -math.inf
    k[3, 1, 7] = math.nan
    t["k"] = k.to(t["k"].dtype)
    v = torch.zeros_like(k)
    v[0, 0, :8] = torch.tensor([448.0, -448.0, 464.0, 2.0 ** -10, 3 * 2.0 ** -10, 127.0, -127.0, 0.5])
    v[1, 1, :4] = torch.tensor([1e-38, -1e-30, 2.0 ** -80, 2.0 ** -130])
    t["v"] = v.to(t["v"].dtype)
    check(t)


@pytest.mark.parametrize("top", [448.0, 449.0, 447.0, 450.0, 112.0, 127.0, 127.5, 63.5, 126.0, 1.75, 1.7578125])
@pytest.mark.parametrize("codes", ["e4m3", "int8"])
def test_scale_of_magnitudes_at_its_limits(device, top, codes):
    t = inputs(device, [2], [2], codes=codes, dtype="bf16", HKV=1, D=16)
    for which in ("k", "v"):
        t[which] = t[which].clamp(-1, 1)
        t[which][1, 0, 3] = top
    check(t)


def test_nothing_but_zeros_gets_the_least_scale(device):
    t = inputs(device, [3], [3])
    t["k"].zero_()
    check(t)
    assert (t["k_scale"][t["block_table"][0, 0].long()] == 2.0 ** -80).all()


def test_tokens_without_a_place_write_nothing(device):
    """Padding, more tokens than rows, positions beyond the table, pages outside the cache."""
    t = inputs(device, [5, 3, 4, 2], [3, 50, 40, 33], page=16, spare_tokens=4)
    t["seqused_kv"][1] = 16 * t["block_table"].shape[1] + 1
    t["block_table"][2, 2] = t["k_cache"].shape[0]
    t["block_table"][3] = -1
    t["cu_seqlens_q"] += 1  # token 0 belongs to nobody
    check(t)


def test_strided_rows(device):
    t = inputs(device, [3, 20], [30, 40], HKV=4)
    both = torch.stack([t["k"], t["v"]], dim=1)  # one projection
    check(dict(t, k=both[:, 0], v=both[:, 1]))
    t = inputs(device, [3, 20], [30, 40], HKV=4, seed=5)
    check(dict(t, k=t["k"].transpose(0, 1).contiguous().transpose(0, 1)))
    wide = torch.cat([t["v"], t["v"][..., :1]], dim=-1)
    check(dict(t, v=wide[..., 1:]))  # rows off 16 bytes
    check(dict(t, k=t["k"][:, :1].expand(-1, 4, -1)))


def test_token_by_token_is_as_the_whole(device):
    """e4m3 without subnormal codes: a block filled one token at a time holds what one call gives."""
    whole = inputs(device, [30], [30], HKV=2, D=64, seed=9)
    for which in ("k", "v"):
        x = whole[which].float()
        whole[which] = (x.sign() * x.abs().clamp(min=0.05, max=3.0)).to(whole[which].dtype)
    steps = {k: v.clone() for k, v in whole.items()}
    call(whole)
    for i in range(30):
        call(dict(steps, k=steps["k"][i:i + 1], v=steps["v"][i:i + 1],
                  cu_seqlens_q=torch.tensor([0, 1], dtype=torch.int32, device=device),
                  seqused_kv=torch.tensor([i + 1], dtype=torch.int32, device=device)))
    for name in ("k_cache", "v_cache", "k_scale", "v_scale"):
        assert torch.equal(whole[name].float(), steps[name].float())


def test_far_pages(device):
    """Pages past 2^32 bytes of the cache."""
    page, HKV, D = 128, 8, 128
    blocks = 2**32 // (page * HKV * D) + 10
    t = inputs(device, [1, 40], [5, 100], HKV=HKV, D=D, page=page)
    small = {k: v.clone() for k, v in t.items()}
    used = t["k_cache"].shape[0]
    far = blocks - 1 - torch.arange(used, device=device)
    for w in ("k", "v"):
        cache = torch.zeros((blocks, page, HKV, D), dtype=torch.uint8, device=device)
        cache[far] = t[w + "_cache"].view(torch.uint8)
        t[w + "_cache"] = cache.view(torch.float8_e4m3fn)
        scale = torch.zeros((blocks, 1, HKV), device=device)
        scale[far] = t[w + "_scale"]
        t[w + "_scale"] = scale
    table = t["block_table"].long()
    t["block_table"] = torch.where(table >= 0, far[table.clamp(min=0)], table).to(torch.int32)
    call(t)
    call(small)
    for w in ("k", "v"):
        assert torch.equal(t[w + "_cache"][far].view(torch.uint8), small[w + "_cache"].view(torch.uint8))
        assert torch.equal(t[w + "_scale"][far], small[w + "_scale"])


def test_captured_and_custom_op(device):
    t = inputs(device, [1, 2], [20, 40])
    first = {k: v.clone() for k, v in t.items()}
    call(t)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(t)
    for step in range(3):
        t["k"].normal_()
        for name in ("k_cache", "v_cache", "k_scale", "v_scale"):
            t[name].copy_(first[name])
        graph.replay()
        torch.cuda.synchronize()
        again = {k: v.clone() for k, v in first.items()}
        again["k"].copy_(t["k"])
        torch.ops.ascendflow_amd.append_quantized_kv(
            again["k"], again["v"], again["k_cache"], again["v_cache"], again["k_scale"], again["v_scale"],
            again["block_table"], again["cu_seqlens_q"], again["seqused_kv"])
        for name in ("k_cache", "v_cache", "k_scale", "v_scale"):
            assert torch.equal(t[name].float(), again[name].float()), step


def test_no_tokens_and_versions(device):
    t = inputs(device, [0], [10])
    call(t)
    assert t["k_cache"]._version == 0
    t = inputs(device, [1], [10])
    call(t)
    assert all(t[n]._version == 1 for n in ("k_cache", "v_cache", "k_scale", "v_scale")) and t["k"]._version == 0


@pytest.mark.parametrize("name,change", [
    ("k", lambda t: t["k"].float()),
    ("k", lambda t: t["k"][..., :32]),
    ("k", lambda t: t["k"].cpu()),
    ("k", lambda t: None),
    ("v", lambda t: t["v"].half()),
    ("v", lambda t: t["v"].transpose(1, 2).contiguous().transpose(1, 2)),
    ("k_cache", lambda t: t["k_cache"].view(torch.uint8)),
    ("k_cache", lambda t: t["k_cache"][:, :24].contiguous()),
    ("v_cache", lambda t: t["v_cache"].view(torch.int8)),
    ("v_cache", lambda t: t["k_cache"]),
    ("v_scale", lambda t: t["k_scale"]),
    ("k_scale", lambda t: t["k_scale"].half()),
    ("k_scale", lambda t: torch.ones((t["k_scale"].shape[0], 4, 2), device="cuda")),  # 8 tokens a scale
    ("block_table", lambda t: t["block_table"].long()),
    ("cu_seqlens_q", lambda t: t["cu_seqlens_q"][1:]),
    ("seqused_kv", lambda t: t["seqused_kv"][1:]),
])
def test_refusals(device, name, change):
    t = inputs(device, [1, 2], [20, 40])
    with pytest.raises(ValueError):
        call(dict(t, **{name: change(t)}))


def test_gradients_are_refused(device):
    t = inputs(device, [1, 2], [20, 40])
    t["k"].requires_grad_(True)
    with pytest.raises(ValueError, match="gradient"):
        call(t)
    with torch.no_grad():
        call(t)
