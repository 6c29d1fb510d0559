"""Every form of the attention over an 8-bit cache against the float64 definition, each test checking the form it runs: tiles of
256 and 128 rows, of 32 and 16; one, two and four heads a workgroup; loads that stay out of the caches; requests in many parts."""

import ctypes as ct
import math

import pytest
import torch

from ascendflow_amd import _native
from oracle import quantized_reference as qr
from tests.quantized_helpers import B16, call, check, compare, paged

pytestmark = pytest.mark.gpu


def form_of(t, causal=True):
    T, HQ, D = t["q"].shape
    blocks, page, HKV, _ = t["k_cache"].shape
    B, W = t["block_table"].shape
    params = _native.QuantizedParams(
        dtype=0 if t["q"].dtype == torch.bfloat16 else 1, code=0 if t["k_cache"].dtype == torch.float8_e4m3fn else 1,
        causal=int(causal), T=T, B=B, HQ=HQ, HKV=HKV, D=D, PAGE=page, GROUP=page // t["k_scale"].shape[1], W=W, BLOCKS=blocks,
        q_stride_t=HQ * D, q_stride_h=D, out_stride_t=HQ * D, out_stride_h=D, scale=1.0)
    form = (ct.c_int64 * 4)()
    assert _native.library().form_quantized_attention(form, ct.byref(params)) == 0
    return list(form)


def tiles(device, counts, lengths, **kw):
    """Inputs that run in the tile form: a table with room for 1536 rows, more than 256 rows a request on average."""
    page = kw.get("page", 32)
    t = paged(device, counts, lengths, width=max(-(-1536 // page), -(-max(lengths) // page)), **kw)
    assert form_of(t)[0] == (128 if kw.get("D", 128) == 256 else 256)
    return t


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("codes", ["e4m3", "int8"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("causal", [True, False])
def test_tiles(device, D, codes, dtype, causal):
    counts, lengths = [130, 1, 200], [430, 90, 200]
    t = tiles(device, counts, lengths, D=D, codes=codes, dtype=dtype, group=16)
    check(device, counts, lengths, tensors=t, causal=causal)


@pytest.mark.parametrize("HQ,HKV", [(3, 1), (5, 5), (32, 4), (24, 8), (16, 1), (13, 13)])
def test_tiles_of_head_layouts(device, HQ, HKV):
    counts, lengths = [300], [333]
    check(device, counts, lengths, tensors=tiles(device, counts, lengths, HQ=HQ, HKV=HKV, D=64, page=16))


@pytest.mark.parametrize("length", [66, 127, 128, 129, 191, 192, 193, 1000, 2000])
@pytest.mark.parametrize("page,group", [(16, 16), (64, 32), (128, 128), (1024, 1024)])
def test_tiles_over_lengths_and_pages(device, length, page, group):
    check(device, [65], [length], tensors=tiles(device, [65], [length], HQ=5, HKV=1, page=page, group=group))


@pytest.mark.parametrize("causal", [True, False])
def test_tiles_whose_rows_see_nothing(device, causal):
    counts, lengths = [200, 0, 90, 40], [20, 20, 0, 9]
    t = tiles(device, counts, lengths, HQ=8, HKV=2, page=16, spare_tokens=6)
    check(device, counts, lengths, tensors=t, causal=causal)


@pytest.mark.parametrize("causal", [True, False])
def test_tiles_and_pages_outside_the_cache(device, causal):
    counts, lengths = [90, 70, 90], [350, 290, 100]
    t = tiles(device, counts, lengths, page=16, seed=3)
    blocks = t["k_cache"].shape[0]
    t["block_table"][0, 0] = -1
    t["block_table"][0, 4:9] = blocks
    t["block_table"][0, 11] = 2**31 - 1
    t["block_table"][1, 5] = -(2**31)
    t["block_table"][2] = blocks + 5  # nothing left of the third
    check(device, counts, lengths, tensors=t, causal=causal)


def test_tiles_of_lengths_beyond_the_table(device):
    counts, lengths = [150, 100], [1536, 1536]
    t = tiles(device, counts, lengths, page=16, spare_tokens=2)
    t["seqused_kv"] += torch.tensor([40, 2**31 - 1 - 1536], dtype=torch.int32, device=device)
    check(device, counts, lengths, tensors=t)
    check(device, counts, lengths, tensors=t, causal=False)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_tiles_of_sharp_and_flat_scores(device, dtype):
    t = tiles(device, [80], [500], HQ=16, HKV=2, page=16, dtype=dtype, seed=5)
    ramp = torch.linspace(-6, 4, 32, device=device).exp2()
    t["k_scale"][t["block_table"][0, :32].long()] *= ramp[:, None, None]
    for scale in (2.0, 1e-4):
        check(device, [80], [500], tensors=t, scale=scale, dtype=dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_tiles_of_value_scales_far_apart(device, dtype):
    t = tiles(device, [80], [320], HQ=16, HKV=2, page=16, dtype=dtype, seed=6)
    rows = t["block_table"][0, :20].long()
    t["v_scale"][rows[0::4]] *= 2.0 ** -30
    t["v_scale"][rows[1::4]] = 2.0 ** -80
    t["v_cache"][rows[1::4]] = 0
    t["v_scale"][rows[3]] = 0.0  # counts as 2^-80
    t["v_cache"][rows[3]] = 0
    check(device, [80], [320], tensors=t, dtype=dtype)


@pytest.mark.parametrize("what", ["nan query", "infinite query", "nan scale"])
def test_tiles_of_scores_that_are_not_finite(device, what):
    n = 300
    t = tiles(device, [n, 2], [500, 90], HQ=4, HKV=2, page=16, seed=8)
    clean = call(t, 0.1)
    if what == "nan query":
        t["q"][n - 1, 3, 5] = math.nan
    elif what == "infinite query":
        t["q"][n - 1, 3].zero_()
        t["q"][n - 1, 3, 5] = math.inf
        t["k_cache"][t["block_table"][0, :32].long(), :, 1, 5] = 2.0
    else:
        t["k_scale"][t["block_table"][0, :32].long(), :, 1] = math.nan
    lse = torch.empty((n + 2, 4), device=device)
    out = call(t, 0.1, lse=lse)
    assert torch.isnan(out[n - 1, 3]).all() and torch.isnan(lse[n - 1, 3])
    others = torch.ones((n + 2, 4), dtype=torch.bool, device=device)
    others[:n, 2:] = False  # the heads that share the keys of the one that was changed
    assert torch.isfinite(out[others]).all() and torch.isfinite(lse[others]).all()
    if what != "infinite query":
        assert torch.equal(out[others], clean[others])


def test_tiles_of_strided_queries_and_output(device):
    t = tiles(device, [150, 140], [160, 141], HQ=10, HKV=5, page=16, heads_first=True)
    check(device, [150, 140], [160, 141], tensors=t)
    out = torch.empty((10, 290, 128), dtype=torch.bfloat16, device=device).transpose(0, 1)
    assert torch.equal(call(t, 0.05, out=out), call(dict(t, q=t["q"].contiguous()), 0.05))


def test_tiles_past_32_bit_offsets(device):
    page, HKV, D = 128, 8, 128
    blocks = 2**32 // (page * HKV * D) + 40
    small = tiles(device, [150], [700], HQ=16, HKV=HKV, D=D, page=page, spare_pages=0)
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


def test_tiles_in_a_graph_and_on_another_stream(device):
    t = tiles(device, [300, 2], [500, 120], HQ=8, page=64, seed=2)
    first = call(t, 0.06)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        second = call(t, 0.06)
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    assert torch.equal(first, second)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(t, 0.06)
    for step in range(3):
        t["q"].normal_()
        t["seqused_kv"] -= step
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call(t, 0.06)), step


# Requests enough that a tile keeps few workgroups of four, two or one heads.
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("HKV,heads", [(4, 4), (8, 4), (2, 2), (6, 2), (3, 1)])
@pytest.mark.parametrize("n", [1, 5])
def test_heads_of_a_workgroup(device, D, HKV, heads, n):
    B = 130
    counts = [n] * B
    lengths = [n + 37 * b % 190 for b in range(B)]
    t = paged(device, counts, lengths, HQ=4 * HKV, HKV=HKV, D=D, page=16, seed=HKV)
    assert form_of(t)[:2] == [32 if n == 5 else 16, heads]
    check(device, counts, lengths, tensors=t)


@pytest.mark.parametrize("codes,dtype", [("e4m3", "bf16"), ("int8", "f16"), ("int8", "bf16"), ("e4m3", "f16")])
def test_few_requests_take_a_head_a_workgroup(device, codes, dtype):
    t = paged(device, [1, 1], [3000, 77], HQ=32, HKV=8, codes=codes, dtype=dtype)
    assert form_of(t)[:2] == [16, 1]
    check(device, [1, 1], [3000, 77], tensors=t)


@pytest.mark.parametrize("D,codes", [(128, "e4m3"), (128, "int8"), (256, "e4m3")])
def test_loads_that_stay_out_of_the_caches(device, D, codes):
    """A cache of 128 MiB and more, most of it nobody's."""
    counts, lengths = [1] * 20, [400 - 19 * b for b in range(20)]
    small = paged(device, counts, lengths, HQ=8, HKV=4, D=D, page=32, codes=codes, seed=4)
    more = (64 << 20) // (32 * 4 * D)
    large = dict(small)
    for w in ("k", "v"):
        cache = small[w + "_cache"]
        large[w + "_cache"] = torch.cat([cache.view(torch.uint8), torch.full((more, *cache.shape[1:]), 0x7f, dtype=torch.uint8, device=device)]).view(cache.dtype)
        large[w + "_scale"] = torch.cat([small[w + "_scale"], torch.full((more, *small[w + "_scale"].shape[1:]), math.nan, device=device)])
    assert form_of(large)[3] == 1 and form_of(small)[3] == 0
    check(device, counts, lengths, tensors=large)
    assert torch.equal(call(large, 0.1), call(small, 0.1))


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n", [1, 6, 700])
def test_one_long_request_in_many_parts(device, D, n):
    """Each part matters: its keys' scores are alike, its values its own."""
    t = paged(device, [n], [9000], HQ=4, HKV=1, D=D, page=64, seed=9)
    assert form_of(t)[0] == (16 if n == 1 else 32 if n == 6 else 128 if D == 256 else 256)
    check(device, [n], [9000], tensors=t, scale=1e-3)
    assert B16["bf16"] is t["q"].dtype


@pytest.mark.parametrize("page,group", [(16, 16), (128, 64)])
def test_tiles_of_many_chunks(device, page, group):
    """A workgroup goes over more chunks than it brings the pages and scales of at once: the definition on the device."""
    n, length = 80, 33000
    t = tiles(device, [n], [length], HQ=128, HKV=32, D=64, page=page, group=group, seed=11)
    assert form_of(t)[1:3] == [1, 8]  # 8 workgroups a head share 2 tiles of 516 chunks
    k, v = (qr.values(t[w + "_cache"], t[w + "_scale"].clamp(min=2.0 ** -80)) for w in ("k", "v"))
    want = qr.attention(t["q"], k, v, t["block_table"], t["cu_seqlens_q"], t["seqused_kv"], 0.125)
    used = t["v_scale"][torch.isfinite(t["v_scale"])]
    lse = torch.empty((n, 128), device=device)
    out = call(t, 0.125, lse=lse)
    largest, exponents = used.max().item() * 448, used.log2().abs().max().item()
    compare(out.cpu(), lse.cpu(), ([x.cpu() for x in want], largest, exponents), torch.bfloat16, length)
