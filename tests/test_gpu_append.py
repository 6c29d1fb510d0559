"""Append of new tokens to paged caches against its definition: split and whole rows, values, widths, pages, tokens
without a place, and refusals."""

import pytest
import torch

from ascendflow_amd.sparse_attention import append_paged_kv, rotary_frequencies
from oracle import latent_reference as lr
from tests.latent_helpers import B16

pytestmark = pytest.mark.gpu


def inputs(device, counts, lengths, *, HKV=1, DK=96, DV=0, R=32, page=16, dtype="bf16", split=False, spare=0, seed=0):
    gen = torch.Generator().manual_seed(seed)
    b16 = B16[dtype]
    T = sum(counts) + spare
    need = [-(-s // page) for s in lengths]
    blocks = sum(need) + 2
    order = torch.randperm(blocks, generator=gen).to(torch.int32)
    table = torch.full((len(counts), max(1, max(need))), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    cu = torch.tensor([0] + [sum(counts[:i + 1]) for i in range(len(counts))], dtype=torch.int32)
    normal = lambda *shape: torch.randn(shape, generator=gen).to(b16).to(device)
    t = dict(k=normal(T, HKV, DK - R if split else DK), k_cache=normal(blocks, page, HKV, DK), block_table=table.to(device),
             cu_seqlens_q=cu.to(device), seqused_kv=torch.tensor(lengths, dtype=torch.int32).to(device))
    extra = dict(frequencies=rotary_frequencies(R, device=device) if R else None)
    if split:
        extra["rope"] = normal(T, HKV, R)
    if DV:
        extra.update(v=normal(T, HKV, DV), v_cache=normal(blocks, page, HKV, DV))
    return t, extra


def check(t, extra, **kw):
    frequencies, rope = extra.get("frequencies"), extra.get("rope")
    cache, v_cache = t["k_cache"].clone(), extra["v_cache"].clone() if "v" in extra else None
    T = t["k"].shape[0]
    want = cache.double().cpu()
    written = torch.zeros(cache.shape[:2], dtype=torch.bool)
    blocks, page = cache.shape[:2]
    keys = t["k"] if rope is None else torch.cat([t["k"], rope], -1)
    R = 0 if frequencies is None else 2 * frequencies.numel()
    offset = kw.get("offset", 0) if rope is None else cache.shape[3] - R
    v_want = None if v_cache is None else v_cache.clone()
    table, cu, used = t["block_table"].cpu(), t["cu_seqlens_q"].cpu(), t["seqused_kv"].cpu()
    for b in range(table.shape[0]):
        for token, position, block, slot in lr.rows_of(cu, used, table, page, blocks, b):
            row = keys[token].cpu()
            if R:
                row = lr.rotate(row[None], torch.tensor([position]), frequencies.cpu(), kw.get("layout", "half"), offset,
                                kw.get("magnitude", 1.0))[0]
            want[block, slot] = row.double()
            written[block, slot] = True
            if v_want is not None:
                v_want[block, slot] = extra["v"][token]
    result = append_paged_kv(**{**t, "k_cache": cache}, **{**extra, **({"v_cache": v_cache} if "v" in extra else {})}, **kw)
    assert (result is cache) if v_cache is None else (result[0] is cache and result[1] is v_cache)
    got = cache.cpu()
    assert torch.equal(got[~written], t["k_cache"].cpu()[~written]), "rows without a new token changed"
    if R:
        top = torch.tensor([int(used.max())])
        absolute, relative = lr.rotation_bound(keys, top, frequencies.cpu(), cache.dtype, kw.get("magnitude", 1.0))
        assert ((got.double() - want).abs() <= absolute + relative * want.abs())[written].all()
        same = [i for i in range(cache.shape[3]) if not offset <= i < offset + R]
    else:
        same = list(range(cache.shape[3]))
    assert torch.equal(got.double()[written][..., same], want[written][..., same])
    if v_want is not None:
        assert torch.equal(v_cache, v_want)
    assert T == t["k"].shape[0]
    return got


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("DK,R", [(576, 64), (96, 32), (64, 64), (30, 10), (40, 16)])
def test_latent_and_rotary_key_as_two_tensors(device, DK, R, layout, dtype):
    t, extra = inputs(device, [1, 5, 2], [40, 33, 2], DK=DK, R=R, split=True, dtype=dtype)
    check(t, extra, layout=layout)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("HKV,DK,DV,R,offset,page", [
    (1, 512, 0, 64, 448, 128), (8, 128, 128, 64, 0, 64), (2, 64, 48, 64, 0, 16), (3, 34, 10, 12, 5, 7), (8, 128, 64, 0, 0, 128),
    (1, 16, 16, 16, 0, 1),
])
def test_keys_and_values(device, HKV, DK, DV, R, offset, page, layout):
    t, extra = inputs(device, [3, 1, 40], [50, 1, 90], HKV=HKV, DK=DK, DV=DV, R=R, page=page)
    check(t, extra, layout=layout, offset=offset, magnitude=1.25)


def test_tokens_without_a_place_write_nothing(device):
    """Padding behind the last request, more tokens than rows, requests without tokens, pages outside the cache."""
    t, extra = inputs(device, [6, 0, 3, 4, 2], [2, 20, 0, 40, 33], DK=96, R=32, split=True, spare=5)
    t["block_table"][3, 2] = t["k_cache"].shape[0]
    t["block_table"][4, 2] = -5
    check(t, extra)
    t["seqused_kv"][4] = 1000  # beyond the table
    check(t, extra)


@pytest.mark.parametrize("B", [1, 63, 64, 65, 200])
def test_many_requests(device, B):
    gen = torch.Generator().manual_seed(B)
    counts = torch.randint(0, 4, (B,), generator=gen).tolist()
    t, extra = inputs(device, counts, [n + 20 for n in counts], DK=64, R=32)
    check(t, extra, offset=32)


def test_strided_rows(device):
    t, extra = inputs(device, [9, 4], [30, 12], HKV=2, DK=64, DV=64, R=32)
    both = torch.stack([t["k"], extra["v"]], dim=1)  # [T, 2, HKV, D], one projection
    want = check(t, extra)
    t["k"], extra["v"] = both[:, 0], both[:, 1]
    assert torch.equal(check(t, extra), want)
    t["k"] = t["k"].transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(check(t, extra), want)
    odd = torch.zeros((13, 2, 67), dtype=torch.bfloat16, device=device)
    odd[..., 1:65] = t["k"]
    t["k"] = odd[..., 1:65]
    assert torch.equal(check(t, extra), want)


def test_rows_past_32_bit_offsets(device):
    blocks = 2**32 // (128 * 576) + 3
    cache = torch.empty((blocks, 128, 1, 576), dtype=torch.bfloat16, device=device)
    cache[-1] = 0
    t, extra = inputs(device, [3], [100], DK=576, R=64, page=128, split=True)
    table = torch.tensor([[blocks - 1]], dtype=torch.int32, device=device)
    append_paged_kv(**{**t, "k_cache": cache, "block_table": table}, **extra)
    small = torch.zeros((1, 128, 1, 576), dtype=torch.bfloat16, device=device)
    append_paged_kv(**{**t, "k_cache": small, "block_table": torch.zeros_like(table)}, **extra)
    assert torch.equal(cache[-1:], small) and (small[0, 97:100] != 0).any()


def test_custom_op_and_capture(device):
    t, extra = inputs(device, [1, 3], [40, 20], DK=576, R=64, split=True)
    want = check(t, extra, layout="interleaved")
    caches = [t["k_cache"].clone() for _ in range(2)]
    args = lambda cache: (t["k"], cache, t["block_table"], t["cu_seqlens_q"], t["seqused_kv"], None, None, extra["rope"],
                          extra["frequencies"], "interleaved")
    for cache in caches:
        torch.ops.ascendflow_amd.append_paged_kv(*args(cache))
        assert torch.equal(cache.cpu(), want)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        torch.ops.ascendflow_amd.append_paged_kv(*args(caches[1]))
    for _ in range(3):
        t["k"].normal_()
        t["seqused_kv"] -= 1
        graph.replay()
        torch.ops.ascendflow_amd.append_paged_kv(*args(caches[0]))
        torch.cuda.synchronize()
        assert torch.equal(caches[0], caches[1])


def test_no_tokens(device):
    t, extra = inputs(device, [0], [10])
    before = t["k_cache"].clone()
    append_paged_kv(**t, **extra)
    assert torch.equal(before, t["k_cache"])


def test_refusals(device):
    t, extra = inputs(device, [2, 3], [20, 30], HKV=2, DK=64, DV=64, R=32)
    cases = [dict(k=t["k"].float()), dict(k=t["k"][:, :1]), dict(k=t["k"].cpu()), dict(k_cache=t["k_cache"].half()),
             dict(k_cache=t["k_cache"][:, ::2]), dict(k_cache=t["k_cache"].float()), dict(block_table=t["block_table"].long()),
             dict(cu_seqlens_q=t["cu_seqlens_q"][1:]), dict(seqused_kv=t["seqused_kv"][:1]), dict(v=None),
             dict(v_cache=None), dict(v=extra["v"][..., :32]), dict(frequencies=extra["frequencies"].float()),
             dict(offset=33), dict(offset=-1), dict(layout="other"), dict(magnitude=float("nan")),
             dict(rope=t["k"][..., :32]),  # k then holds 32 columns only
             dict(rope=t["k"][..., :32], frequencies=None), dict(v_cache=t["k_cache"])]
    for change in cases:
        with pytest.raises(ValueError):
            append_paged_kv(**{**t, **extra, **change})
    with pytest.raises(ValueError, match="overlap"):
        append_paged_kv(**{**t, **extra, "k": t["k_cache"].view(-1, 2, 64)[:5]})


def test_tokens_ahead_of_the_first_request_write_nothing(device):
    t, extra = inputs(device, [4, 3], [9, 20], spare=2)
    t["cu_seqlens_q"] = t["cu_seqlens_q"] + 2  # two tokens of no request, then seven
    got = check(t, extra)
    changed = (got != t["k_cache"].cpu()).any(-1).flatten(1).any(-1)
    assert changed.sum() <= 3  # the pages of the seven rows
