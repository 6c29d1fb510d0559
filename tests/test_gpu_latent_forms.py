"""Every form of the two latent attentions against the float64 definitions, each checked to be the one that runs: tiles of
64 and 128 rows, keys shared by all workgroups or a tile a workgroup, few and many parts, streamed caches; expanded tiles of
256, 128 and 64 rows and split keys."""

import ctypes as ct
import math

import pytest
import torch

from ascendflow_amd import _native
from oracle import latent_reference as lr
from tests import test_gpu_latent_expanded as expanded
from tests.latent_helpers import B16, call, check, compare, paged

pytestmark = pytest.mark.gpu


def latent_form(T, B, H, L, R, page, width, blocks):
    got = (ct.c_int64 * 2)()
    params = _native.LatentParams(T=T, B=B, H=H, L=L, R=R, PAGE=page, W=width, BLOCKS=blocks, scale=1.0)
    assert _native.library().form_latent_attention(got, ct.byref(params)) == 0
    return list(got)


def form_of(t):
    T, H, L = t["q"].shape
    blocks, page, _, row = t["kv_cache"].shape
    B, width = t["block_table"].shape
    return latent_form(T, B, H, L, row - L, page, width, blocks)


def check_on_device(device, t, counts, lengths, causal=True, dtype="bf16"):
    """As ``check``, with the definition worked out on the device."""
    T, H, L = t["q"].shape
    scale = L ** -0.5
    out = torch.full((T, H, L), 7.0, dtype=B16[dtype], device=device)
    lse = torch.full((T, H), 7.0, device=device)
    call(t, scale, causal, out, lse)
    expected = lr.latent_attention(t["q"], t["q_rope"], t["kv_cache"], t["block_table"].cpu(), t["cu_seqlens_q"].cpu(),
                                   t["seqused_kv"].cpu(), scale, causal)
    finite = t["kv_cache"][torch.isfinite(t["kv_cache"])]
    compare(out, lse, expected, B16[dtype], max(lengths), finite.abs().max().item())
    assert (out[sum(counts):] == 7).all() and (lse[sum(counts):] == 7).all()


@pytest.mark.parametrize("L,R", [(128, 0), (128, 64), (256, 64), (512, 0), (512, 64)])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_128_row_tiles_shared_by_all_workgroups(device, L, R, dtype):
    """Two requests of a tile and a half each; chunks of 64 rows through rings of two and three slots."""
    t = paged(device, [2, 1, 3], [700, 65, 64], H=96, L=L, R=R, page=32, dtype=dtype)
    assert form_of(t) == [128, 256]
    check(device, [2, 1, 3], [700, 65, 64], tensors=t, dtype=dtype)


@pytest.mark.parametrize("length", [1, 63, 64, 65, 127, 128, 129, 192, 193, 1000])
def test_lengths_of_128_row_tiles(device, length):
    t = paged(device, [1], [length], H=128, L=512, R=64, page=16)
    assert form_of(t) == [128, 256]
    check(device, [1], [length], tensors=t)


@pytest.mark.parametrize("L", [256, 512])
def test_pages_outside_the_cache_between_full_chunks(device, L):
    """Chunks with fewer loads than their neighbours, in rings of two and three slots."""
    t = paged(device, [1, 2], [900, 500], H=96, L=L, R=64, page=16, seed=3)
    for page in (0, 7, 8, 20, 21, 22, 23, 24, 40, 55):
        t["block_table"][0, page] = -1 if page % 2 else t["kv_cache"].shape[0]
    t["block_table"][1, 4:12] = -7
    assert form_of(t) == [128, 256]
    check(device, [1, 2], [900, 500], tensors=t)


@pytest.mark.parametrize("causal", [True, False])
def test_a_128_row_tile_per_workgroup(device, causal):
    counts, lengths = [600, 1, 500], [700, 90, 500]
    t = paged(device, counts, lengths, H=128, L=128, R=64, page=64, spare_tokens=3)
    assert form_of(t) == [128, 0]
    check_on_device(device, t, counts, lengths, causal)


def test_a_64_row_tile_per_workgroup(device):
    gen = torch.Generator().manual_seed(1)
    counts = torch.randint(0, 2, (4200,), generator=gen).tolist()
    lengths = torch.randint(0, 40, (4200,), generator=gen).tolist()
    t = paged(device, counts, lengths, H=8, L=128, R=0, page=16)
    assert form_of(t) == [64, 0]
    check(device, counts, lengths, tensors=t)


@pytest.mark.parametrize("H,L", [(16, 512), (128, 512), (16, 128), (128, 256)])
def test_many_requests_in_many_parts(device, H, L):
    """More tiles than one workgroup per row group joins with 16 waves; lengths from none to some chunks."""
    gen = torch.Generator().manual_seed(H)
    counts = torch.randint(0, 3, (50,), generator=gen).tolist()
    lengths = [int(x) for x in torch.randint(0, 1500, (50,), generator=gen)]
    t = paged(device, counts, lengths, H=H, L=L, R=64, page=64)
    assert form_of(t)[1] > 0
    check_on_device(device, t, counts, lengths)


def test_one_request_in_as_many_parts_as_workgroups(device):
    for H in (16, 100):
        t = paged(device, [1], [70000], H=H, L=128, R=64, page=128)
        assert form_of(t)[1] > 0
        check_on_device(device, t, [1], [70000])


@pytest.mark.parametrize("H", [16, 128])
def test_streamed_cache(device, H):
    """Non-temporal loads: one tile a request, a cache of 128 MiB or more. The same results as a small cache's."""
    t = paged(device, [1, 1, 1], [900, 33, 300], H=H, L=512, R=64, page=128)
    check(device, [1, 1, 1], [900, 33, 300], tensors=t)
    large = torch.full((1000, 128, 1, 576), math.nan, dtype=torch.bfloat16, device=device)
    large[:t["kv_cache"].shape[0]] = t["kv_cache"]
    assert large.numel() * 2 >= 128 << 20
    assert torch.equal(call(t, 0.05), call(dict(t, kv_cache=large), 0.05))


@pytest.mark.parametrize("seed", range(8))
def test_random_ragged_batches(device, seed):
    gen = torch.Generator().manual_seed(100 + seed)
    pick = lambda *options: options[int(torch.randint(0, len(options), (1,), generator=gen))]
    B = pick(1, 2, 5, 9)
    H, L, R, page = pick(1, 8, 24, 64, 130), pick(128, 256, 512), pick(0, 64), pick(16, 32, 64, 128)
    counts = [int(x) for x in torch.randint(0, pick(2, 7, 60), (B,), generator=gen)]
    counts[0] = max(1, counts[0])
    lengths = [int(x) for x in torch.randint(0, 400, (B,), generator=gen)]
    check(device, counts, lengths, H=H, L=L, R=R, page=page, dtype=pick("bf16", "f16"), causal=pick(True, False), seed=seed,
          spare_tokens=pick(0, 2))


def test_parts_do_not_depend_on_what_the_workspace_held(device):
    """The same call after its workspace's memory was filled with NaN."""
    t = paged(device, [1, 2], [900, 400], H=64, L=512, R=64, page=64)
    first = call(t, 0.05)
    params = (3, 2, 64, 512, 64, 64, t["block_table"].shape[1], t["kv_cache"].shape[0])
    assert latent_form(*params)[1] > 0
    torch.cuda.synchronize()
    poison = torch.full((300 << 20,), 255, dtype=torch.uint8, device=device)  # NaN as float32
    del poison  # the caching allocator hands this memory out next
    assert torch.equal(first, call(t, 0.05))


# ---- expanded -------------------------------------------------------------------------


def expanded_form(nq, nk, H, causal=True):
    got = (ct.c_int64 * 2)()
    params = _native.LatentExpandedParams(causal=int(causal), Tq=sum(nq), Tk=sum(nk), B=len(nq), H=H, D=128, R=64, scale=1.0)
    assert _native.library().form_latent_attention_expanded(got, ct.byref(params)) == 0
    return list(got)


def check_expanded(device, nq, nk, H, causal=True, dtype="bf16", seed=0, spare=0):
    t = expanded.inputs(device, nq, nk, H=H, dtype=dtype, seed=seed, spare=spare)
    out = torch.full((t["q"].shape[0], H, 128), 7.0, dtype=B16[dtype], device=device)
    lse = torch.full(out.shape[:2], 7.0, device=device)
    expanded.call(t, causal, out=out, softmax_lse=lse)
    expected = lr.latent_attention_expanded(t["q"], t["k_nope"], t["k_rope"], t["v"], t["cu_q"].cpu(), t["cu_k"].cpu(),
                                            expanded.SCALE, causal)
    values = t["v"][torch.isfinite(t["v"])].abs().max().item()
    compare(out, lse, expected, B16[dtype], max(nk), values)
    assert (out[sum(nq):] == 7).all() and (lse[sum(nq):] == 7).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("nq,nk,H,causal,form", [
    ([1900], [1901], 64, False, [256, 1]),
    ([1000, 770], [1000, 900], 64, True, [128, 1]),
    ([300, 45], [300, 333], 20, True, [64, 1]),
])
def test_tiles(device, nq, nk, H, causal, form, dtype):
    assert expanded_form(nq, nk, H, causal) == form
    check_expanded(device, nq, nk, H, causal, dtype, spare=2)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("nq,nk", [([1], [3000]), ([20, 0, 70, 3], [2500, 100, 900, 0]), ([90], [1700]), ([5, 64], [64, 4000])])
def test_split_keys(device, nq, nk, causal):
    assert expanded_form(nq, nk, 3, causal)[1] > 1
    check_expanded(device, nq, nk, 3, causal, spare=5)


def test_split_keys_captured_and_replayed(device):
    t = expanded.inputs(device, [40, 3], [2000, 900], H=4)
    assert expanded_form([40, 3], [2000, 900], 4)[1] > 1
    expanded.call(t)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = expanded.call(t)
    for _ in range(3):
        t["q"].normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, expanded.call(t))


@pytest.mark.parametrize("seed", range(8))
def test_random_ragged_prompts(device, seed):
    gen = torch.Generator().manual_seed(200 + seed)
    pick = lambda *options: options[int(torch.randint(0, len(options), (1,), generator=gen))]
    B, H = pick(1, 3, 7), pick(1, 4, 16, 40)
    nk = [int(x) for x in torch.randint(1, pick(80, 700, 3000), (B,), generator=gen)]
    nq = [int(torch.randint(0, min(n, 400) + 1, (1,), generator=gen)) for n in nk]
    nq[0] = max(1, nq[0])
    check_expanded(device, nq, nk, H, pick(True, False), pick("bf16", "f16"), seed, pick(0, 3))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("counts,lengths,H", [
    ([150], [1500], 96),                  # 113 tiles that token boundaries cut, shared
    ([151, 0, 3, 40], [151, 70, 3000, 2000], 128),
    ([70, 33], [40, 33], 80),             # queries before their request's first row
])
def test_unequal_tiles_of_a_request_are_shared(device, counts, lengths, H, causal):
    """Causal tiles of a request, paired from both ends, odd and even numbers of them."""
    t = paged(device, counts, lengths, H=H, L=128, R=64, page=32, spare_tokens=2)
    assert form_of(t) == [128, 256]
    check_on_device(device, t, counts, lengths, causal)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("counts,lengths,H", [
    ([128], [128], 128),                  # a tile a workgroup
    ([1] * 200, [500] * 200, 128),
    ([100, 101, 0, 99], [100, 101, 5, 99], 128),  # some a workgroup
    ([70] * 7, list(range(70, 77)), 96),
])
def test_short_tiles_are_kept_whole(device, counts, lengths, H, causal):
    t = paged(device, counts, lengths, H=H, L=128, R=64, page=16, spare_tokens=3)
    assert form_of(t) == [128, 256]
    check_on_device(device, t, counts, lengths, causal)


def test_whole_and_shared_tiles_of_one_captured_call(device):
    """Which of the two a call does follows from its lengths on the device, at each replay of a graph."""
    t = paged(device, [1] * 40, [900] * 40, H=16, L=128, R=64, page=64)
    assert form_of(t) == [64, 512]
    scale = 128 ** -0.5
    out, lse = torch.empty_like(t["q"]), torch.empty(40, 16, device=device)
    call(t, scale, True, out, lse)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(t, scale, True, out, lse)
    for lengths in ([900] * 40, [30] * 40, [900] + [1] * 39, [0] * 40, [64] * 40):
        t["seqused_kv"].copy_(torch.tensor(lengths, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        replayed, replayed_lse = out.clone(), lse.clone()
        expected = lr.latent_attention(t["q"], t["q_rope"], t["kv_cache"], t["block_table"].cpu(), t["cu_seqlens_q"].cpu(),
                                       t["seqused_kv"].cpu(), scale, True)
        finite = t["kv_cache"][torch.isfinite(t["kv_cache"])]
        compare(replayed, replayed_lse, expected, B16["bf16"], max(1, *lengths), finite.abs().max().item())


def test_a_single_request_that_fills_its_rounds(device):
    t = paged(device, [230], [260], H=128, L=128, R=64, page=32)
    assert form_of(t) == [128, 0]
    check_on_device(device, t, [230], [260])
