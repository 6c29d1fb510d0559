"""How the split form of absorbed latent attention shares its work: more requests than a workgroup has threads, whole and
shared tiles told apart by the workspace, streamed loads and both joins by the form."""

import ctypes as ct

import pytest
import torch

from ascendflow_amd import _native
from oracle import latent_reference as lr
from tests.latent_helpers import call, compare, paged
from tests.test_gpu_latent_forms import form_of

pytestmark = pytest.mark.gpu


def params_of(t, out, scale, causal=True):
    T, H, L = t["q"].shape
    blocks, page, _, row = t["kv_cache"].shape
    B, width = t["block_table"].shape
    strides = lambda x: x.stride()[:2]
    (qt, qh), (rt, rh), (ot, oh) = strides(t["q"]), strides(t["q_rope"]) if row > L else (0, 0), strides(out)
    return _native.LatentParams(dtype=_native.AFA_DTYPE["f16" if out.dtype == torch.float16 else "bf16"], causal=int(causal),
                                T=T, B=B, H=H, L=L, R=row - L, PAGE=page, W=width, BLOCKS=blocks, q_stride_t=qt, q_stride_h=qh,
                                q_rope_stride_t=rt, q_rope_stride_h=rh, out_stride_t=ot, out_stride_h=oh, scale=scale)


def split_form(t):
    got = (ct.c_int64 * 2)()
    assert _native.library().split_form_latent_attention(got, ct.byref(params_of(t, t["q"], 1.0))) == 0
    return list(got)


def run(t, scale, causal=True):
    """(out, lse, tiles that the call shared, 0 if it kept them whole): the C entry with a workspace that is looked at."""
    lib, device = _native.library(), t["q"].device
    out = torch.full_like(t["q"], 7.0)
    lse = torch.full(out.shape[:2], 7.0, device=device)
    params, nbytes = params_of(t, out, scale, causal), ct.c_uint64(0)
    assert lib.workspace_size_latent_attention(ct.byref(nbytes), ct.byref(params)) == 0
    rows, workers = form_of(t)
    assert workers > 0
    workspace = torch.full((nbytes.value,), 255, dtype=torch.uint8, device=device)  # NaN as float32
    pointer = lambda x: ct.c_void_p(0 if x is None else x.data_ptr())
    names = ("q", "q_rope", "kv_cache", "block_table", "cu_seqlens_q", "seqused_kv")
    assert lib.launch_latent_attention(ct.c_void_p(torch.cuda.current_stream().cuda_stream), *(pointer(t[n]) for n in names),
                                       pointer(out), pointer(lse), pointer(workspace), nbytes.value, ct.byref(params)) == 0
    torch.cuda.synchronize()
    at = 2 * workers * rows * (out.shape[2] + 2) * 4
    return out, lse, workspace[at:at + 4].view(torch.int32).item()


def check(t, counts, lengths, scale, causal=True):
    out, lse, shared = run(t, scale, causal)
    expected = lr.latent_attention(t["q"], t["q_rope"], t["kv_cache"], t["block_table"].cpu(), t["cu_seqlens_q"].cpu(),
                                   t["seqused_kv"].cpu(), scale, causal)
    finite = t["kv_cache"][torch.isfinite(t["kv_cache"])]
    compare(out, lse, expected, out.dtype, max(1, *lengths), finite.abs().max().item())
    assert (out[sum(counts):] == 7).all() and (lse[sum(counts):] == 7).all()
    assert torch.equal(out[:sum(counts)], call(t, scale, causal)[:sum(counts)])
    return shared


@pytest.mark.parametrize("B,H,rows,per", [(300, 16, 64, 2), (1000, 16, 64, 4), (513, 8, 64, 3), (600, 65, 128, 2)])
@pytest.mark.parametrize("shape", ["equal", "one long", "random"])
def test_more_requests_than_threads(device, B, H, rows, per, shape):
    """``per`` consecutive requests a thread, empty ones of both kinds among them."""
    gen = torch.Generator().manual_seed(B)
    counts = torch.randint(0, 3 if H == 16 and B < 1000 else 2, (B,), generator=gen).tolist()
    lengths = torch.randint(0, 90, (B,), generator=gen).tolist()
    if shape == "equal":
        lengths = [64] * B
    elif shape == "one long":
        counts[B // 2 + 1], lengths[B // 2 + 1] = 1, 9000
    if H == 65:
        counts = [2 * n for n in counts]
    t = paged(device, counts, lengths, H=H, L=128, R=64, page=16, spare_tokens=2)
    assert form_of(t) == [rows, 256 if rows == 128 else 512] and -(-B // (4 * rows)) == per
    shared = check(t, counts, lengths, 0.1)
    tiles = sum(-(-n * H // rows) for n in counts)
    assert shared == (tiles if shape == "one long" else 0)


@pytest.mark.parametrize("counts,lengths,H,page,whole", [
    ([128], [128], 128, 16, True), ([1] * 200, [500] * 200, 128, 16, True), ([100, 101, 0, 99], [100, 101, 5, 99], 128, 16, True),
    ([70] * 7, list(range(70, 77)), 96, 16, True), ([1] * 40, [30] * 40, 16, 64, True), ([1] * 40, [4000] * 40, 16, 64, False),
    ([150], [1500], 96, 32, False), ([1], [5000], 16, 64, False), ([0, 3], [10, 0], 16, 64, True),
])
def test_whole_and_shared_tiles(device, counts, lengths, H, page, whole):
    t = paged(device, counts, lengths, H=H, L=128, R=64, page=page, spare_tokens=3)
    rows = form_of(t)[0]
    assert check(t, counts, lengths, 0.1) == (0 if whole else sum(-(-n * H // rows) for n in counts))


@pytest.mark.parametrize("H", [16, 128])
def test_streamed_cache(device, H):
    t = paged(device, [1, 1, 1], [900, 33, 300], H=H, L=512, R=64, page=128)
    assert split_form(t)[0] == 0
    large = torch.full((1000, 128, 1, 576), float("nan"), dtype=torch.bfloat16, device=device)
    large[:t["kv_cache"].shape[0]] = t["kv_cache"]
    large = dict(t, kv_cache=large)
    assert split_form(large)[0] == 1
    a, b = run(t, 0.05), run(large, 0.05)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and a[2] == b[2] > 0


@pytest.mark.parametrize("counts,lengths,H,L,waves", [
    ([1], [5000], 16, 512, 16), ([1] * 12, [3000] * 12, 16, 512, 16), ([1] * 20, [3000] * 20, 16, 512, 1),
    ([1, 2], [5000, 900], 96, 512, 16), ([2] * 6, [2000] * 6, 128, 512, 1),
])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_both_joins(device, counts, lengths, H, L, waves, dtype):
    t = paged(device, counts, lengths, H=H, L=L, R=64, page=64, dtype=dtype)
    assert split_form(t)[1] == waves
    assert check(t, counts, lengths, 0.05) > 0
