"""CPU checks of the latent-attention path's C ABI and entries: rejections before any launch, workspace sizes, forms, and
the rotary frequencies."""

import ctypes as ct
import math

import pytest
import torch

from ascendflow_amd import _native
from ascendflow_amd.flash_attention import latent_attention_expanded
from ascendflow_amd.sparse_attention import append_paged_kv, apply_rotary, latent_attention, rotary_frequencies, rotary_magnitude

P = ct.c_void_p


@pytest.fixture(scope="module")
def lib():
    return _native.library()


def rotary(**changes):
    fields = dict(dtype=0, layout=0, inverse=0, position_bytes=4, H=2, D=64, R=32, offset=0, B=1, S=3, x_stride_s=128,
                  x_stride_h=64, out_stride_s=128, out_stride_h=64, magnitude=1.0)
    return _native.RotaryParams(**{**fields, **changes})


def append(**changes):
    fields = dict(dtype=0, layout=0, T=3, B=2, W=4, PAGE=16, BLOCKS=8, HKV=1, DK=96, DV=0, R=32, offset=64, k_stride_t=96,
                  magnitude=1.0)
    return _native.AppendPagedKvParams(**{**fields, **changes})


def latent(**changes):
    fields = dict(dtype=0, causal=1, T=3, B=2, H=16, L=512, R=64, PAGE=128, W=4, BLOCKS=8, q_stride_t=16 * 576, q_stride_h=576,
                  q_rope_stride_t=16 * 576, q_rope_stride_h=576, out_stride_t=16 * 512, out_stride_h=512, scale=0.07)
    return _native.LatentParams(**{**fields, **changes})


def expanded(**changes):
    fields = dict(dtype=0, causal=1, Tq=300, Tk=300, B=2, H=16, D=128, R=64, q_stride_t=16 * 192, q_stride_h=192,
                  k_stride_t=16 * 256, k_stride_h=256, k_rope_stride_t=64, v_stride_t=16 * 256, v_stride_h=256,
                  out_stride_t=16 * 128, out_stride_h=128, scale=0.07)
    return _native.LatentExpandedParams(**{**fields, **changes})


@pytest.mark.parametrize("changes,status", [
    ({"dtype": 2}, -3), ({"R": 0}, -2), ({"R": 31}, -2), ({"R": 1026, "D": 2048}, -2), ({"offset": 33}, -2),
    ({"offset": -1}, -2), ({"D": 16385}, -2), ({"H": 0}, -2), ({"layout": 2}, -2), ({"position_bytes": 2}, -2),
    ({"B": -1}, -2), ({"S": 0}, 0), ({"B": 0}, 0),
])
def test_rotary_rejections(lib, changes, status):
    args = [None] + [P(16)] * 4
    assert lib.launch_apply_rotary(*args, ct.byref(rotary(**changes))) == status
    assert lib.launch_apply_rotary(None, None, P(16), P(16), P(16), ct.byref(rotary())) == -1
    assert lib.launch_apply_rotary(*args, None) == -1


def test_rotary_in_place_needs_equal_strides(lib):
    args = (None, P(1024), P(16), P(16), P(1024))
    assert lib.launch_apply_rotary(*args, ct.byref(rotary(S=3, out_stride_s=256))) == -2


@pytest.mark.parametrize("changes,status", [
    ({"dtype": 5}, -3), ({"T": -1}, -2), ({"B": 0}, -2), ({"W": 0}, -2), ({"PAGE": 0}, -2), ({"BLOCKS": 0}, -2), ({"HKV": 0}, -2),
    ({"DK": 0}, -2), ({"DV": -1}, -2), ({"R": 33}, -2), ({"offset": 65}, -2), ({"offset": -1}, -2), ({"layout": 3}, -2),
    ({"DK": 20000}, -2), ({"R": 2048, "DK": 4096, "offset": 0}, -2), ({"HKV": 1 << 16}, -2), ({"T": 0}, 0),
])
def test_append_rejections(lib, changes, status):
    args = [None, P(16), None, None] + [P(16)] * 5 + [None]
    assert lib.launch_append_paged_kv(*args, ct.byref(append(**changes))) == status
    assert lib.launch_append_paged_kv(*args, None) == -1


def test_append_pointers(lib):
    call = lambda *pointers, **changes: lib.launch_append_paged_kv(None, *pointers, ct.byref(append(**changes)))
    p = P(16)
    assert call(None, None, None, p, p, p, p, p, None) == -1             # no k
    assert call(p, None, None, p, p, p, None, p, None) == -1             # no frequencies
    assert call(p, None, None, p, p, p, p, p, None, DV=8) == -1          # no v
    assert call(p, p, None, p, p, p, p, p, None, offset=0) == -2         # rope: the row's last columns only
    assert call(p, p, None, p, p, p, p, p, None, R=0, offset=0) == -2    # rope without a rotated part


@pytest.mark.parametrize("changes,status", [
    ({"dtype": 2}, -3), ({"T": -1}, -2), ({"B": 0}, -2), ({"H": 0}, -2), ({"W": 0}, -2), ({"BLOCKS": 0}, -2), ({"L": 384}, -2),
    ({"R": 32}, -2), ({"PAGE": 8}, -2), ({"PAGE": 48}, -2), ({"scale": 0.0}, -2), ({"scale": -1.0}, -2),
    ({"scale": math.nan}, -2), ({"T": 1 << 27, "H": 16}, -2), ({"W": 1 << 24}, -2), ({"q_stride_h": 577}, -2),
    ({"out_stride_t": 4}, -2), ({"q_rope_stride_t": 7}, -2), ({"T": 0}, 0),
])
def test_latent_rejections(lib, changes, status):
    args = [None] + [P(16)] * 7 + [None, P(16), 1 << 40]
    params = latent(**changes)
    assert lib.launch_latent_attention(*args, ct.byref(params)) == status
    assert lib.launch_latent_attention(*args, None) == -1


def test_latent_workspace_and_pointers(lib):
    size = ct.c_uint64(0)
    assert lib.workspace_size_latent_attention(ct.byref(size), ct.byref(latent())) == 0 and size.value > 0
    args = [None] + [P(16)] * 7 + [None]
    for workspace, nbytes in ((None, 1 << 40), (P(16), size.value - 1), (P(24), size.value)):
        assert lib.launch_latent_attention(*args, workspace, nbytes, ct.byref(latent())) == -4
    for missing in (1, 2, 3, 4, 5, 6, 7):
        broken = list(args)
        broken[missing] = None
        assert lib.launch_latent_attention(*broken, P(16), size.value, ct.byref(latent())) == -1
    odd = list(args)
    odd[3] = P(8)
    assert lib.launch_latent_attention(*odd, P(16), size.value, ct.byref(latent())) == -2
    assert lib.workspace_size_latent_attention(ct.byref(size), ct.byref(latent(T=0))) == 0 and size.value == 0
    assert lib.workspace_size_latent_attention(None, ct.byref(latent())) == -1
    assert lib.workspace_size_latent_attention(ct.byref(size), None) == -1
    assert lib.workspace_size_latent_attention(ct.byref(size), ct.byref(latent(L=100))) == -2


@pytest.mark.parametrize("sizes,form", [
    (dict(T=1, B=1, H=64), [64, 512]),             # 64 rows: one tile of four waves
    (dict(T=1, B=1, H=65), [128, 256]),
    (dict(T=64, B=64, H=128), [128, 256]),
    (dict(T=32, B=32, H=16), [64, 512]),
    (dict(T=2000, B=1, H=128), [128, 0]),          # more tiles than the GPU holds four times: a tile a workgroup
    (dict(T=3000, B=3000, H=16), [64, 0]),
])
def test_latent_forms(lib, sizes, form):
    got = (ct.c_int64 * 2)()
    assert lib.form_latent_attention(got, ct.byref(latent(**sizes))) == 0 and list(got) == form
    size = ct.c_uint64(1)
    assert lib.workspace_size_latent_attention(ct.byref(size), ct.byref(latent(**sizes))) == 0
    rows, workers = form
    if workers == 0:
        assert size.value == 0
    else:  # parts of 512 columns, a maximum and a sum per row; a record per tile and their count
        tiles = sizes["T"] * sizes["H"] // rows + sizes["B"]
        assert size.value == 2 * workers * rows * (512 + 2) * 4 + tiles * 20 + 16
    assert lib.form_latent_attention(None, ct.byref(latent())) == -1 and lib.form_latent_attention(got, None) == -1


@pytest.mark.parametrize("changes,status", [
    ({"dtype": 2}, -3), ({"Tq": -1}, -2), ({"Tk": -1}, -2), ({"B": 0}, -2), ({"H": 0}, -2), ({"D": 64}, -2), ({"R": 32}, -2),
    ({"scale": 0.0}, -2), ({"q_stride_t": 12}, -2), ({"k_stride_t": 1 << 23}, -2), ({"k_rope_stride_t": -64}, -2),
    ({"v_stride_h": 130}, -2), ({"H": 1 << 26}, -2), ({"Tq": 0}, 0),
])
def test_expanded_rejections(lib, changes, status):
    args = [None] + [P(16)] * 7 + [None, P(16), 1 << 40]
    assert lib.launch_latent_attention_expanded(*args, ct.byref(expanded(**changes))) == status
    assert lib.launch_latent_attention_expanded(*args, None) == -1


@pytest.mark.parametrize("sizes,form", [
    (dict(Tq=8192, Tk=8192, B=1, H=32), [256, 1]),
    (dict(Tq=1500, Tk=1500, B=1, H=128), [128, 1]),
    (dict(Tq=2048, Tk=2048, B=1, H=16), [64, 1]),
    (dict(Tq=160, Tk=24000, B=8, H=8), [64, None]),
])
def test_expanded_forms(lib, sizes, form):
    got = (ct.c_int64 * 2)()
    assert lib.form_latent_attention_expanded(got, ct.byref(expanded(**sizes))) == 0
    assert got[0] == form[0] and (got[1] > 1 if form[1] is None else got[1] == form[1])
    size = ct.c_uint64(1)
    assert lib.workspace_size_latent_attention_expanded(ct.byref(size), ct.byref(expanded(**sizes))) == 0
    assert size.value == (got[1] * sizes["Tq"] * sizes["H"] * 130 * 4 if got[1] > 1 else 0)
    if size.value:
        args = [None] + [P(16)] * 7 + [None]
        for workspace, nbytes in ((None, size.value), (P(16), size.value - 1), (P(8), size.value)):
            assert lib.launch_latent_attention_expanded(*args, workspace, nbytes, ct.byref(expanded(**sizes))) == -4
    assert lib.form_latent_attention_expanded(None, ct.byref(expanded())) == -1
    assert lib.workspace_size_latent_attention_expanded(None, ct.byref(expanded())) == -1


def test_plain_frequencies():
    f = rotary_frequencies(64, 10000.0, device="cpu")
    assert f.dtype == torch.float64 and f.shape == (32,)
    assert torch.allclose(f, torch.tensor([10000.0 ** (-2 * i / 64) for i in range(32)], dtype=torch.float64), rtol=1e-14)
    assert torch.equal(rotary_frequencies(64, scaling="linear", factor=8.0, device="cpu"), f / 8)


def test_scaled_frequencies():
    f = rotary_frequencies(64, device="cpu")
    ntk = rotary_frequencies(64, scaling="ntk", factor=4.0, device="cpu")
    assert ntk[0] == f[0] and math.isclose(ntk[-1], f[-1] / 4, rel_tol=1e-12)
    yarn = rotary_frequencies(64, scaling="yarn", factor=40.0, original_length=4096, device="cpu")
    turns = 4096 * f / (2 * math.pi)
    ratio = f / yarn
    assert torch.allclose(ratio[turns > 40], torch.ones_like(ratio[turns > 40]))       # fast pairs are kept
    assert torch.allclose(ratio[turns < 0.8], torch.full_like(ratio[turns < 0.8], 40.0))  # slow ones are divided
    assert (ratio[1:] >= ratio[:-1] - 1e-9).all()
    assert rotary_magnitude(1.0) == 1.0 and math.isclose(rotary_magnitude(40.0), 0.1 * math.log(40.0) + 1)
    for bad in (dict(R=63), dict(R=0), dict(scaling="other"), dict(factor=0.5), dict(base=1.0),
                dict(scaling="yarn", factor=2.0, beta_fast=1.0, beta_slow=2.0)):
        with pytest.raises(ValueError):
            rotary_frequencies(**{"R": 64, "device": "cpu", **bad})


def test_entries_refuse_what_is_not_on_a_device():
    b16, i32 = torch.bfloat16, torch.int32
    frequencies = rotary_frequencies(32, device="cpu")
    zeros = lambda *shape, dtype=b16: torch.zeros(shape, dtype=dtype)
    with pytest.raises(ValueError, match="ROCm"):
        apply_rotary(zeros(3, 2, 64), zeros(3, dtype=i32), frequencies)
    with pytest.raises(ValueError, match="ROCm"):
        append_paged_kv(zeros(3, 1, 64), zeros(4, 16, 1, 64), zeros(2, 2, dtype=i32), zeros(3, dtype=i32), zeros(2, dtype=i32))
    with pytest.raises(ValueError, match="ROCm"):
        latent_attention(zeros(3, 2, 128), zeros(4, 16, 1, 128), zeros(2, 2, dtype=i32), zeros(3, dtype=i32),
                         zeros(2, dtype=i32), SCALE=0.1)
    with pytest.raises(ValueError, match="ROCm"):
        latent_attention_expanded(zeros(3, 2, 192), zeros(5, 2, 128), zeros(5, 64), zeros(5, 2, 128), zeros(2, dtype=i32),
                                  zeros(2, dtype=i32), SCALE=0.1)
    for call in (lambda: apply_rotary([1.0], zeros(3, dtype=i32), frequencies),
                 lambda: append_paged_kv(None, zeros(4, 16, 1, 64), None, None, None),
                 lambda: latent_attention(zeros(3, 2, 128), None, None, None, None, SCALE=0.1),
                 lambda: latent_attention_expanded(zeros(3, 2, 192), None, None, None, None, None, SCALE=0.1)):
        with pytest.raises(ValueError):
            call()


def test_absorbed_and_expanded_definitions_agree():
    """The two float64 definitions give the same attention through absorbed projections."""
    from oracle import latent_reference as lr

    gen = torch.Generator().manual_seed(0)
    normal = lambda *shape: torch.randn(shape, generator=gen, dtype=torch.float64)
    H, L, page, n, s = 3, 128, 16, 5, 21
    w_k, w_v = normal(H, L, 128) * 0.1, normal(H, L, 128) * 0.1
    c, k_rope, q = normal(s, L), normal(s, 64), normal(n, H, 192)
    k, v = torch.einsum("sl,hld->shd", c, w_k), torch.einsum("sl,hld->shd", c, w_v)
    cu = torch.tensor([0, n])
    out, lse, *_ = lr.latent_attention_expanded(q, k, k_rope, v, cu, torch.tensor([0, s]), 0.07)
    cache = torch.zeros(2, page, 1, L + 64, dtype=torch.float64)
    cache.view(-1, L + 64)[:s] = torch.cat([c, k_rope], -1)
    absorbed = torch.einsum("nhd,hld->nhl", q[..., :128], w_k)
    o, lse2, *_ = lr.latent_attention(absorbed, q[..., 128:], cache, torch.tensor([[0, 1]]), cu, torch.tensor([s]), 0.07)
    assert torch.allclose(lse, lse2, atol=1e-12) and torch.allclose(torch.einsum("nhl,hld->nhd", o, w_v), out, atol=1e-12)


def test_infinite_scales_are_refused(lib):
    args = [None] + [P(16)] * 7 + [None, P(16), 1 << 40]
    assert lib.launch_latent_attention(*args, ct.byref(latent(scale=math.inf))) == -2
    assert lib.launch_latent_attention_expanded(*args, ct.byref(expanded(scale=math.inf))) == -2
