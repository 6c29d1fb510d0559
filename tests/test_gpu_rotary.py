"""Rotary positions against their float64 definition: layouts, parts of the head, widths, strides, far positions, the
inverse and the gradient."""

import pytest
import torch

from ascendflow_amd.sparse_attention import apply_rotary, rotary_frequencies, rotary_magnitude
from oracle import latent_reference as lr
from tests.latent_helpers import B16

pytestmark = pytest.mark.gpu
LAYOUTS = ["half", "interleaved"]


def check(x, positions, frequencies, **kw):
    got = apply_rotary(x, positions, frequencies, **kw)
    order = (0, 2, 1, 3) if x.dim() == 4 else (0, 1, 2)  # [B, H, S, D] as [B, S, H, D]
    want = lr.rotate(x.detach().permute(order), positions, frequencies, kw.get("layout", "half"), kw.get("offset", 0),
                     kw.get("magnitude", 1.0), kw.get("inverse", False)).permute(order)
    absolute, relative = lr.rotation_bound(x, positions, frequencies, x.dtype, kw.get("magnitude", 1.0))
    assert ((got.double() - want).abs() <= absolute + relative * want.abs()).all()
    R, offset = 2 * frequencies.numel(), kw.get("offset", 0)
    assert torch.equal(got[..., :offset], x[..., :offset]) and torch.equal(got[..., offset + R:], x[..., offset + R:])
    return got


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("T,H,D,R,offset", [
    (1, 1, 2, 2, 0), (1, 1, 64, 64, 0), (5, 3, 192, 64, 128), (3, 64, 512, 64, 448), (700, 16, 128, 64, 0),
    (7, 5, 30, 10, 3), (9, 2, 34, 32, 1), (2, 4, 40, 24, 8), (33, 7, 80, 16, 32), (300, 33, 96, 96, 0), (4, 2, 24, 8, 16),
])
def test_shapes(device, T, H, D, R, offset, layout, dtype):
    gen = torch.Generator().manual_seed(T + D)
    x = torch.randn((T, H, D), generator=gen).to(B16[dtype]).to(device)
    positions = torch.randint(0, 5000, (T,), generator=gen).to(torch.int32).to(device)
    check(x, positions, rotary_frequencies(R, device=device), layout=layout, offset=offset)


@pytest.mark.parametrize("scaling", [None, "linear", "ntk", "yarn"])
def test_far_positions_and_scaled_frequencies(device, scaling):
    frequencies = rotary_frequencies(64, 10000.0, scaling=scaling, factor=40.0 if scaling else 1.0, device=device)
    x = torch.randn((8, 4, 64), device=device).bfloat16()
    magnitude = rotary_magnitude(40.0) if scaling == "yarn" else 1.0
    for dtype in (torch.int32, torch.int64):
        positions = torch.tensor([0, 1, -1, 4095, 131071, 1048575, 2**31 - 1, -(2**31)], dtype=dtype, device=device)
        check(x, positions, frequencies, magnitude=magnitude)


@pytest.mark.parametrize("layout", LAYOUTS)
def test_batch_heads_first_layout_and_shared_positions(device, layout):
    x = torch.randn((2, 5, 70, 128), device=device).half()
    frequencies = rotary_frequencies(64, device=device)
    own = torch.randint(0, 9999, (2, 70), device=device)
    check(x, own, frequencies, layout=layout, offset=64)
    check(x, own[0], frequencies, layout=layout, offset=64)
    check(x, own.t().contiguous().t()[:, :70].contiguous(), frequencies, layout=layout)


def test_strides_and_views(device):
    wide = torch.randn((40, 6, 200), device=device).bfloat16()
    positions = torch.arange(40, device=device)
    frequencies = rotary_frequencies(64, device=device)
    for view in (wide[..., 128:192], wide[..., 3:67], wide[:, ::2, 8:72], wide[::3, :, :64],
                 torch.randn((6, 40, 64), device=device).bfloat16().transpose(0, 1)):
        check(view, positions[:view.shape[0]].to(torch.int32), frequencies)


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("offset", [0, 3, 64])
def test_in_place_leaves_the_other_columns(device, layout, offset):
    x = torch.randn((50, 8, 128), device=device).bfloat16()
    positions = torch.arange(50, device=device)
    frequencies = rotary_frequencies(64 if offset != 3 else 50, device=device)
    want = apply_rotary(x, positions, frequencies, layout=layout, offset=offset)
    part = x.clone()
    assert apply_rotary(part, positions, frequencies, layout=layout, offset=offset, out=part) is part
    assert torch.equal(part, want)
    whole = torch.zeros((50, 8, 140), dtype=torch.bfloat16, device=device)
    view = whole[..., 8:136]
    view.copy_(x)
    apply_rotary(view, positions, frequencies, layout=layout, offset=offset, out=view)
    assert torch.equal(view, want) and (whole[..., :8] == 0).all() and (whole[..., 136:] == 0).all()


@pytest.mark.parametrize("layout", LAYOUTS)
def test_inverse_returns(device, layout):
    """Two roundings and two rotations in float32 apart from where it began."""
    x = torch.randn((300, 4, 64), device=device).half()
    positions = torch.randint(0, 10**6, (300,), device=device)
    frequencies = rotary_frequencies(64, device=device)
    there = apply_rotary(x, positions, frequencies, layout=layout)
    check(there, positions, frequencies, layout=layout, inverse=True)
    back = apply_rotary(there, positions, frequencies, layout=layout, inverse=True)
    u = torch.finfo(torch.float16).eps / 2
    # Each of the pair's rounded values is off by u times itself at most, and the turn back mixes both.
    assert ((back.double() - x.double()).abs() <= 3 * u * 2 * x.abs().max().item()).all()


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("entry", ["call", "op"])
def test_gradient_is_the_inverse_rotation(device, layout, entry):
    x = torch.randn((60, 3, 48), device=device).bfloat16().requires_grad_(True)
    positions = torch.arange(60, device=device) * 1000
    frequencies = rotary_frequencies(32, device=device)
    if entry == "call":
        y = apply_rotary(x, positions, frequencies, layout=layout, offset=16, magnitude=1.25)
    else:
        y = torch.ops.ascendflow_amd.apply_rotary(x, positions, frequencies, layout, 16, 1.25, False)
    grad = torch.randn_like(y)
    got, = torch.autograd.grad(y, x, grad, retain_graph=True)
    want = check(grad, positions, frequencies, layout=layout, offset=16, magnitude=1.25, inverse=True)
    assert torch.equal(got, want)
    # The map is linear: a difference of the definition along any direction is the definition of that direction,
    # and <grad, J d> = <J^T grad, d>.
    d = torch.randn(x.shape, dtype=torch.float64, device=device)
    along = lr.rotate(x.detach().double() + d, positions, frequencies, layout, 16, 1.25) - lr.rotate(
        x.detach().double(), positions, frequencies, layout, 16, 1.25)
    lhs, rhs = (grad.double() * along).sum(), (got.double() * d).sum()
    # Each of the n gradient elements is off by u |g| at most.
    u = torch.finfo(torch.bfloat16).eps / 2
    assert (lhs - rhs).abs() <= (1.01 * u * got.double().abs() * d.abs()).sum() + 1e-3
    expanded, = torch.autograd.grad(y.sum(), x)  # a gradient expanded from one element
    assert torch.equal(expanded, apply_rotary(torch.ones_like(y), positions, frequencies, layout=layout, offset=16,
                                              magnitude=1.25, inverse=True))


def test_second_derivative_is_the_rotation(device):
    x = torch.randn((5, 2, 16), device=device).half().requires_grad_(True)
    positions, frequencies = torch.arange(5, device=device), rotary_frequencies(16, device=device)
    g = torch.randn_like(x).requires_grad_(True)
    first, = torch.autograd.grad(apply_rotary(x, positions, frequencies), x, g, create_graph=True)
    h = torch.randn_like(x)
    second, = torch.autograd.grad(first, g, h)
    assert torch.equal(second, apply_rotary(h, positions, frequencies))


def test_empty_calls(device):
    frequencies = rotary_frequencies(8, device=device)
    none = torch.empty(0, dtype=torch.int32, device=device)
    assert apply_rotary(torch.empty((0, 4, 8), device=device).half(), none, frequencies).shape == (0, 4, 8)
    assert apply_rotary(torch.empty((2, 4, 0, 8), device=device).half(), none, frequencies).shape == (2, 4, 0, 8)


def test_not_finite_columns_pass(device):
    """Infinities and NaN outside the rotated part are copied, inside they stay in their pair."""
    x = torch.zeros((1, 1, 32), device=device).bfloat16()
    x[0, 0, 0], x[0, 0, 20], x[0, 0, 9] = float("inf"), float("nan"), float("nan")
    y = apply_rotary(x, torch.zeros(1, dtype=torch.int32, device=device), rotary_frequencies(16, device=device), offset=8)
    assert torch.isinf(y[0, 0, 0])
    bad = torch.isnan(y[0, 0]).nonzero().flatten().tolist()
    assert bad == [9, 12, 17, 20]


def test_captured_call(device):
    x = torch.randn((64, 8, 128), device=device).bfloat16()
    positions = torch.arange(64, device=device, dtype=torch.int32)
    frequencies = rotary_frequencies(64, device=device)
    apply_rotary(x, positions, frequencies)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = apply_rotary(x, positions, frequencies)
    for _ in range(3):
        x.normal_()
        positions += 64
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, apply_rotary(x, positions, frequencies))


def test_captured_gradient(device):
    x = torch.randn((16, 4, 64), device=device).bfloat16().requires_grad_(True)
    positions, frequencies = torch.arange(16, device=device), rotary_frequencies(64, device=device)
    grad = torch.randn_like(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(apply_rotary(x, positions, frequencies), x, grad)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, = torch.autograd.grad(apply_rotary(x, positions, frequencies), x, grad)
    for _ in range(3):
        grad.normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, apply_rotary(grad, positions, frequencies, inverse=True))


@pytest.mark.parametrize("entry", ["call", "op"])
def test_gradient_under_capture_is_refused_while_an_eager_graph_of_the_leaf_lives(device, entry, monkeypatch):
    """Nothing is captured here: such a capture would end the process, so the call has to refuse before it."""
    x = torch.randn((16, 4, 64), device=device).bfloat16().requires_grad_(True)
    positions, frequencies = torch.arange(16, device=device), rotary_frequencies(64, device=device)
    call = apply_rotary if entry == "call" else torch.ops.ascendflow_amd.apply_rotary
    eager = call(x, positions, frequencies)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="eagerly"):
        call(x, positions, frequencies)
    with torch.no_grad():
        call(x, positions, frequencies)
    del eager
    call(x, positions, frequencies)


def test_refusals(device):
    x = torch.randn((4, 2, 64), device=device).bfloat16()
    positions, frequencies = torch.arange(4, device=device), rotary_frequencies(32, device=device)
    good = dict(x=x, positions=positions, frequencies=frequencies)
    for change in (dict(x=x.float()), dict(x=x[0]), dict(x=x.cpu()), dict(x=x.transpose(1, 2)), dict(positions=positions[:3]),
                   dict(positions=positions.float()), dict(positions=positions.cpu()),
                   dict(frequencies=frequencies.float()), dict(frequencies=frequencies[:0]), dict(offset=33),
                   dict(offset=-1), dict(layout="quarter"), dict(magnitude=float("inf")),
                   dict(out=torch.empty((4, 2, 32), device=device).bfloat16()), dict(out=torch.empty_like(x).half()),
                   dict(out=x[:1].expand(4, 2, 64))):
        call = {**good, **change}
        with pytest.raises(ValueError):
            apply_rotary(call.pop("x"), call.pop("positions"), call.pop("frequencies"), **call)
    wide = torch.zeros((4, 2, 72), device=device).bfloat16()
    with pytest.raises(ValueError, match="overlap"):
        apply_rotary(wide[..., :64], positions, frequencies, out=wide[..., 8:])
    with pytest.raises(ValueError, match="gradient"):
        apply_rotary(x.clone().requires_grad_(True), positions, frequencies, out=torch.empty_like(x))
