"""What the rotary, append and latent-attention calls do where a derivative is taken: the rotation's forward-mode one, and
refusals of those that no call computes. None is dropped without a word."""

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from ascendflow_amd.sparse_attention import append_paged_kv, apply_rotary, rotary_frequencies
from tests import test_gpu_latent_expanded as expanded
from tests.latent_helpers import call, paged

pytestmark = pytest.mark.gpu


def rotary(device):
    x = torch.randn((6, 3, 64), device=device).bfloat16()
    return x, torch.arange(6, device=device) * 1000, rotary_frequencies(32, device=device)


HOW = dict(layout="interleaved", offset=16, magnitude=1.25)


@pytest.mark.parametrize("inverse", [True, False])
def test_forward_mode_of_the_rotation(device, inverse):
    x, positions, frequencies = rotary(device)
    tangent = torch.randn_like(x)
    want = apply_rotary(x, positions, frequencies, inverse=inverse, **HOW)
    turned = apply_rotary(tangent, positions, frequencies, inverse=inverse, **HOW)
    for leaf in (x, x.clone().requires_grad_(True)):
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(leaf, tangent)
            y = forward_ad.unpack_dual(apply_rotary(dual, positions, frequencies, inverse=inverse, **HOW))
            assert torch.equal(y.primal, want) and torch.equal(y.tangent, turned)
            assert forward_ad.unpack_dual(apply_rotary(x, positions, frequencies, **HOW)).tangent is None
    spread = torch.randn(64, device=device).bfloat16()[:, None, None].expand(64, 3, 6).permute(2, 1, 0)
    with forward_ad.dual_level():  # a tangent of other strides
        y = forward_ad.unpack_dual(apply_rotary(forward_ad.make_dual(x, spread), positions, frequencies, **HOW))
        assert torch.equal(y.tangent, apply_rotary(spread.contiguous(), positions, frequencies, **HOW))


def test_gradient_of_the_forward_mode_result(device):
    x, positions, frequencies = rotary(device)
    tangent, grad = torch.randn_like(x).requires_grad_(True), torch.randn_like(x)
    with forward_ad.dual_level():
        y = forward_ad.unpack_dual(apply_rotary(forward_ad.make_dual(x, tangent), positions, frequencies, **HOW)).tangent
        got, = torch.autograd.grad(y, tangent, grad)
    assert torch.equal(got, apply_rotary(grad, positions, frequencies, inverse=True, **HOW))


def test_forward_mode_refusals_of_the_rotation(device):
    x, positions, frequencies = rotary(device)
    op = torch.ops.ascendflow_amd.apply_rotary
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            op(dual, positions, frequencies)
        with pytest.raises(ValueError, match="tangent"):
            apply_rotary(dual, positions, frequencies, out=torch.empty_like(x))
        with pytest.raises(NotImplementedError, match="frequencies"):
            apply_rotary(x, positions, forward_ad.make_dual(frequencies, torch.ones_like(frequencies)))
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda x: op(x, positions, frequencies), (x,), (torch.ones_like(x),))
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda x: apply_rotary(x, positions, frequencies), (x,), (torch.ones_like(x),))


def with_tangent(tensors, name):
    return {**tensors, name: forward_ad.make_dual(tensors[name], torch.ones_like(tensors[name]))}


@pytest.mark.parametrize("name", ["q", "q_rope", "kv_cache"])
def test_forward_mode_refusals_of_the_absorbed_form(device, name):
    t = paged(device, [1, 2], [40, 70], H=8, page=64)
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(with_tangent(t, name), 0.1)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            d = with_tangent(t, name)
            torch.ops.ascendflow_amd.latent_attention(d["q"], d["q_rope"], d["kv_cache"], t["block_table"], t["cu_seqlens_q"],
                                                      t["seqused_kv"], 0.1)
        assert torch.equal(call(t, 0.1), call(t, 0.1))  # nothing carries a tangent


@pytest.mark.parametrize("name", ["q", "k_nope", "k_rope", "v"])
def test_forward_mode_refusals_of_the_expanded_form(device, name):
    t = expanded.inputs(device, [5, 3], [40, 30], H=8)
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            expanded.call(with_tangent(t, name))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            d = with_tangent(t, name)
            torch.ops.ascendflow_amd.latent_attention_expanded(d["q"], d["k_nope"], d["k_rope"], d["v"], t["cu_q"], t["cu_k"], 0.1)
        expanded.call(t)


def append_inputs(device):
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=device)
    zeros = lambda *shape: torch.zeros(shape, dtype=torch.bfloat16, device=device)
    return dict(k=zeros(3, 2, 32), k_cache=zeros(2, 16, 2, 64), block_table=i32(1, 0)[None], cu_seqlens_q=i32(0, 3),
                seqused_kv=i32(20), v=zeros(3, 2, 64), v_cache=zeros(2, 16, 2, 64), rope=zeros(3, 2, 32),
                frequencies=rotary_frequencies(32, device=device))


@pytest.mark.parametrize("name", ["k", "rope", "v", "frequencies", "k_cache", "v_cache"])
def test_forward_mode_refusals_of_the_append(device, name):
    t = append_inputs(device)
    with forward_ad.dual_level():
        for entry in (append_paged_kv, torch.ops.ascendflow_amd.append_paged_kv):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                entry(**with_tangent(t, name))
        append_paged_kv(**t)


def test_gradients_of_the_frequencies_are_refused(device):
    x, positions, frequencies = rotary(device)
    learned = frequencies.clone().requires_grad_(True)
    for leaf in (x, x.clone().requires_grad_(True)):
        for entry in (apply_rotary, torch.ops.ascendflow_amd.apply_rotary):
            with pytest.raises(ValueError, match="frequencies"):
                entry(leaf, positions, learned)
    with pytest.raises(ValueError, match="frequencies"):
        apply_rotary(x, positions, learned, out=torch.empty_like(x))
    with torch.no_grad():
        assert torch.equal(apply_rotary(x, positions, learned), apply_rotary(x, positions, frequencies))


def wanting(tensors, name):
    return {**tensors, name: tensors[name].clone().requires_grad_(True)}


def check_forward_only(run, tensors, name):
    """``run(tensors, **outputs)``: the plain result, whose backward pass raises; no result is written without a word."""
    plain = run(tensors)
    t = wanting(tensors, name)
    out = run(t)
    assert torch.equal(out, plain)
    with pytest.raises(RuntimeError, match="forward only"):
        (out.sum() + t[name].sum()).backward()
    for given in (dict(out=torch.empty_like(plain)),
                  dict(softmax_lse=torch.empty(plain.shape[:2], dtype=torch.float32, device=plain.device))):
        with pytest.raises(ValueError, match="gradient"):
            run(t, **given)
        with torch.no_grad():
            assert torch.equal(run(t, **given), plain)
    with torch.inference_mode():
        assert torch.equal(run(t), plain)


@pytest.mark.parametrize("name", ["q", "q_rope", "kv_cache"])
def test_the_absorbed_form_is_forward_only(device, name):
    t = paged(device, [1, 2], [40, 70], H=8, page=64)
    check_forward_only(lambda t, out=None, softmax_lse=None: call(t, 0.1, True, out, softmax_lse), t, name)
    t = wanting(t, name)
    out, _ = torch.ops.ascendflow_amd.latent_attention(t["q"], t["q_rope"], t["kv_cache"], t["block_table"], t["cu_seqlens_q"],
                                                       t["seqused_kv"], 0.1)
    with pytest.raises((RuntimeError, NotImplementedError)):
        out.sum().backward()


@pytest.mark.parametrize("name", ["q", "k_nope", "k_rope", "v"])
def test_the_expanded_form_is_forward_only(device, name):
    t = expanded.inputs(device, [5, 3], [40, 30], H=8)
    check_forward_only(lambda t, **kw: expanded.call(t, **kw), t, name)
    t = wanting(t, name)
    out, _ = torch.ops.ascendflow_amd.latent_attention_expanded(t["q"], t["k_nope"], t["k_rope"], t["v"], t["cu_q"], t["cu_k"], 0.1)
    with pytest.raises((RuntimeError, NotImplementedError)):
        out.sum().backward()


@pytest.mark.parametrize("name", ["k", "rope", "v", "frequencies", "k_cache", "v_cache"])
def test_the_append_records_no_gradient(device, name):
    t = wanting(append_inputs(device), name)
    with pytest.raises(ValueError, match="gradient"):
        append_paged_kv(**t)
    with torch.no_grad():
        append_paged_kv(**t)
