"""Rotary positions of queries, keys and attention outputs.

The attention operators take query and cache rows already rotated.
``apply_rotary`` turns the pairs of a part of each head by ``position *
frequency``, in either pair layout, in place or into a new tensor; ``inverse=True`` turns them back, which an attention
whose values carry the rotation (``sparse_mla`` with the rotated columns inside
D) needs on its output. ``rotary_frequencies`` gives the frequencies, scaled for
long contexts or not.

The result carries its gradient (the inverse rotation of the incoming one), and
the call is registered as the torch custom op ``ascendflow_amd::apply_rotary``
with a shape-only fake and the same gradient.
"""

from __future__ import annotations

import ctypes as ct
import math
from operator import index

import torch

from .. import _native
from .._tensors import (DTYPES, CheckedCalls, check_apart, check_distinct_rows, check_operands, check_rows, extents,
                        forward_mode, has_tangent, launch_on, live_strides, mark_written, pointers_apart,
                        refuse_forward_mode, require, signature)

LAYOUTS = {"half": 0, "interleaved": 1}
_STORAGE = {dt: name for name, dt in DTYPES.items()}


def rotary_frequencies(R, base=10000.0, *, scaling=None, factor=1.0, original_length=4096, beta_fast=32.0, beta_slow=1.0,
                       device="cuda"):
    """Float64 [R / 2]: radians per position of each pair, ``base ** (-2 i / R)``.

    ``scaling`` stretches a model trained at ``original_length`` tokens to
    ``factor`` times that: ``"linear"`` divides every frequency by ``factor``,
    ``"ntk"`` raises the base so that the lowest frequency is divided by it, and
    ``"yarn"`` keeps the pairs that turn at least ``beta_fast`` times within
    ``original_length``, divides those that turn at most ``beta_slow`` times and
    blends the others between (with ``rotary_magnitude(factor)`` as magnitude).
    """
    require(isinstance(R, int) and R >= 2 and R % 2 == 0, "R must be a positive even number")
    require(scaling in (None, "linear", "ntk", "yarn"), 'scaling must be None, "linear", "ntk" or "yarn"')
    require(base > 1.0 and factor >= 1.0 and original_length > 0, "base > 1, factor >= 1, original_length > 0")
    if scaling == "ntk" and R > 2:
        base = base * factor ** (R / (R - 2))
    frequencies = base ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)
    if scaling == "linear":
        frequencies = frequencies / factor
    elif scaling == "yarn":
        require(beta_fast > beta_slow > 0, "beta_fast > beta_slow > 0")
        # Pair index at which a frequency turns `turns` times within the original length.
        low, high = (R * math.log(original_length / (turns * 2 * math.pi)) / (2 * math.log(base))
                     for turns in (beta_fast, beta_slow))
        low, high = max(0, math.floor(low)), min(R - 1, math.ceil(high))
        ramp = ((torch.arange(R // 2, dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0, 1)
        frequencies = frequencies / factor * ramp + frequencies * (1 - ramp)
    return frequencies.to(device)


def rotary_magnitude(factor, coefficient=1.0):
    """Magnitude that goes with ``"yarn"`` frequencies: 0.1 coefficient ln(factor) + 1."""
    return 0.1 * coefficient * math.log(factor) + 1.0 if factor > 1.0 else 1.0


NAMES = ("x", "positions", "frequencies", "out")
_calls = CheckedCalls()


class _Call:
    """Checked sizes of a call: launcher parameters and each operand's bytes (none changes afterwards)."""

    __slots__ = ("params", "sizes", "launch")


def _check(lib, x, positions, frequencies, out, layout, offset, magnitude, inverse):
    require(x.dim() in (3, 4), "x must be [T, H, D] or [B, H, S, D]")
    require(x.dtype in _STORAGE, f"x dtype {x.dtype} is not supported; expected bf16 or f16")
    if x.dim() == 3:
        (S, H, D), B = x.shape, 1
    else:
        B, H, S, D = x.shape
    require(H > 0 and 0 < D <= 16384, "x must have heads, and at most 16384 columns")
    require(positions.dtype in (torch.int32, torch.int64), "positions must be an int32 or int64 tensor")
    require(tuple(positions.shape) == (S,) or (x.dim() == 4 and tuple(positions.shape) == (B, S)),
            f"positions shape {tuple(positions.shape)} does not fit x {tuple(x.shape)}")
    require(frequencies.dim() == 1 and frequencies.numel() > 0, "frequencies must be a float64 [R / 2] tensor")
    check_rows("x", x, x.shape, x.dtype)
    device = x.device
    check_rows("out", out, x.shape, x.dtype, device)
    check_rows("positions", positions, positions.shape, positions.dtype, device)
    check_rows("frequencies", frequencies, frequencies.shape, torch.float64, device)
    check_distinct_rows("out", out)
    R = 2 * frequencies.numel()
    require(R <= 1024, "at most 1024 columns can be rotated")
    require(layout in LAYOUTS, 'layout must be "half" or "interleaved"')
    require(0 <= offset <= D - R, f"the rotated columns {offset} to {offset + R} must lie inside the head ({D})")
    require(math.isfinite(ct.c_float(magnitude).value), "magnitude must be finite, as a float32 too")
    xs, os = live_strides(x), live_strides(out)
    xs, os = ((0, xs[0], xs[1]), (0, os[0], os[1])) if x.dim() == 3 else ((xs[0], xs[2], xs[1]), (os[0], os[2], os[1]))
    call = _Call()
    call.params = ct.pointer(_native.RotaryParams(
        dtype=_native.AFA_DTYPE[_STORAGE[x.dtype]], layout=LAYOUTS[layout], inverse=int(inverse),
        position_bytes=positions.element_size(), H=H, D=D, R=R, offset=offset, B=B, S=S, x_stride_b=xs[0],
        x_stride_s=xs[1], x_stride_h=xs[2], out_stride_b=os[0], out_stride_s=os[1], out_stride_h=os[2],
        position_stride_b=live_strides(positions)[0] if positions.dim() == 2 else 0, magnitude=magnitude, reserved=0))
    call.sizes = extents(x, positions, frequencies, out)
    call.launch = lib.launch_apply_rotary
    return call


def _rotate(x, positions, frequencies, layout, offset, magnitude, inverse, out):
    lib = _native.library()
    new = out is None
    if new:
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    tensors = (x, positions, frequencies, out)
    key = (lib, signature(*tensors), layout, offset, magnitude, inverse)
    call = _calls.get(key) or _calls.keep(key, _check(lib, *tensors, layout, offset, magnitude, inverse))
    pointers = [t.data_ptr() for t in tensors]
    if not new and not pointers_apart(pointers, call.sizes, (3,)):
        in_place = pointers[0] == pointers[3] and live_strides(x) == live_strides(out)
        check_apart([("x", None if in_place else x, False), ("positions", positions, False),
                     ("frequencies", frequencies, False), ("out", out, True)])
    if x.numel():
        status = launch_on(x.get_device(), call.launch, *pointers, call.params)
        if status:
            _native.check(status, "launch_apply_rotary")
        if not new:
            mark_written([out])
    return out


_EAGER = "ascendflow_amd_eager_graph"


def _watch_leaf(ctx, x):
    """Marks the node that takes the gradient of a leaf as part of an eager graph, or, under capture, refuses it if marked.

    That node remembers the stream it was made on for as long as some graph holds
    it. A backward pass captured into a HIP graph would record an event on that
    other stream, which breaks the capture and ends the process."""
    node = ctx.next_functions[0][0] if ctx.next_functions else None
    if node is None or node.next_functions or not x.is_cuda:  # x is no leaf, or refused later on
        return
    if not torch.cuda.is_current_stream_capturing():
        node.metadata[_EAGER] = True
    elif node.metadata.get(_EAGER):
        raise RuntimeError("a gradient cannot be captured while a graph recorded eagerly from the same tensor lives: "
                           "drop its results before the capture")


def _refuse_frequencies(wanted):
    require(not wanted, "no gradient with respect to frequencies is computed: detach them")


class _Rotary(torch.autograd.Function):
    """The rotation as a differentiable map of x: its gradient is the inverse rotation, magnitude kept."""

    @staticmethod
    def forward(ctx, x, positions, frequencies, layout, offset, magnitude, inverse):
        _watch_leaf(ctx, x)
        _refuse_frequencies(ctx.needs_input_grad[2])
        ctx.save_for_backward(positions, frequencies)
        if forward_mode():
            ctx.save_for_forward(positions, frequencies)
        ctx.how = layout, offset, magnitude, inverse
        return _rotate(x, positions, frequencies, layout, offset, magnitude, inverse, None)

    @staticmethod
    def backward(ctx, grad):
        layout, offset, magnitude, inverse = ctx.how
        positions, frequencies = ctx.saved_tensors
        grad = _dense_rows(grad)
        if not torch.is_grad_enabled():
            turned = _rotate(grad, positions, frequencies, layout, offset, magnitude, not inverse, None)
        else:
            turned = _Rotary.apply(grad, positions, frequencies, layout, offset, magnitude, not inverse)
        return turned, None, None, None, None, None, None

    @staticmethod
    def jvp(ctx, tangent, *constants):
        positions, frequencies = ctx.saved_tensors
        return _Rotary.apply(_dense_rows(tangent), positions, frequencies, *ctx.how)


def _dense_rows(grad):
    """A gradient or tangent with contiguous rows (a sum's arrives expanded from one element)."""
    return grad if grad.shape[-1] <= 1 or grad.stride(-1) == 1 else grad.contiguous()


def apply_rotary(x, positions, frequencies, *, layout="half", offset=0, magnitude=1.0, inverse=False, out=None):
    """Returns ``x`` with the R = 2 len(frequencies) columns from ``offset`` on of every head rotated.

    ``x`` is [T, H, D] with ``positions`` [T], or [B, H, S, D] with ``positions``
    [S] or [B, S]; bf16 or f16, any strides of tokens and heads, contiguous
    columns. ``frequencies``: float64 [R / 2], radians per position. Pair i is
    columns (i, i + R / 2) of the part with ``layout="half"``, (2 i, 2 i + 1) with
    ``"interleaved"``. The rotated pairs are multiplied by ``magnitude``;
    ``inverse`` turns them by the negative angle. Positions may be any integers
    of their type, negative ones included; angles are formed in float64.

    Without ``out`` the result is a new contiguous tensor and carries its
    gradient, or forward-mode tangent, with respect to ``x`` (a captured backward
    pass of a leaf needs the leaf's eager graphs gone, and is refused otherwise;
    ``frequencies`` that require a gradient are refused too); with ``out`` (``x``
    itself for a rotation in place, otherwise memory apart from it) it is written
    there, without one.
    Raises ``ValueError`` for shapes, types, devices or overlaps that do not fit.
    """
    offset = index(offset)
    check_operands(NAMES, (x, positions, frequencies, out), optional=("out",))
    if forward_mode() and has_tangent(x, frequencies, out):
        require(out is None, "out cannot be given where a tangent is carried")
        if has_tangent(frequencies):
            raise NotImplementedError("apply_rotary has no derivative with respect to frequencies")
    elif out is not None or not (torch.is_grad_enabled() and x.requires_grad):
        if torch.is_grad_enabled():
            _refuse_frequencies(frequencies.requires_grad)
            require(out is None or not (x.requires_grad or out.requires_grad),
                    "out cannot be given where a gradient is recorded")
        return _rotate(x, positions, frequencies, layout, offset, float(magnitude), bool(inverse), out)
    return _Rotary.apply(x, positions, frequencies, layout, offset, float(magnitude), bool(inverse))


@torch.library.custom_op("ascendflow_amd::apply_rotary", mutates_args=())
def apply_rotary_op(
    x: torch.Tensor,
    positions: torch.Tensor,
    frequencies: torch.Tensor,
    layout: str = "half",
    offset: int = 0,
    magnitude: float = 1.0,
    inverse: bool = False,
) -> torch.Tensor:
    """Framework-facing form of ``apply_rotary``: returns a new contiguous tensor; no forward-mode derivative."""
    refuse_forward_mode("apply_rotary")
    return _rotate(x, positions, frequencies, layout, offset, magnitude, inverse, None)


@apply_rotary_op.register_fake
def _(x, positions, frequencies, layout="half", offset=0, magnitude=1.0, inverse=False):
    return torch.empty(x.shape, dtype=x.dtype, device=x.device)


def _op_context(ctx, inputs, output):
    x, positions, frequencies, *how = inputs
    _watch_leaf(ctx, x)
    _refuse_frequencies(ctx.needs_input_grad[2])
    ctx.save_for_backward(positions, frequencies)
    ctx.how = how


def _op_gradient(ctx, grad):
    layout, offset, magnitude, inverse = ctx.how
    turned = apply_rotary_op(_dense_rows(grad), *ctx.saved_tensors, layout, offset, magnitude, not inverse)
    return turned, None, None, None, None, None, None


apply_rotary_op.register_autograd(_op_gradient, setup_context=_op_context)
