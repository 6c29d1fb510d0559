"""Latent attention of prompts, expanded form.

Keys and values of every head are expanded from the latents by the caller (one
matrix product), and each head's keys share one rotary part:
``s_j = SCALE (q[:128] . k_nope[j, h] + q[128:] . k_rope[j])``,
``out = softmax(s) v[:, h]``. 640 flops a (query, key, head) instead of the
absorbed form's 2176 at a latent of 512
(``ascendflow_amd.sparse_attention.latent_attention``). The two parts of a key
are read from where they lie: no per-head copy of ``k_rope`` is made.
"""

from __future__ import annotations

import ctypes as ct
import math

import torch

from .. import _native
from .._tensors import (DTYPES, CheckedCalls, ForwardOnly, check_apart, check_distinct_rows, check_operands,
                        check_rows, check_tensor, extents, forward_mode, launch_on, live_strides, mark_written,
                        pointers_apart, refuse_forward_mode, refuse_tangents, require, signature)

_STORAGE = {dt: name for name, dt in DTYPES.items()}
D, R = 128, 64  # columns of k_nope and v, and of k_rope


NAMES = ("q", "k_nope", "k_rope", "v", "cu_seqlens_q", "cu_seqlens_k", "out", "softmax_lse")
_calls = CheckedCalls()


class _Call:
    """Checked sizes of a call: launcher parameters, workspace bytes and each operand's bytes (none changes afterwards)."""

    __slots__ = ("params", "nbytes", "sizes", "launch")


def _check(lib, q, k_nope, k_rope, v, cu_seqlens_q, cu_seqlens_k, out, softmax_lse, SCALE, causal):
    require(q.dim() == 3, f"q must be [Tq, H, {D + R}]")
    b16 = q.dtype
    require(b16 in _STORAGE, f"q dtype {b16} is not supported; expected bf16 or f16")
    Tq, H = q.shape[:2]
    require(k_rope.dim() == 2, f"k_rope must be [Tk, {R}]")
    Tk = k_rope.shape[0]
    check_rows("q", q, (Tq, H, D + R), b16)
    device = q.device
    check_rows("k_nope", k_nope, (Tk, H, D), b16, device)
    check_rows("k_rope", k_rope, (Tk, R), b16, device)
    check_rows("v", v, (Tk, H, D), b16, device)
    require(cu_seqlens_q.dim() == 1, "cu_seqlens_q must be int32 [B + 1]")
    B = cu_seqlens_q.numel() - 1
    check_tensor("cu_seqlens_q", cu_seqlens_q, (B + 1,), torch.int32, device)
    check_tensor("cu_seqlens_k", cu_seqlens_k, (B + 1,), torch.int32, device)
    check_rows("out", out, (Tq, H, D), b16, device)
    check_distinct_rows("out", out)
    if softmax_lse is not None:
        check_tensor("softmax_lse", softmax_lse, (Tq, H), torch.float32, device)
    require(B > 0 and H > 0, "positive request and head counts")
    require(0 < SCALE < math.inf, "positive, finite attention scale")
    strides = []
    for name, t in (("q", q), ("k_nope", k_nope), ("k_rope", k_rope), ("v", v), ("out", out)):
        mine = live_strides(t)[:-1]
        require(all(s % 8 == 0 for s in mine), f"{name} rows must lie on 16-byte boundaries")
        if name in ("k_nope", "k_rope", "v"):
            require(mine[0] < 2**23, f"{name} tokens may lie at most 2^23 - 1 elements apart")
        strides += mine
    qt, qh, kt, kh, rt, vt, vh, ot, oh = strides
    params = _native.LatentExpandedParams(
        dtype=_native.AFA_DTYPE[_STORAGE[b16]], causal=int(causal), Tq=Tq, Tk=Tk, B=B, H=H, D=D, R=R, q_stride_t=qt,
        q_stride_h=qh, k_stride_t=kt, k_stride_h=kh, k_rope_stride_t=rt, v_stride_t=vt, v_stride_h=vh, out_stride_t=ot,
        out_stride_h=oh, scale=SCALE, reserved=0)
    nbytes = ct.c_uint64(0)
    _native.check(lib.workspace_size_latent_attention_expanded(ct.byref(nbytes), ct.byref(params)),
                  "workspace_size_latent_attention_expanded")
    call = _Call()
    call.params, call.nbytes = ct.pointer(params), nbytes.value
    call.sizes = extents(q, k_nope, k_rope, v, cu_seqlens_q, cu_seqlens_k, out, softmax_lse)
    call.launch = lib.launch_latent_attention_expanded
    return call


def latent_attention_expanded(q, k_nope, k_rope, v, cu_seqlens_q, cu_seqlens_k, *, SCALE, CAUSAL=True, out=None,
                              softmax_lse=None):
    """Returns ``out`` [Tq, H, 128]: attention of ragged requests over their own keys.

    ``q`` [Tq, H, 192] (128 columns against ``k_nope``, 64 rotated ones against
    ``k_rope``), ``k_nope`` and ``v`` [Tk, H, 128], ``k_rope`` [Tk, 64]: bf16 or
    f16, any strides of tokens and heads (views of one projection), rows on 16
    bytes. ``cu_seqlens_q`` and ``cu_seqlens_k`` int32 [B + 1]. With ``CAUSAL``
    query i of a request's nq sees keys up to nk - nq + i (the queries are the
    last of the context), without all of them. ``softmax_lse`` (optional float32
    [Tq, H]) receives ln(sum_j exp(s_j)).

    A query that sees no key gets zeros and -inf; queries at or past
    ``cu_seqlens_q[B]`` are left as they were (uninitialised in a new ``out``). One
    whose scores are NaN or overflow to +inf gets NaN in both.
    Keys and values that some query of a request sees have to be finite.

    Forward only: a backward pass that reaches the result raises; with ``out`` or
    ``softmax_lse`` the call is refused where a gradient would be recorded.
    """
    lib = _native.library()
    new = out is None
    if new:
        require(isinstance(q, torch.Tensor) and q.dim() == 3, f"q must be [Tq, H, {D + R}]")
        out = torch.empty((*q.shape[:2], D), dtype=q.dtype, device=q.device)
    tensors = (q, k_nope, k_rope, v, cu_seqlens_q, cu_seqlens_k, out, softmax_lse)
    check_operands(NAMES, tensors, optional=("softmax_lse",))
    if forward_mode():
        refuse_tangents("latent_attention_expanded", *tensors)
    graph = torch.is_grad_enabled() and (
        q.requires_grad or k_nope.requires_grad or k_rope.requires_grad or v.requires_grad
        or out.requires_grad or (softmax_lse is not None and softmax_lse.requires_grad))
    require(not graph or (new and softmax_lse is None), "out and softmax_lse cannot be given where a gradient is recorded")
    SCALE, CAUSAL = float(SCALE), bool(CAUSAL)
    key = (lib, signature(*tensors), SCALE, CAUSAL)
    call = _calls.get(key) or _calls.keep(key, _check(lib, *tensors, SCALE, CAUSAL))
    pointers = [0 if t is None else t.data_ptr() for t in tensors]
    for i in (0, 1, 2, 3, 6):
        require(pointers[i] % 16 == 0, f"{NAMES[i]} rows must lie on 16-byte boundaries")
    if not pointers_apart(pointers, call.sizes, (7,) if new and softmax_lse is not None else () if new else (6, 7)):
        check_apart([(n, t, n in ("out", "softmax_lse")) for n, t in zip(NAMES, tensors)])
    if q.shape[0]:
        workspace = None
        if call.nbytes:
            # Partial results of split keys; the caching allocator keeps the block for this stream.
            scratch = torch.empty(call.nbytes, dtype=torch.uint8, device=q.device)
            workspace = scratch.data_ptr()
        status = launch_on(q.get_device(), call.launch, *pointers, workspace, call.nbytes, call.params)
        if status:
            _native.check(status, "launch_latent_attention_expanded")
        if not new or softmax_lse is not None:
            mark_written([t for t in (None if new else out, softmax_lse) if t is not None])
    return ForwardOnly.apply("latent_attention_expanded", out, q, k_nope, k_rope, v) if graph else out


@torch.library.custom_op("ascendflow_amd::latent_attention_expanded", mutates_args=())
def latent_attention_expanded_op(
    q: torch.Tensor,
    k_nope: torch.Tensor,
    k_rope: torch.Tensor,
    v: torch.Tensor,
    cu_seqlens_q: torch.Tensor,
    cu_seqlens_k: torch.Tensor,
    softmax_scale: float,
    causal: bool = True,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Framework-facing form of ``latent_attention_expanded``: returns (out, softmax_lse float32 [Tq, H])."""
    refuse_forward_mode("latent_attention_expanded")
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device)
    out = latent_attention_expanded(q, k_nope, k_rope, v, cu_seqlens_q, cu_seqlens_k, SCALE=softmax_scale, CAUSAL=causal,
                                    softmax_lse=lse)
    return out, lse


@latent_attention_expanded_op.register_fake
def _(q, k_nope, k_rope, v, cu_seqlens_q, cu_seqlens_k, softmax_scale, causal=True):
    return (torch.empty((*q.shape[:2], D), dtype=q.dtype, device=q.device),
            q.new_empty(q.shape[:2], dtype=torch.float32))
