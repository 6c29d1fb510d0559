"""Latent attention over a paged cache, absorbed form.

The dense counterpart of ``sparse_mla`` over the same kind of cache: every
token of the context is attended, no row is selected. A cache row holds the
latent c of a token, which is key and value of all heads, and behind it the
rotary key that all heads share (or nothing, where the rotation lies inside c as
in ``ori_kv``). With the key projection absorbed into the query,
``s_j = SCALE (q . c_j + q_rope . k_rope_j)`` and ``out = softmax(s) c``; the
value projection is applied to ``out`` by the caller. One call serves single-token
decode, verification of several tokens a request, and chunks of prompts
(whole prompts are cheaper in the expanded form,
``ascendflow_amd.flash_attention.latent_attention_expanded``).
"""

from __future__ import annotations

import ctypes as ct
import math
from typing import Optional

import torch

from .. import _native
from .._tensors import (DTYPES, CheckedCalls, ForwardOnly, check_apart, check_distinct_rows, check_operands,
                        check_rows, check_tensor, extents, forward_mode, launch_on, live_strides, mark_written,
                        pointers_apart, refuse_forward_mode, refuse_tangents, require, signature)

_STORAGE = {dt: name for name, dt in DTYPES.items()}


NAMES = ("q", "q_rope", "kv_cache", "block_table", "cu_seqlens_q", "seqused_kv", "out", "softmax_lse")
_calls = CheckedCalls()


def row_strides(name, tensor):
    """(token, head) strides of a tensor whose rows the kernels read in 16-byte pieces."""
    t, h = live_strides(tensor)[:2]
    require(t % 8 == 0 and h % 8 == 0, f"{name} rows must lie on 16-byte boundaries")
    return t, h


class _Call:
    """Checked sizes of a call: launcher parameters, workspace bytes and each operand's bytes (none changes afterwards)."""

    __slots__ = ("params", "nbytes", "sizes", "launch")


def _check(lib, q, q_rope, kv_cache, block_table, cu_seqlens_q, seqused_kv, out, softmax_lse, SCALE, causal):
    require(isinstance(q, torch.Tensor) and q.dim() == 3, "q must be [T, H, L]")
    b16 = q.dtype
    require(b16 in _STORAGE, f"q dtype {b16} is not supported; expected bf16 or f16")
    T, H, L = q.shape
    R = 0
    if q_rope is not None:
        require(isinstance(q_rope, torch.Tensor) and q_rope.dim() == 3, "q_rope must be [T, H, R]")
        R = q_rope.shape[2]
    require(isinstance(kv_cache, torch.Tensor) and kv_cache.dim() == 4, "kv_cache must be [BLOCKS, PAGE, 1, L + R]")
    BLOCKS, PAGE = kv_cache.shape[:2]
    require(isinstance(block_table, torch.Tensor) and block_table.dim() == 2, "block_table must be int32 [B, W]")
    B, W = block_table.shape
    i32 = torch.int32
    check_rows("q", q, q.shape, b16)
    device = q.device
    check_tensor("kv_cache", kv_cache, (BLOCKS, PAGE, 1, L + R), b16, device)
    check_tensor("block_table", block_table, (B, W), i32, device)
    check_tensor("cu_seqlens_q", cu_seqlens_q, (B + 1,), i32, device)
    check_tensor("seqused_kv", seqused_kv, (B,), i32, device)
    if q_rope is not None:
        check_rows("q_rope", q_rope, (T, H, R), b16, device)
    check_rows("out", out, (T, H, L), b16, device)
    check_distinct_rows("out", out)
    if softmax_lse is not None:
        check_tensor("softmax_lse", softmax_lse, (T, H), torch.float32, device)
    require(H > 0 and B > 0 and W > 0 and BLOCKS > 0, "heads, requests and pages must not be empty")
    require(L in (128, 256, 512), "the latent width (columns of q) must be 128, 256 or 512")
    require(R in (0, 64), "the rotary width must be 64, or 0 without q_rope")
    require(PAGE >= 16 and PAGE & (PAGE - 1) == 0, "PAGE must be a power of two from 16 on")
    require(0 < SCALE < math.inf, "positive, finite attention scale")
    qt, qh = row_strides("q", q)
    rt, rh = (0, 0) if q_rope is None else row_strides("q_rope", q_rope)
    ot, oh = row_strides("out", out)
    params = _native.LatentParams(
        dtype=_native.AFA_DTYPE[_STORAGE[b16]], causal=int(causal), T=T, B=B, H=H, L=L, R=R, PAGE=PAGE, W=W,
        BLOCKS=BLOCKS, q_stride_t=qt, q_stride_h=qh, q_rope_stride_t=rt, q_rope_stride_h=rh, out_stride_t=ot,
        out_stride_h=oh, scale=SCALE, reserved=0)
    nbytes = ct.c_uint64(0)
    _native.check(lib.workspace_size_latent_attention(ct.byref(nbytes), ct.byref(params)), "workspace_size_latent_attention")
    call = _Call()
    call.params, call.nbytes = ct.pointer(params), nbytes.value
    call.sizes = extents(q, q_rope, kv_cache, block_table, cu_seqlens_q, seqused_kv, out, softmax_lse)
    call.launch = lib.launch_latent_attention
    return call


def latent_attention(q, kv_cache, block_table, cu_seqlens_q, seqused_kv, *, SCALE, q_rope=None, CAUSAL=True, out=None,
                     softmax_lse=None):
    """Returns ``out`` [T, H, L]: dense attention of every token over its request's cache rows.

    ``q`` [T, H, L] (L 128, 256 or 512) and ``q_rope`` [T, H, 64], or None:
    bf16 or f16, any strides of tokens and heads, rows on 16 bytes. ``kv_cache``
    [BLOCKS, PAGE, 1, L + R], contiguous, R the width of ``q_rope`` or 0, PAGE a
    power of two from 16 on. ``block_table`` int32 [B, W], ``cu_seqlens_q`` int32
    [B + 1], ``seqused_kv`` int32 [B]: rows of each request, the new tokens'
    included (``append_paged_kv`` writes them). With ``CAUSAL`` token j of a
    request's n sees rows up to ``seqused_kv[b] - n + j``, without all of them.
    Rows past the table are not there; the limit goes by ``seqused_kv[b]`` as it is, as the append's places do.
    ``softmax_lse`` (optional float32 [T, H]) receives ln(sum_j exp(s_j)).

    A token that sees no row gets zeros and -inf; tokens at or past
    ``cu_seqlens_q[B]`` are left as they were (uninitialised in a new ``out``). One
    whose scores are NaN or overflow to +inf gets NaN in both.
    Rows behind ``seqused_kv`` are never read and pages outside the cache hold no
    keys, but the rows that some token of a request sees have to be finite.

    Forward only: a backward pass that reaches the result raises; with ``out`` or
    ``softmax_lse`` the call is refused where a gradient would be recorded.
    """
    lib = _native.library()
    new = out is None
    if new:
        require(isinstance(q, torch.Tensor), "q must be [T, H, L]")
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    tensors = (q, q_rope, kv_cache, block_table, cu_seqlens_q, seqused_kv, out, softmax_lse)
    check_operands(NAMES, tensors, optional=("q_rope", "softmax_lse"))
    if forward_mode():
        refuse_tangents("latent_attention", *tensors)
    graph = torch.is_grad_enabled() and (
        q.requires_grad or kv_cache.requires_grad or (q_rope is not None and q_rope.requires_grad)
        or out.requires_grad or (softmax_lse is not None and softmax_lse.requires_grad))
    require(not graph or (new and softmax_lse is None), "out and softmax_lse cannot be given where a gradient is recorded")
    SCALE, CAUSAL = float(SCALE), bool(CAUSAL)
    key = (lib, signature(*tensors), SCALE, CAUSAL)
    call = _calls.get(key) or _calls.keep(key, _check(lib, *tensors, SCALE, CAUSAL))
    pointers = [0 if t is None else t.data_ptr() for t in tensors]
    for i in (0, 1, 2, 6):
        require(pointers[i] % 16 == 0, f"{NAMES[i]} rows must lie on 16-byte boundaries")
    if not pointers_apart(pointers, call.sizes, (7,) if new and softmax_lse is not None else () if new else (6, 7)):
        check_apart([(n, t, n in ("out", "softmax_lse")) for n, t in zip(NAMES, tensors)])
    if q.shape[0]:
        workspace = None
        if call.nbytes:
            # Partial results; the caching allocator keeps the block for this stream.
            scratch = torch.empty(call.nbytes, dtype=torch.uint8, device=q.device)
            workspace = scratch.data_ptr()
        status = launch_on(q.get_device(), call.launch, *pointers, workspace, call.nbytes, call.params)
        if status:
            _native.check(status, "launch_latent_attention")
        if not new or softmax_lse is not None:
            mark_written([t for t in (None if new else out, softmax_lse) if t is not None])
    return ForwardOnly.apply("latent_attention", out, q, q_rope, kv_cache) if graph else out


@torch.library.custom_op("ascendflow_amd::latent_attention", mutates_args=())
def latent_attention_op(
    q: torch.Tensor,
    q_rope: Optional[torch.Tensor],
    kv_cache: torch.Tensor,
    block_table: torch.Tensor,
    cu_seqlens_q: torch.Tensor,
    seqused_kv: torch.Tensor,
    softmax_scale: float,
    causal: bool = True,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Framework-facing form of ``latent_attention``: returns (out [T, H, L], softmax_lse float32 [T, H])."""
    refuse_forward_mode("latent_attention")
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device)
    out = latent_attention(q, kv_cache, block_table, cu_seqlens_q, seqused_kv, SCALE=softmax_scale, q_rope=q_rope,
                           CAUSAL=causal, softmax_lse=lse)
    return out, lse


@latent_attention_op.register_fake
def _(q, q_rope, kv_cache, block_table, cu_seqlens_q, seqused_kv, softmax_scale, causal=True):
    return torch.empty(q.shape, dtype=q.dtype, device=q.device), q.new_empty(q.shape[:2], dtype=torch.float32)
