"""Attention of grouped query heads over a paged cache held in 8 bits.

``ascendflow_amd.sparse_attention.append_quantized_kv`` fills the cache: codes
(float8_e4m3fn or int8) with a scale for each block of tokens and head.
``s_j = SCALE ks_j (q . k_j)``, ``out = sum_j e^(s_j) vs_j v_j / sum_j e^(s_j)``.
One call serves single-token decode, verification of several tokens a request,
and chunks of prompts; the metadata are those of the other paged attentions.
"""

from __future__ import annotations

import ctypes as ct
import math

import torch

from .. import _native
from .._tensors import (DTYPES, CheckedCalls, ForwardOnly, check_apart, check_distinct_rows, check_operands,
                        check_rows, check_tensor, extents, forward_mode, launch_on, live_strides, mark_written,
                        pointers_apart, refuse_forward_mode, refuse_tangents, require, signature)
from ..sparse_attention.quantized import CODES, quantized_sizes

_STORAGE = {dt: name for name, dt in DTYPES.items()}

NAMES = ("q", "k_cache", "v_cache", "k_scale", "v_scale", "block_table", "cu_seqlens_q", "seqused_kv", "out", "softmax_lse")
_calls = CheckedCalls()


class _Call:
    """Checked sizes of a call: launcher parameters, workspace bytes and each operand's bytes (none changes afterwards)."""

    __slots__ = ("params", "nbytes", "sizes", "launch")


def _check(lib, q, k_cache, v_cache, k_scale, v_scale, block_table, cu_seqlens_q, seqused_kv, out, softmax_lse, SCALE,
           causal):
    require(q.dim() == 3, "q must be [T, HQ, D]")
    b16 = q.dtype
    require(b16 in _STORAGE, f"q dtype {b16} is not supported; expected bf16 or f16")
    T, HQ, D = q.shape
    check_rows("q", q, q.shape, b16)
    device = q.device
    BLOCKS, PAGE, HKV, columns, GROUP = quantized_sizes(k_cache, v_cache, k_scale, v_scale)
    require(k_cache.device == device, f"k_cache is on {k_cache.device}, expected {device}")
    require(columns == D, f"the cache's rows have {columns} columns, q has {D}")
    require(HQ > 0 and HQ % HKV == 0, "query heads must be a multiple of the cache's heads")
    require(block_table.dim() == 2, "block_table must be int32 [B, W]")
    B, W = block_table.shape
    i32 = torch.int32
    check_tensor("block_table", block_table, (B, W), i32, device)
    check_tensor("cu_seqlens_q", cu_seqlens_q, (B + 1,), i32, device)
    check_tensor("seqused_kv", seqused_kv, (B,), i32, device)
    check_rows("out", out, (T, HQ, D), b16, device)
    check_distinct_rows("out", out)
    if softmax_lse is not None:
        check_tensor("softmax_lse", softmax_lse, (T, HQ), torch.float32, device)
    require(B > 0 and W > 0, "requests and pages must not be empty")
    require(W * PAGE <= 1 << 30 and B < 1 << 30, "a table of at most 2^30 rows, and fewer requests")
    require(D in (64, 128, 256), "the columns of a head must be 64, 128 or 256")
    require(0 < SCALE < math.inf, "positive, finite attention scale")
    qt, qh = live_strides(q)[:2]
    ot, oh = live_strides(out)[:2]
    require(qt % 8 == 0 and qh % 8 == 0, "q rows must lie on 16-byte boundaries")
    require(ot % 8 == 0 and oh % 8 == 0, "out rows must lie on 16-byte boundaries")
    params = _native.QuantizedParams(
        dtype=_native.AFA_DTYPE[_STORAGE[b16]], code=_native.AFA_CODE[CODES[k_cache.dtype]], causal=int(causal), T=T, B=B,
        HQ=HQ, HKV=HKV, D=D, PAGE=PAGE, GROUP=GROUP, W=W, BLOCKS=BLOCKS, q_stride_t=qt, q_stride_h=qh, out_stride_t=ot,
        out_stride_h=oh, scale=SCALE, reserved=0)
    nbytes = ct.c_uint64(0)
    _native.check(lib.workspace_size_quantized_attention(ct.byref(nbytes), ct.byref(params)),
                  "workspace_size_quantized_attention")
    call = _Call()
    call.params, call.nbytes = ct.pointer(params), nbytes.value
    call.sizes = extents(q, k_cache, v_cache, k_scale, v_scale, block_table, cu_seqlens_q, seqused_kv, out, softmax_lse)
    call.launch = lib.launch_quantized_attention
    return call


def quantized_attention(q, k_cache, v_cache, k_scale, v_scale, block_table, cu_seqlens_q, seqused_kv, *, SCALE, CAUSAL=True,
                        out=None, softmax_lse=None):
    """Returns ``out`` [T, HQ, D]: attention of every token over its request's rows of an 8-bit cache.

    ``q`` [T, HQ, D] (D 64, 128 or 256): bf16 or f16, any strides of tokens and
    heads, rows on 16 bytes; query head h reads cache head h / (HQ / HKV).
    ``k_cache`` and ``v_cache`` [BLOCKS, PAGE, HKV, D]: contiguous, float8_e4m3fn or
    int8, PAGE a power of two from 16 on; ``k_scale`` and ``v_scale`` float32
    [BLOCKS, PAGE / GROUP, HKV], GROUP a power of two, 16 to 1024.
    ``block_table`` int32 [B, W] (at most 2^30 rows), ``cu_seqlens_q`` int32 [B + 1], ``seqused_kv`` int32
    [B]: rows of each request, the new tokens' included (``append_quantized_kv``
    writes them). With ``CAUSAL`` token j of a request's n sees rows up to
    ``seqused_kv[b] - n + j``, without all of them. Rows past the table are not
    there; the limit goes by ``seqused_kv[b]`` as it is.
    ``softmax_lse`` (optional float32 [T, HQ]) receives ln(sum_j exp(s_j)).

    A token that sees no row gets zeros and -inf; tokens at or past
    ``cu_seqlens_q[B]`` are left as they were (uninitialised in a new ``out``). One
    whose scores are NaN or overflow to +inf gets NaN in both.
    Rows behind ``seqused_kv`` have no effect and pages outside the cache hold no
    keys, but the rows that some token of a request sees have to be finite, and
    their scales finite and positive (value scales below 2^-80 count as 2^-80).
    However far the value scales lie apart, every key has its weight in the sum;
    in ``out``, values whose weight times scale is below 2^-126 of a row's largest
    are lost. Value scales more than about 2^85 apart cost a second pass over keys.

    Forward only: a backward pass that reaches the result raises; with ``out`` or
    ``softmax_lse`` the call is refused where a gradient would be recorded.
    """
    lib = _native.library()
    new = out is None
    if new:
        require(isinstance(q, torch.Tensor), "q must be a torch.Tensor")
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    tensors = (q, k_cache, v_cache, k_scale, v_scale, block_table, cu_seqlens_q, seqused_kv, out, softmax_lse)
    check_operands(NAMES, tensors, optional=("softmax_lse",))
    if forward_mode():
        refuse_tangents("quantized_attention", *tensors)
    graph = torch.is_grad_enabled() and (
        q.requires_grad or k_cache.requires_grad or v_cache.requires_grad or k_scale.requires_grad or v_scale.requires_grad
        or out.requires_grad or (softmax_lse is not None and softmax_lse.requires_grad))
    require(not graph or (new and softmax_lse is None), "out and softmax_lse cannot be given where a gradient is recorded")
    SCALE, CAUSAL = float(SCALE), bool(CAUSAL)
    key = (lib, signature(*tensors), SCALE, CAUSAL)
    call = _calls.get(key) or _calls.keep(key, _check(lib, *tensors, SCALE, CAUSAL))
    pointers = [0 if t is None else t.data_ptr() for t in tensors]
    for i in (0, 1, 2, 8):
        require(pointers[i] % 16 == 0, f"{NAMES[i]} rows must lie on 16-byte boundaries")
    if not pointers_apart(pointers, call.sizes, (9,) if new and softmax_lse is not None else () if new else (8, 9)):
        check_apart([(n, t, n in ("out", "softmax_lse")) for n, t in zip(NAMES, tensors)])
    if q.shape[0]:
        workspace = None
        if call.nbytes:
            # Partial results; the caching allocator keeps the block for this stream.
            scratch = torch.empty(call.nbytes, dtype=torch.uint8, device=q.device)
            workspace = scratch.data_ptr()
        status = launch_on(q.get_device(), call.launch, *pointers, workspace, call.nbytes, call.params)
        if status:
            _native.check(status, "launch_quantized_attention")
        if not new or softmax_lse is not None:
            mark_written([t for t in (None if new else out, softmax_lse) if t is not None])
    return ForwardOnly.apply("quantized_attention", out, q, k_cache, v_cache, k_scale, v_scale) if graph else out


@torch.library.custom_op("ascendflow_amd::quantized_attention", mutates_args=())
def quantized_attention_op(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_scale: torch.Tensor,
    v_scale: torch.Tensor,
    block_table: torch.Tensor,
    cu_seqlens_q: torch.Tensor,
    seqused_kv: torch.Tensor,
    softmax_scale: float,
    causal: bool = True,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Framework-facing form of ``quantized_attention``: returns (out [T, HQ, D], softmax_lse float32 [T, HQ])."""
    refuse_forward_mode("quantized_attention")
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device)
    out = quantized_attention(q, k_cache, v_cache, k_scale, v_scale, block_table, cu_seqlens_q, seqused_kv,
                              SCALE=softmax_scale, CAUSAL=causal, softmax_lse=lse)
    return out, lse


@quantized_attention_op.register_fake
def _(q, k_cache, v_cache, k_scale, v_scale, block_table, cu_seqlens_q, seqused_kv, softmax_scale, causal=True):
    return torch.empty(q.shape, dtype=q.dtype, device=q.device), q.new_empty(q.shape[:2], dtype=torch.float32)
