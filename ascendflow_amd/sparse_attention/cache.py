"""Append of new tokens to the paged caches that the attention operators read.

The attention operators take their paged caches filled. ``append_paged_kv`` writes a step's new
rows into the pages that ``block_table`` names, with the rotation of their
positions applied on the way: ``ori_kv`` of ``sparse_mla``, the latent cache of
``latent_attention``, or key and value caches of several heads. It takes the
attention call's own metadata: ``seqused_kv`` counts the new tokens, as
``seqused_ori_kv`` does there, so the last new token of request b is row
``seqused_kv[b] - 1``.
"""

from __future__ import annotations

import ctypes as ct
import math
from operator import index
from typing import Optional

import torch

from .. import _native
from .._tensors import (DTYPES, CheckedCalls, check_apart, check_operands, check_rows, check_tensor, extents,
                        forward_mode, launch_on, live_strides, mark_written, pointers_apart, refuse_forward_mode,
                        refuse_tangents, require, signature)
from .rotary import LAYOUTS

_STORAGE = {dt: name for name, dt in DTYPES.items()}


NAMES = ("k", "rope", "v", "block_table", "cu_seqlens_q", "seqused_kv", "frequencies", "k_cache", "v_cache")
_OPTIONAL = ("rope", "v", "frequencies", "v_cache")
_calls = CheckedCalls()


class _Call:
    """Checked sizes of a call: launcher parameters and each operand's bytes (none changes afterwards)."""

    __slots__ = ("params", "sizes", "launch")


def _check(lib, k, rope, v, block_table, cu_seqlens_q, seqused_kv, frequencies, k_cache, v_cache, layout, offset, magnitude):
    require(k_cache.dim() == 4, "k_cache must be [BLOCKS, PAGE, HKV, DK]")
    require(k.dim() == 3, "k must be [T, HKV, columns]")
    b16 = k_cache.dtype
    require(b16 in _STORAGE, f"k_cache dtype {b16} is not supported; expected bf16 or f16")
    BLOCKS, PAGE, HKV, DK = k_cache.shape
    T = k.shape[0]
    device = k_cache.device
    R = 0
    if frequencies is not None:
        require(frequencies.dim() == 1 and frequencies.numel() > 0, "frequencies must be a float64 [R / 2] tensor")
        R = 2 * frequencies.numel()
    check_tensor("k_cache", k_cache, k_cache.shape, b16)
    if rope is not None:
        require(R > 0, "rope needs frequencies")
        check_rows("rope", rope, (T, HKV, R), b16, device)
        offset = DK - R
    check_rows("k", k, (T, HKV, DK - R if rope is not None else DK), b16, device)
    require((v is None) == (v_cache is None), "v and v_cache go together")
    DV = 0
    if v is not None:
        require(v_cache.dim() == 4, "v_cache must be [BLOCKS, PAGE, HKV, DV]")
        DV = v_cache.shape[3]
        check_tensor("v_cache", v_cache, (BLOCKS, PAGE, HKV, DV), b16, device)
        check_rows("v", v, (T, HKV, DV), b16, device)
    require(block_table.dim() == 2, "block_table must be int32 [B, W]")
    B, W = block_table.shape
    i32 = torch.int32
    check_tensor("block_table", block_table, (B, W), i32, device)
    check_tensor("cu_seqlens_q", cu_seqlens_q, (B + 1,), i32, device)
    check_tensor("seqused_kv", seqused_kv, (B,), i32, device)
    if frequencies is not None:
        check_tensor("frequencies", frequencies, (R // 2,), torch.float64, device)
    require(R <= 1024 and DK <= 16384 and DV <= 16384 and HKV <= 32768,
            "at most 1024 rotated and 16384 columns, and 32768 heads")
    require(layout in LAYOUTS, 'layout must be "half" or "interleaved"')
    require(R == 0 or 0 <= offset <= DK - R, f"the rotated columns {offset} to {offset + R} must lie inside the row ({DK})")
    require(math.isfinite(ct.c_float(magnitude).value), "magnitude must be finite, as a float32 too")
    require(B > 0 and W > 0 and BLOCKS > 0 and PAGE > 0 and HKV > 0 and DK > 0,
            "requests, pages, heads and columns must not be empty")
    kt, kh = live_strides(k)[:2]
    rt, rh = (0, 0) if rope is None else live_strides(rope)[:2]
    vt, vh = (0, 0) if v is None else live_strides(v)[:2]
    call = _Call()
    call.params = ct.pointer(_native.AppendPagedKvParams(
        dtype=_native.AFA_DTYPE[_STORAGE[b16]], layout=LAYOUTS[layout], T=T, B=B, W=W, PAGE=PAGE, BLOCKS=BLOCKS, HKV=HKV,
        DK=DK, DV=DV, R=R, offset=offset if R else 0, k_stride_t=kt, k_stride_h=kh, rope_stride_t=rt, rope_stride_h=rh,
        v_stride_t=vt, v_stride_h=vh, magnitude=magnitude, reserved=0))
    call.sizes = extents(k, rope, v, block_table, cu_seqlens_q, seqused_kv, frequencies, k_cache, v_cache)
    call.launch = lib.launch_append_paged_kv
    return call


def append_paged_kv(k, k_cache, block_table, cu_seqlens_q, seqused_kv, v=None, v_cache=None, *, rope=None,
                    frequencies=None, layout="half", offset=0, magnitude=1.0):
    """Writes new rows ``k`` (and ``v``) into the paged ``k_cache`` (and ``v_cache``); returns the cache or both.

    ``k_cache`` [BLOCKS, PAGE, HKV, DK], ``v_cache`` [BLOCKS, PAGE, HKV, DV]:
    contiguous, bf16 or f16, at most 16384 columns and 32768 heads. ``k`` [T, HKV,
    DK] and ``v`` [T, HKV, DV]: any strides of tokens and heads. ``block_table``
    int32 [B, W], ``cu_seqlens_q`` int32 [B + 1], ``seqused_kv`` int32 [B]. Token j
    of the n new ones of request b goes to position ``seqused_kv[b] - n + j``.

    With ``frequencies`` (float64 [R / 2], as for ``apply_rotary``) the R columns
    from ``offset`` on of every key row are rotated by that position. With
    ``rope`` [T, HKV, R] as well, the rotated columns come from it, are the last
    of the row (``offset`` is not read), and ``k`` holds the DK - R others: the
    latent and the rotary key of a token as two tensors.

    Tokens of no request (at or past ``cu_seqlens_q[B]``), negative positions,
    positions beyond the table and pages outside the cache write nothing. Two new
    tokens must not name the same row. Forward only: refused where a gradient would
    be recorded. The call reads no values on the host and can be captured in a graph.
    """
    lib = _native.library()
    tensors = (k, rope, v, block_table, cu_seqlens_q, seqused_kv, frequencies, k_cache, v_cache)
    check_operands(NAMES, tensors, _OPTIONAL)
    if forward_mode():
        refuse_tangents("append_paged_kv", *tensors)
    if torch.is_grad_enabled() and (
            k.requires_grad or k_cache.requires_grad or (rope is not None and rope.requires_grad)
            or (frequencies is not None and frequencies.requires_grad)
            or (v is not None and v.requires_grad) or (v_cache is not None and v_cache.requires_grad)):
        raise ValueError("append_paged_kv records no gradient: call it under torch.no_grad(), or on detached tensors")
    offset, magnitude = index(offset), float(magnitude)
    key = (lib, signature(*tensors), layout, offset, magnitude)
    call = _calls.get(key) or _calls.keep(key, _check(lib, *tensors, layout, offset, magnitude))
    pointers = [0 if t is None else t.data_ptr() for t in tensors]
    if not pointers_apart(pointers, call.sizes, (7, 8)):
        check_apart([(n, t, n in ("k_cache", "v_cache")) for n, t in zip(NAMES, tensors)])
    if k.shape[0]:
        status = launch_on(k_cache.get_device(), call.launch, *pointers, call.params)
        if status:
            _native.check(status, "launch_append_paged_kv")
        mark_written([k_cache] if v is None else [k_cache, v_cache])
    return k_cache if v is None else (k_cache, v_cache)


@torch.library.custom_op("ascendflow_amd::append_paged_kv", mutates_args=("k_cache", "v_cache"))
def append_paged_kv_op(
    k: torch.Tensor,
    k_cache: torch.Tensor,
    block_table: torch.Tensor,
    cu_seqlens_q: torch.Tensor,
    seqused_kv: torch.Tensor,
    v: Optional[torch.Tensor] = None,
    v_cache: Optional[torch.Tensor] = None,
    rope: Optional[torch.Tensor] = None,
    frequencies: Optional[torch.Tensor] = None,
    layout: str = "half",
    offset: int = 0,
    magnitude: float = 1.0,
) -> None:
    """Framework-facing form of ``append_paged_kv``, without its refusal of gradients: torch takes the rows as constants."""
    refuse_forward_mode("append_paged_kv")
    append_paged_kv(k, k_cache, block_table, cu_seqlens_q, seqused_kv, v, v_cache, rope=rope, frequencies=frequencies,
                    layout=layout, offset=offset, magnitude=magnitude)
