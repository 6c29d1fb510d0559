"""Append of new tokens to a paged cache held in 8 bits.

The 8-bit counterpart of ``append_paged_kv`` for key and value caches of several
heads: a block of tokens of one head shares a scale, and the codes of its rows
stand for code times scale. ``ascendflow_amd.flash_attention.quantized_attention``
reads such a cache. The tokens go where ``append_paged_kv`` would put them:
``seqused_kv`` counts the new tokens, so the last new token of request b is row
``seqused_kv[b] - 1``. Keys are rotated first, by ``apply_rotary``.
"""

from __future__ import annotations

import ctypes as ct

import torch

from .. import _native
from .._tensors import (DTYPES, CheckedCalls, check_apart, check_operands, check_rows, check_tensor, extents,
                        forward_mode, launch_on, live_strides, mark_written, pointers_apart, refuse_forward_mode,
                        refuse_tangents, require, signature)

_STORAGE = {dt: name for name, dt in DTYPES.items()}
CODES = {torch.float8_e4m3fn: "e4m3", torch.int8: "int8"}

NAMES = ("k", "v", "block_table", "cu_seqlens_q", "seqused_kv", "k_cache", "v_cache", "k_scale", "v_scale")
_calls = CheckedCalls()


class _Call:
    """Checked sizes of a call: launcher parameters and each operand's bytes (none changes afterwards)."""

    __slots__ = ("params", "sizes", "launch")


def quantized_sizes(k_cache, v_cache, k_scale, v_scale):
    """(BLOCKS, PAGE, HKV, D, GROUP) of a quantised cache whose four tensors belong together."""
    require(k_cache.dim() == 4, "k_cache must be [BLOCKS, PAGE, HKV, D]")
    codes = k_cache.dtype
    require(codes in CODES, f"k_cache dtype {codes} is not supported; expected float8_e4m3fn or int8")
    BLOCKS, PAGE, HKV, D = k_cache.shape
    require(BLOCKS > 0 and HKV > 0 and D > 0, "pages, heads and columns must not be empty")
    require(PAGE >= 16 and PAGE & (PAGE - 1) == 0, "PAGE must be a power of two from 16 on")
    check_tensor("k_cache", k_cache, k_cache.shape, codes)
    device = k_cache.device
    check_tensor("v_cache", v_cache, k_cache.shape, codes, device)
    require(k_scale.dim() == 3 and k_scale.shape[1] > 0 and PAGE % k_scale.shape[1] == 0,
            "k_scale must be float32 [BLOCKS, PAGE / GROUP, HKV]")
    GROUP = PAGE // k_scale.shape[1]
    check_tensor("k_scale", k_scale, (BLOCKS, PAGE // GROUP, HKV), torch.float32, device)
    check_tensor("v_scale", v_scale, (BLOCKS, PAGE // GROUP, HKV), torch.float32, device)
    require(16 <= GROUP <= 1024 and GROUP & (GROUP - 1) == 0, "a scale must cover 16 to 1024 tokens, a power of two of them")
    return BLOCKS, PAGE, HKV, D, GROUP


def _check(lib, k, v, block_table, cu_seqlens_q, seqused_kv, k_cache, v_cache, k_scale, v_scale):
    BLOCKS, PAGE, HKV, D, GROUP = quantized_sizes(k_cache, v_cache, k_scale, v_scale)
    device = k_cache.device
    require(k.dim() == 3, "k must be [T, HKV, D]")
    b16 = k.dtype
    require(b16 in _STORAGE, f"k dtype {b16} is not supported; expected bf16 or f16")
    T = k.shape[0]
    check_rows("k", k, (T, HKV, D), b16, device)
    check_rows("v", v, (T, HKV, D), b16, device)
    require(block_table.dim() == 2, "block_table must be int32 [B, W]")
    B, W = block_table.shape
    i32 = torch.int32
    check_tensor("block_table", block_table, (B, W), i32, device)
    check_tensor("cu_seqlens_q", cu_seqlens_q, (B + 1,), i32, device)
    check_tensor("seqused_kv", seqused_kv, (B,), i32, device)
    require(B > 0 and W > 0, "requests and pages must not be empty")
    require(D <= 1024 and HKV <= 32768 and T < 1 << 23 and B < 1 << 23,
            "at most 1024 columns, 32768 heads, and 2^23 - 1 tokens and requests")
    require(W * PAGE <= 1 << 30, "a table of at most 2^30 rows")
    kt, kh = live_strides(k)[:2]
    vt, vh = live_strides(v)[:2]
    call = _Call()
    call.params = ct.pointer(_native.AppendQuantizedKvParams(
        dtype=_native.AFA_DTYPE[_STORAGE[b16]], code=_native.AFA_CODE[CODES[k_cache.dtype]], T=T, B=B, W=W, PAGE=PAGE,
        GROUP=GROUP, BLOCKS=BLOCKS, HKV=HKV, D=D, k_stride_t=kt, k_stride_h=kh, v_stride_t=vt, v_stride_h=vh))
    call.sizes = extents(k, v, block_table, cu_seqlens_q, seqused_kv, k_cache, v_cache, k_scale, v_scale)
    call.launch = lib.launch_append_quantized_kv
    return call


def append_quantized_kv(k, v, k_cache, v_cache, k_scale, v_scale, block_table, cu_seqlens_q, seqused_kv):
    """Writes new rows ``k`` and ``v`` into a paged cache of 8-bit codes; returns ``(k_cache, v_cache)``.

    ``k`` and ``v`` [T, HKV, D]: bf16 or f16, any strides of tokens and heads, at
    most 1024 columns. ``k_cache`` and ``v_cache`` [BLOCKS, PAGE, HKV, D]:
    contiguous, float8_e4m3fn or int8, PAGE a power of two from 16 on. ``k_scale``
    and ``v_scale`` float32 [BLOCKS, PAGE / GROUP, HKV]: a scale for each block of
    GROUP tokens (a power of two, 16 to 1024) and head. ``block_table`` int32
    [B, W] (at most 2^30 rows), ``cu_seqlens_q`` int32 [B + 1], ``seqused_kv`` int32 [B]. Token j of the
    n new ones of request b goes to position ``seqused_kv[b] - n + j``.

    The scale of a block is the least power of two (from 2^-80 on) that holds its
    rows' largest finite magnitude with the largest code (448 or 127). A block
    that held rows before the new ones keeps its scale while that is enough;
    where it grows, those rows are rounded anew (in e4m3 exactly, but for codes
    that become subnormal; int8 codes stay within one step of the last scale, but
    depend on how the block was filled). Values are rounded to nearest, ties to even;
    infinities become the largest code, NaN e4m3's NaN or, in int8, 0.

    Tokens of no request, negative positions, positions beyond the table and pages
    outside the cache write nothing; rows behind the new ones are left as they are.
    Two new tokens must not name the same row, nor two requests append to one block
    (``fork_pages`` gives requests that share a page their own). Forward only:
    refused where a gradient would be recorded. The call reads no values on the
    host and can be captured in a graph.
    """
    lib = _native.library()
    tensors = (k, v, block_table, cu_seqlens_q, seqused_kv, k_cache, v_cache, k_scale, v_scale)
    check_operands(NAMES, tensors)
    if forward_mode():
        refuse_tangents("append_quantized_kv", *tensors)
    if torch.is_grad_enabled() and (k.requires_grad or v.requires_grad or k_cache.requires_grad or v_cache.requires_grad
                                    or k_scale.requires_grad or v_scale.requires_grad):
        raise ValueError("append_quantized_kv records no gradient: call it under torch.no_grad(), or on detached tensors")
    key = (lib, signature(*tensors))
    call = _calls.get(key) or _calls.keep(key, _check(lib, *tensors))
    pointers = [t.data_ptr() for t in tensors]
    if not pointers_apart(pointers, call.sizes, (5, 6, 7, 8)):
        check_apart([(n, t, n in ("k_cache", "v_cache", "k_scale", "v_scale")) for n, t in zip(NAMES, tensors)])
    if k.shape[0]:
        status = launch_on(k_cache.get_device(), call.launch, *pointers, call.params)
        if status:
            _native.check(status, "launch_append_quantized_kv")
        mark_written([k_cache, v_cache, k_scale, v_scale])
    return k_cache, v_cache


@torch.library.custom_op("ascendflow_amd::append_quantized_kv", mutates_args=("k_cache", "v_cache", "k_scale", "v_scale"))
def append_quantized_kv_op(
    k: torch.Tensor,
    v: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_scale: torch.Tensor,
    v_scale: torch.Tensor,
    block_table: torch.Tensor,
    cu_seqlens_q: torch.Tensor,
    seqused_kv: torch.Tensor,
) -> None:
    """Framework-facing form of ``append_quantized_kv``, without its refusal of gradients: torch takes the rows as constants."""
    refuse_forward_mode("append_quantized_kv")
    append_quantized_kv(k, v, k_cache, v_cache, k_scale, v_scale, block_table, cu_seqlens_q, seqused_kv)
