"""Upkeep of the pages of a paged cache: copies, forks with copies on write, releases, reservations and compaction.

A row of ``block_table`` [B, W] names the pages of one request, -1 where it has
none; ``page_counts`` [BLOCKS] holds the number of references of each page, 0 for
a free one. The calls change both on the device and read no values on the host,
so that a decode loop that samples several continuations, ends requests and
starts others can run in a captured graph. They serve every cache whose first
dimension is the page: those of ``append_paged_kv`` and ``append_quantized_kv``,
scales included, ``ori_kv`` and ``cmp_kv``.
"""

from __future__ import annotations

import ctypes as ct
from operator import index

import torch

from .. import _native
from .._tensors import (CheckedCalls, check_apart, check_operands, check_tensor, extents, forward_mode, launch_on,
                        mark_written, pointers_apart, refuse_forward_mode, refuse_tangents, require, signature)

_copies, _forks, _compactions = CheckedCalls(), CheckedCalls(), CheckedCalls()


class _Call:
    """Checked sizes of a call: launcher arguments and each operand's bytes (none changes afterwards)."""

    __slots__ = ("params", "nbytes", "sizes", "launch", "written")


def _check_copies(lib, source, destination, caches):
    require(len(caches) > 0, "caches must name at least one tensor")
    first = caches[0]
    require(first.dim() >= 2 and first.numel() > 0, "a cache must be [BLOCKS, ...], not empty")
    BLOCKS, device = first.shape[0], first.device
    require(BLOCKS < 1 << 31 and source.numel() < 1 << 31, "at most 2^31 - 1 pages and pairs")
    for i, cache in enumerate(caches):
        require(cache.dim() >= 2 and cache.numel() > 0, "a cache must be [BLOCKS, ...], not empty")
        check_tensor(f"caches[{i}]", cache, (BLOCKS, *cache.shape[1:]), cache.dtype, device)
    require(source.dim() == 1, "source must be int32 [pairs]")
    pairs = source.shape[0]
    check_tensor("source", source, (pairs,), torch.int32, device)
    check_tensor("destination", destination, (pairs,), torch.int32, device)
    n = len(caches)
    call = _Call()
    call.params = (BLOCKS, pairs, n, (ct.c_uint64 * n)(*[c.numel() // BLOCKS * c.element_size() for c in caches]))
    call.sizes = extents(source, destination, *caches)
    call.launch = lib.launch_copy_pages
    call.written = tuple(range(2, 2 + n))
    return call


def copy_pages(caches, source, destination):
    """Copies page ``source[i]`` to page ``destination[i]`` in every one of ``caches``; returns None.

    ``caches``: a tensor or a sequence of them, contiguous, of any type, the first
    dimension the page (key, value and scale tensors of all layers at once).
    ``source`` and ``destination`` int32 [pairs], as ``fork_pages`` and
    ``compact_pages`` give them: a pair with a number outside the cache (-1) copies
    nothing. No page may be a destination twice, or a destination and a source.
    A list that ``compact_pages`` returns is taken whatever its length; a call that
    is refused has copied nothing.
    Refused where a gradient would be recorded; can be captured in a graph.
    """
    lib = _native.library()
    caches = (caches,) if isinstance(caches, torch.Tensor) else tuple(caches)
    tensors = (source, destination, *caches)
    check_operands(("source", "destination", *(f"caches[{i}]" for i in range(len(caches)))), tensors)
    if forward_mode():
        refuse_tangents("copy_pages", *tensors)
    if torch.is_grad_enabled() and any([c.requires_grad for c in caches]):
        raise ValueError("copy_pages records no gradient: call it under torch.no_grad(), or on detached tensors")
    key = (lib, signature(*tensors))
    call = _copies.get(key) or _copies.keep(key, _check_copies(lib, *tensors[:2], caches))
    pointers = [t.data_ptr() for t in tensors]
    if len(set(pointers[2:])) < len(caches) or not pointers_apart(pointers, call.sizes, call.written):
        check_apart([(n, t, n[0] == "c") for n, t in zip(
            ("source", "destination", *(f"caches[{i}]" for i in range(len(caches)))), tensors)])
    BLOCKS, pairs, n, page_bytes = call.params
    if pairs:
        status = launch_on(source.get_device(), call.launch, (ct.c_void_p * n)(*pointers[2:]), page_bytes, n, *pointers[:2],
                           pairs, BLOCKS)
        if status:
            _native.check(status, "launch_copy_pages")
        mark_written(list(caches))


def _check_tables(block_table, page_counts):
    require(block_table.dim() == 2, "block_table must be int32 [B, W]")
    B, W = block_table.shape
    require(page_counts.dim() == 1, "page_counts must be int32 [BLOCKS]")
    BLOCKS = page_counts.shape[0]
    check_tensor("block_table", block_table, (B, W), torch.int32)
    check_tensor("page_counts", page_counts, (BLOCKS,), torch.int32, block_table.device)
    require(B > 0 and W > 0 and BLOCKS > 0, "requests and pages must not be empty")
    return B, W, BLOCKS


def _check_fork(lib, block_table, page_counts, parents, seqused_kv, PAGE, reserve):
    B, W, BLOCKS = _check_tables(block_table, page_counts)
    check_tensor("parents", parents, (B,), torch.int32, block_table.device)
    check_tensor("seqused_kv", seqused_kv, (B,), torch.int32, block_table.device)
    require(PAGE > 0 and PAGE & (PAGE - 1) == 0 and PAGE <= 1 << 20, "PAGE must be a power of two up to 2^20")
    require(0 <= reserve <= 1 << 20, "reserve must be 0 to 2^20 tokens")
    require(B <= 8192 and B * W < 1 << 31 and BLOCKS <= 1 << 28,
            "at most 8192 requests, 2^31 - 1 entries of a table and 2^28 pages")
    params = _native.ForkPagesParams(B=B, W=W, PAGE=PAGE, BLOCKS=BLOCKS, reserve=reserve)
    nbytes = ct.c_uint64(0)
    _native.check(lib.workspace_size_fork_pages(ct.byref(nbytes), ct.byref(params)), "workspace_size_fork_pages")
    call = _Call()
    call.params, call.nbytes = ct.pointer(params), nbytes.value
    call.sizes = extents(block_table, page_counts, parents, seqused_kv)
    call.launch = lib.launch_fork_pages
    return call


def fork_pages(block_table, page_counts, parents, seqused_kv, *, PAGE, reserve=0):
    """Makes row b of ``block_table`` a copy of row ``parents[b]``; returns ``(source, destination, missing)``.

    ``block_table`` int32 [B, W] (at most 8192 rows) and ``page_counts`` int32 [BLOCKS] are changed in
    place. ``parents`` int32 [B] names rows as they are before the call:
    ``parents[b] == b`` goes on, another number continues from that row (a beam, a
    further sample of a prompt), a number outside the table (-1) ends the row and
    releases its pages. ``seqused_kv`` int32 [B] is the length of row b
    afterwards: it keeps the pages of its tokens and gets free ones for
    ``reserve`` tokens more, the lowest first, row by row.

    Full pages are shared. A page that row b will go on writing to (its last one,
    partly filled) is replaced by a free one where others hold it too (the lowest
    of the rows that write to it keeps it, unless somebody else holds it), and has
    to be copied: ``copy_pages(caches, source, destination)``, both int32 [B], -1
    where there is nothing to copy. ``missing`` int32 [1] counts the pages that
    were wanted beyond the free ones or the table's width, whose entries are -1:
    the attentions find no keys there and the appends write nothing.

    A call that lacks pages loses state: a row whose partly filled page had to be
    copied and could not be has -1 in its place, its tokens there are gone for
    that row (whoever else holds the page keeps it), and no later call wants that
    entry again or counts it in ``missing``. Where pages may run out, keep
    copies of ``block_table`` and ``page_counts`` from before the call and read
    ``missing`` before ``copy_pages``, appends or new lengths: the call writes no cache,
    so putting both back undoes it, and it can be made again once rows have ended.

    Can be captured in a graph.
    """
    lib = _native.library()
    tensors = (block_table, page_counts, parents, seqused_kv)
    names = ("block_table", "page_counts", "parents", "seqused_kv")
    check_operands(names, tensors)
    PAGE, reserve = index(PAGE), index(reserve)
    key = (lib, signature(*tensors), PAGE, reserve)
    call = _forks.get(key) or _forks.keep(key, _check_fork(lib, *tensors, PAGE, reserve))
    pointers = [t.data_ptr() for t in tensors]
    if not pointers_apart(pointers, call.sizes, (0, 1)):
        check_apart([(n, t, i < 2) for i, (n, t) in enumerate(zip(names, tensors))])
    device, B = block_table.device, block_table.shape[0]
    moves = torch.empty(2 * B + 1, dtype=torch.int32, device=device)
    # The caching allocator keeps the block for this stream.
    scratch = torch.empty(call.nbytes, dtype=torch.uint8, device=device)
    at = moves.data_ptr()
    status = launch_on(block_table.get_device(), call.launch, *pointers, at, at + 4 * B, at + 8 * B, scratch.data_ptr(),
                       call.nbytes, call.params)
    if status:
        _native.check(status, "launch_fork_pages")
    mark_written([block_table, page_counts])
    return moves[:B], moves[B:2 * B], moves[2 * B:]


def _check_compact(lib, block_table, page_counts):
    B, W, BLOCKS = _check_tables(block_table, page_counts)
    require(BLOCKS <= 1 << 28 and B * W < 1 << 31, "at most 2^28 pages and 2^31 - 1 entries of a table")
    params = _native.CompactPagesParams(B=B, W=W, BLOCKS=BLOCKS)
    nbytes = ct.c_uint64(0)
    _native.check(lib.workspace_size_compact_pages(ct.byref(nbytes), ct.byref(params)), "workspace_size_compact_pages")
    call = _Call()
    call.params, call.nbytes = ct.pointer(params), nbytes.value
    call.sizes = extents(block_table, page_counts)
    call.launch = lib.launch_compact_pages
    return call


def compact_pages(block_table, page_counts):
    """Renames pages so that those in use are the lowest; returns ``(source, destination)``, the pages to copy.

    With n pages in use (``page_counts`` above 0), the k-th of those from page n on
    becomes the k-th free page below n, in ``block_table`` int32 [B, W] and
    ``page_counts`` int32 [BLOCKS], both changed in place. ``source`` and
    ``destination`` int32 [BLOCKS / 2] list the moves in order, then -1:
    ``copy_pages(caches, source, destination)`` carries them out, after which pages
    n to BLOCKS - 1 of every cache are free. Whoever holds pages outside the table
    renames them by the same lists. Can be captured in a graph.
    """
    lib = _native.library()
    tensors = (block_table, page_counts)
    check_operands(("block_table", "page_counts"), tensors)
    key = (lib, signature(*tensors))
    call = _compactions.get(key) or _compactions.keep(key, _check_compact(lib, *tensors))
    pointers = [t.data_ptr() for t in tensors]
    if not pointers_apart(pointers, call.sizes, (0, 1)):
        check_apart([("block_table", block_table, True), ("page_counts", page_counts, True)])
    device, half = block_table.device, page_counts.shape[0] // 2
    moves = torch.empty(2 * half, dtype=torch.int32, device=device)
    scratch = torch.empty(call.nbytes, dtype=torch.uint8, device=device)
    at = moves.data_ptr()
    status = launch_on(block_table.get_device(), call.launch, *pointers, at, at + 4 * half, scratch.data_ptr(), call.nbytes,
                       call.params)
    if status:
        _native.check(status, "launch_compact_pages")
    mark_written([block_table, page_counts])
    return moves[:half], moves[half:]


@torch.library.custom_op("ascendflow_amd::copy_pages", mutates_args=("caches",))
def copy_pages_op(caches: list[torch.Tensor], source: torch.Tensor, destination: torch.Tensor) -> None:
    """Framework-facing form of ``copy_pages``, without its refusal of gradients: torch takes the pages as constants."""
    refuse_forward_mode("copy_pages")
    copy_pages([c.detach() for c in caches], source, destination)


@torch.library.custom_op("ascendflow_amd::fork_pages", mutates_args=("block_table", "page_counts"))
def fork_pages_op(
    block_table: torch.Tensor,
    page_counts: torch.Tensor,
    parents: torch.Tensor,
    seqused_kv: torch.Tensor,
    page: int,
    reserve: int = 0,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Framework-facing form of ``fork_pages``."""
    return tuple(t.clone() for t in fork_pages(block_table, page_counts, parents, seqused_kv, PAGE=page, reserve=reserve))


@fork_pages_op.register_fake
def _(block_table, page_counts, parents, seqused_kv, page, reserve=0):
    B = block_table.shape[0]
    return block_table.new_empty(B), block_table.new_empty(B), block_table.new_empty(1)


@torch.library.custom_op("ascendflow_amd::compact_pages", mutates_args=("block_table", "page_counts"))
def compact_pages_op(block_table: torch.Tensor, page_counts: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Framework-facing form of ``compact_pages``."""
    return tuple(t.clone() for t in compact_pages(block_table, page_counts))


@compact_pages_op.register_fake
def _(block_table, page_counts):
    half = page_counts.shape[0] // 2
    return block_table.new_empty(half), block_table.new_empty(half)
