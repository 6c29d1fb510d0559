"""Append of the widest rows and the most heads that are documented, on 16-byte groups and off them: the same bits."""

import ctypes as ct

import pytest
import torch

from ascendflow_amd import _native
from ascendflow_amd.sparse_attention import append_paged_kv, rotary_frequencies

pytestmark = pytest.mark.gpu


def odd(x):
    """The same rows at an odd address and an odd token stride."""
    T, H, D = x.shape
    flat = torch.zeros((T, H * D + 1), dtype=x.dtype, device=x.device)
    view = flat[:, 1:].unflatten(1, (H, D))
    view.copy_(x)
    return view


@pytest.mark.parametrize("T,HKV,DK,DV,R", [
    (3, 1, 16384, 16384, 0), (3, 8, 16384, 16384, 64), (40, 3, 16384, 16384, 1024), (2100, 1, 16384, 16384, 64), (9, 8, 8192, 8192, 1024),
    (5, 32768, 8, 8, 0), (2, 32768, 64, 64, 64), (3000, 700, 16, 16, 16),
])
def test_wide_rows(device, T, HKV, DK, DV, R):
    gen = torch.Generator(device=device).manual_seed(T)
    normal = lambda *shape: torch.randn(shape, generator=gen, device=device).bfloat16()
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=device)
    page, blocks = 16, (T + 5) // 16 + 2
    table, cu, used = torch.arange(blocks, dtype=torch.int32, device=device).flip(0)[None].contiguous(), i32(0, T), i32(T + 5)
    k, v = normal(T, HKV, DK), normal(T, HKV, DV)
    frequencies = rotary_frequencies(R, device=device) if R else None
    results = []
    for keys, values in ((k, v), (odd(k), odd(v))):
        caches = [torch.zeros((blocks, page, HKV, D), dtype=torch.bfloat16, device=device) for D in (DK, DV)]
        append_paged_kv(keys, caches[0], table, cu, used, values, caches[1], frequencies=frequencies, layout="interleaved")
        results.append(caches)
    for aligned, other in zip(*results):
        assert torch.equal(aligned, other)
    at = torch.arange(5, T + 5, device=device)
    rows = lambda cache: cache[table[0].long()[at // page], at % page]
    assert torch.equal(rows(results[0][1]), v) and torch.equal(rows(results[0][0])[..., R:], k[..., R:])
    for cache in results[0]:
        assert cache.flatten(2).any(-1).sum() == T  # no other row


def test_more_heads_are_refused(device):
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=device)
    rows, cache = (torch.zeros(shape, dtype=torch.bfloat16, device=device) for shape in ((1, 32769, 2), (1, 1, 32769, 2)))
    with pytest.raises(ValueError, match="32768"):
        append_paged_kv(rows, cache, i32(0)[None], i32(0, 1), i32(1))
    p = ct.c_void_p(16)
    params = _native.AppendPagedKvParams(T=1, B=1, W=1, PAGE=1, BLOCKS=1, HKV=32769, DK=2, magnitude=1.0)
    assert _native.library().launch_append_paged_kv(None, p, None, None, p, p, p, None, p, None, ct.byref(params)) == -2
