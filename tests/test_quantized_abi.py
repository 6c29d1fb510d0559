"""CPU checks of the 8-bit paged cache's C ABI and entries: rejections before any launch, workspace sizes, forms, and
operands that are no tensors or no GPU's."""

import ctypes as ct
import math

import pytest
import torch

from ascendflow_amd import _native
from ascendflow_amd.flash_attention import quantized_attention
from ascendflow_amd.sparse_attention import append_quantized_kv, compact_pages, copy_pages, fork_pages

P = ct.c_void_p
p16 = P(16)


@pytest.fixture(scope="module")
def lib():
    return _native.library()


def append(**changes):
    fields = dict(dtype=0, code=0, T=3, B=2, W=4, PAGE=32, GROUP=16, BLOCKS=8, HKV=2, D=64, k_stride_t=128, k_stride_h=64,
                  v_stride_t=128, v_stride_h=64)
    return _native.AppendQuantizedKvParams(**{**fields, **changes})


def attention(**changes):
    fields = dict(dtype=0, code=0, causal=1, T=3, B=2, HQ=8, HKV=2, D=128, PAGE=32, GROUP=16, W=4, BLOCKS=8,
                  q_stride_t=8 * 128, q_stride_h=128, out_stride_t=8 * 128, out_stride_h=128, scale=0.07)
    return _native.QuantizedParams(**{**fields, **changes})


@pytest.mark.parametrize("changes,status", [
    ({"dtype": 2}, -3), ({"code": 2}, -3), ({"code": -1}, -3), ({"T": -1}, -2), ({"T": 1 << 23}, -2), ({"B": 0}, -2), ({"W": 0}, -2),
    ({"BLOCKS": 0}, -2), ({"HKV": 0}, -2), ({"HKV": 32769}, -2), ({"D": 0}, -2), ({"D": 1025}, -2), ({"GROUP": 8}, -2),
    ({"GROUP": 24}, -2), ({"GROUP": 64}, -2), ({"PAGE": 48}, -2), ({"GROUP": 2048, "PAGE": 2048}, -2), ({"PAGE": 0}, -2), ({"T": 0}, 0),
    ({"W": (1 << 25) + 1}, -2), ({"W": 1 << 25, "T": 0}, 0),
])
def test_append_rejections(lib, changes, status):
    assert lib.launch_append_quantized_kv(None, *[p16] * 9, ct.byref(append(**changes))) == status
    assert lib.launch_append_quantized_kv(None, *[p16] * 9, None) == -1


@pytest.mark.parametrize("missing", range(9))
def test_append_pointers(lib, missing):
    assert lib.launch_append_quantized_kv(None, *[None if i == missing else p16 for i in range(9)], ct.byref(append())) == -1


@pytest.mark.parametrize("changes,status", [
    ({"dtype": 2}, -3), ({"code": 3}, -3), ({"T": -1}, -2), ({"B": 0}, -2), ({"HQ": 0}, -2), ({"HKV": 0}, -2), ({"HQ": 7}, -2),
    ({"D": 96}, -2), ({"D": 512}, -2), ({"PAGE": 8}, -2), ({"PAGE": 48}, -2), ({"GROUP": 64}, -2), ({"GROUP": 8}, -2), ({"GROUP": 0}, -2),
    ({"W": 0}, -2), ({"BLOCKS": 0}, -2), ({"W": (1 << 25) + 1}, -2), ({"T": 1 << 29}, -2), ({"HKV": 65536, "HQ": 65536}, -2),
    ({"scale": 0.0}, -2), ({"scale": -1.0}, -2), ({"scale": math.nan}, -2), ({"scale": math.inf}, -2),
])
def test_attention_rejections(lib, changes, status):
    size, form = ct.c_uint64(), (ct.c_int64 * 4)()
    params = ct.byref(attention(**changes))
    assert lib.launch_quantized_attention(None, *[p16] * 11, 1 << 30, params) == status
    assert lib.workspace_size_quantized_attention(ct.byref(size), params) == status
    assert lib.form_quantized_attention(form, params) == status


def test_attention_pointers_strides_and_workspace(lib):
    size, form = ct.c_uint64(), (ct.c_int64 * 4)()
    params = ct.byref(attention())
    launch = lambda pointers, workspace, nbytes, p=params: lib.launch_quantized_attention(None, *pointers, workspace, nbytes, p)
    pointers = [p16] * 9 + [None]
    for i in range(9):
        assert launch([None if j == i else x for j, x in enumerate(pointers)], p16, 1 << 30) == -1
    assert launch(pointers, p16, 1 << 30, None) == -1
    for i in (0, 1, 2, 8):  # q, caches and out on 16 bytes
        assert launch([P(24) if j == i else x for j, x in enumerate(pointers)], p16, 1 << 30) == -2
    for name in ("q_stride_t", "q_stride_h", "out_stride_t", "out_stride_h"):
        assert launch(pointers, p16, 1 << 30, ct.byref(attention(**{name: 100}))) == -2
    assert lib.workspace_size_quantized_attention(ct.byref(size), params) == 0 and size.value > 0
    assert launch(pointers, None, size.value) == -4 and launch(pointers, p16, size.value - 1) == -4
    assert launch(pointers, P(8), size.value) == -4
    assert launch(pointers, None, 0, ct.byref(attention(T=0))) == 0
    assert lib.workspace_size_quantized_attention(None, params) == -1 and lib.form_quantized_attention(None, params) == -1
    assert lib.form_quantized_attention(form, params) == 0 and list(form) == [16, 1, 256, 0]


@pytest.mark.parametrize("changes,form", [
    (dict(T=64, B=64, HQ=64, HKV=8, W=256, PAGE=64, BLOCKS=16384), [16, 4, 256, 1]),   # 64 requests of 16K
    (dict(T=64, B=64, HQ=64, HKV=8, W=256, PAGE=64, BLOCKS=500), [16, 4, 256, 0]),     # 65 MB of cache
    (dict(T=64, B=64, HQ=64, HKV=8, D=64, W=256, PAGE=64, BLOCKS=16384), [16, 4, 256, 0]),
    (dict(T=64, B=64, HQ=64, HKV=8, D=256, W=256, PAGE=64, BLOCKS=16384), [16, 4, 128, 1]),
    (dict(T=192, B=48, HQ=32, HKV=4, D=64), [32, 4, 512, 0]),
    (dict(T=1, B=1, HQ=32, HKV=8), [16, 1, 64, 0]),
    (dict(T=2000, B=1, HQ=32, HKV=8, PAGE=128, W=157, BLOCKS=157), [256, 1, 32, 0]),
    (dict(T=2000, B=1, HQ=32, HKV=8, PAGE=128, W=11, BLOCKS=157), [32, 4, 256, 0]),    # no room for 1536 rows
    (dict(T=2000, B=1, HQ=32, HKV=8, D=256, PAGE=128, W=157, BLOCKS=157), [128, 1, 32, 0]),
    (dict(T=64, B=1, HQ=32, HKV=8, PAGE=128, W=157, BLOCKS=157), [32, 1, 64, 0]),
    (dict(T=5, B=5, HQ=2000, HKV=2000, W=157), [16, 4, 1, 0]),
])
def test_forms(lib, changes, form):
    got = (ct.c_int64 * 4)()
    assert lib.form_quantized_attention(got, ct.byref(attention(**changes))) == 0 and list(got) == form


def test_copy_rejections(lib):
    one, bytes_ = (P * 1)(16), (ct.c_uint64 * 1)(64)
    call = lambda caches=one, page=bytes_, n=1, s=p16, d=p16, pairs=2, blocks=4: lib.launch_copy_pages(None, caches, page, n, s, d, pairs, blocks)
    assert call(n=-1) == call(pairs=-1) == call(blocks=0) == call(page=(ct.c_uint64 * 1)(0)) == -2
    assert call(page=(ct.c_uint64 * 1)(1 << 40)) == -2 and call(page=(ct.c_uint64 * 1)(1 << 36), pairs=1 << 24) == -2
    assert call(caches=None) == call(page=None) == call(s=None) == call(d=None) == call(caches=(P * 1)(None)) == -1
    assert call(n=0) == call(pairs=0) == 0


def test_pages_and_pairs_past_32_bits_are_refused():
    many, few, number = torch.empty(1 << 32, 1, dtype=torch.int8), torch.empty(2, 1, dtype=torch.int8), torch.zeros(1, dtype=torch.int32)
    for operands in ((many, number, number), (few, number.expand(1 << 31), number)):
        with pytest.raises(ValueError, match="at most 2\\^31 - 1 pages"):
            copy_pages(*operands)


@pytest.mark.parametrize("changes,status", [
    ({"B": 0}, -2), ({"B": 8193}, -2), ({"W": 0}, -2), ({"W": 1 << 25}, -2), ({"PAGE": 0}, -2), ({"PAGE": 24}, -2), ({"BLOCKS": 0}, -2),
    ({"reserve": -1}, -2), ({"BLOCKS": (1 << 28) + 1}, -2),
])
def test_fork_rejections(lib, changes, status):
    params = ct.byref(_native.ForkPagesParams(**{**dict(B=2, W=4, PAGE=16, BLOCKS=9, reserve=1), **changes}))
    size = ct.c_uint64()
    assert lib.workspace_size_fork_pages(ct.byref(size), params) == status
    assert lib.launch_fork_pages(None, *[p16] * 8, 1 << 30, params) == status


def test_fork_and_compact_pointers(lib):
    params, size = ct.byref(_native.ForkPagesParams(B=2, W=4, PAGE=16, BLOCKS=9, reserve=1)), ct.c_uint64()
    assert lib.workspace_size_fork_pages(ct.byref(size), params) == 0 and size.value >= 4 * (8 + 9)
    for i in range(7):
        assert lib.launch_fork_pages(None, *[None if j == i else p16 for j in range(8)], size.value, params) == -1
    assert lib.launch_fork_pages(None, *[p16] * 7, None, size.value, params) == -4
    assert lib.launch_fork_pages(None, *[p16] * 8, size.value - 1, params) == -4
    assert lib.launch_fork_pages(None, *[p16] * 8, size.value, None) == -1
    params = ct.byref(_native.CompactPagesParams(B=2, W=4, BLOCKS=9))
    assert lib.workspace_size_compact_pages(ct.byref(size), params) == 0 and size.value >= 4 * 9
    for i in range(4):
        assert lib.launch_compact_pages(None, *[None if j == i else p16 for j in range(5)], size.value, params) == -1
    assert lib.launch_compact_pages(None, *[p16] * 4, None, size.value, params) == -4
    assert lib.launch_compact_pages(None, *[p16] * 5, size.value - 1, params) == -4
    for changes in (dict(B=0), dict(W=0), dict(BLOCKS=0), dict(BLOCKS=1 << 29)):
        bad = ct.byref(_native.CompactPagesParams(**{**dict(B=2, W=4, BLOCKS=9), **changes}))
        assert lib.launch_compact_pages(None, *[p16] * 5, 1 << 30, bad) == -2


def cpu_tensors():
    i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32)
    cache, scale = torch.zeros((4, 32, 2, 64), dtype=torch.int8), torch.ones((4, 2, 2))
    rows = torch.zeros((3, 2, 64), dtype=torch.bfloat16)
    return dict(k=rows, v=rows.clone(), q=torch.zeros((3, 8, 64), dtype=torch.bfloat16), k_cache=cache, v_cache=cache.clone(), k_scale=scale,
                v_scale=scale.clone(), block_table=i32(1, 2), cu_seqlens_q=i32(2), seqused_kv=i32(1), parents=i32(1), page_counts=i32(4),
                source=i32(2), destination=i32(2))


CALLS = {
    "append": (lambda t: append_quantized_kv(*[t[n] for n in APPEND]), APPEND := (
        "k", "v", "k_cache", "v_cache", "k_scale", "v_scale", "block_table", "cu_seqlens_q", "seqused_kv")),
    "attention": (lambda t: quantized_attention(*[t[n] for n in ATTENTION], SCALE=0.1), ATTENTION := (
        "q", "k_cache", "v_cache", "k_scale", "v_scale", "block_table", "cu_seqlens_q", "seqused_kv")),
    "fork": (lambda t: fork_pages(*[t[n] for n in FORK], PAGE=16), FORK := ("block_table", "page_counts", "parents", "seqused_kv")),
    "compact": (lambda t: compact_pages(t["block_table"], t["page_counts"]), ("block_table", "page_counts")),
    "copy": (lambda t: copy_pages([t["k_cache"]], t["source"], t["destination"]), ("source", "destination")),
}


@pytest.mark.parametrize("call,name", [(c, n) for c, (_, names) in CALLS.items() for n in names])
def test_operands_that_are_no_tensors_are_refused_by_name(call, name):
    for value in (None, 3, [1.0]):
        with pytest.raises(ValueError, match=f"{name} must be a torch.Tensor"):
            CALLS[call][0]({**cpu_tensors(), name: value})


@pytest.mark.parametrize("call", CALLS)
def test_operands_off_the_gpu_are_refused(call):
    with pytest.raises(ValueError, match="ROCm"):
        CALLS[call][0](cpu_tensors())


def test_counts_that_are_no_integers_are_refused():
    t = cpu_tensors()
    for kw in (dict(PAGE=16.0), dict(PAGE=16, reserve=1.5), dict(PAGE="16")):
        with pytest.raises(TypeError):
            fork_pages(t["block_table"], t["page_counts"], t["parents"], t["seqused_kv"], **kw)
