"""Copies, forks and compaction of pages against their definitions: random tables and lengths, shared and foreign references,
too few free pages, sizes of pages, graphs and refusals."""

import random

import pytest
import torch

from ascendflow_amd.sparse_attention import compact_pages, copy_pages, fork_pages
from oracle import quantized_reference as qr

pytestmark = pytest.mark.gpu


def i32(device, x):
    return torch.tensor(x, dtype=torch.int32, device=device)


# ---- copies ----------------------------------------------------------------------


@pytest.mark.parametrize("shape,dtype", [
    ((3,), torch.uint8), ((5, 7), torch.bfloat16), ((2,), torch.float32), ((1, 2), torch.float32), ((16, 2, 128), torch.float8_e4m3fn),
    ((64, 8, 128), torch.int8), ((33, 1, 24), torch.float16), ((128, 1, 576), torch.bfloat16),
])
def test_copies(device, shape, dtype):
    gen = torch.Generator().manual_seed(1)
    blocks = 23
    cache = torch.randint(0, 100, (blocks, *shape), generator=gen).to(dtype).to(device)
    order = torch.randperm(blocks, generator=gen).tolist()
    source, destination = order[:9], order[9:18]
    source[3], destination[5], source[7], destination[7] = -1, blocks, 2**31 - 1, -(2**31)
    want = cache.clone()
    for s, d in zip(source, destination):
        if 0 <= s < blocks and 0 <= d < blocks:
            want.view(torch.uint8)[d] = cache.view(torch.uint8)[s]
    assert copy_pages(cache, i32(device, source), i32(device, destination)) is None
    assert torch.equal(cache.view(torch.uint8), want.view(torch.uint8))


@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 150])
def test_many_caches_at_once(device, n):
    gen = torch.Generator().manual_seed(2)
    shapes = [((16, 2, 64), torch.float8_e4m3fn), ((1, 2), torch.float32), ((3,), torch.uint8), ((700, 3), torch.int32)]
    caches = [torch.randint(0, 100, (6, *shapes[i % 4][0]), generator=gen).to(shapes[i % 4][1]).to(device) for i in range(n)]
    want = [c.clone() for c in caches]
    for c, w in zip(caches, want):
        w.view(torch.uint8)[5], w.view(torch.uint8)[0] = c.view(torch.uint8)[2], c.view(torch.uint8)[4]
    copy_pages(caches, i32(device, [2, 4]), i32(device, [5, 0]))
    assert all(torch.equal(c.view(torch.uint8), w.view(torch.uint8)) for c, w in zip(caches, want))
    assert all(c._version == 1 for c in caches)


def test_large_pages_and_far_ones(device):
    page = torch.arange(1 << 20, device=device, dtype=torch.int32)
    cache = torch.zeros((1100, 1 << 20), dtype=torch.int32, device=device)  # 4.6 GB
    cache[1] = page
    copy_pages(cache, i32(device, [1]), i32(device, [1099]))
    assert torch.equal(cache[1099], page) and not cache[1098].any() and not cache[2:10].any()


def test_caches_off_sixteen_bytes(device):
    flat = torch.arange(4 * 64 + 8, device=device, dtype=torch.uint8)
    for off in (1, 2, 4, 8):
        cache = flat.clone()[off:off + 256].view(4, 64)
        want = cache.clone()
        want[3] = want[1]
        copy_pages(cache, i32(device, [1]), i32(device, [3]))
        assert torch.equal(cache, want)


def test_a_page_onto_itself_and_no_pairs(device):
    cache = torch.arange(64, device=device).view(4, 16).clone()
    want = cache.clone()
    copy_pages(cache, i32(device, [2]), i32(device, [2]))
    copy_pages(cache, i32(device, []), i32(device, []))
    assert torch.equal(cache, want)


@pytest.mark.parametrize("change", [
    lambda c, s, d: ([], s, d), lambda c, s, d: ([c, c], s, d), lambda c, s, d: ([c, c[:3]], s, d), lambda c, s, d: (c[:, ::2], s, d),
    lambda c, s, d: (c.cpu(), s, d), lambda c, s, d: ([c, None], s, d), lambda c, s, d: (c, s.long(), d), lambda c, s, d: (c, s, d[:1]),
    lambda c, s, d: (c, s.cpu(), d), lambda c, s, d: (c[0], s, d), lambda c, s, d: (s.view(2, 1), s, d), lambda c, s, d: (c[:0], s, d),
    lambda c, s, d: (c.float().requires_grad_(True), s, d),
])
def test_copy_refusals(device, change):
    cache, s, d = torch.zeros((4, 16), dtype=torch.uint8, device=device), i32(device, [0, 1]), i32(device, [2, 3])
    with pytest.raises(ValueError):
        copy_pages(*change(cache, s, d))


def test_copy_op(device):
    caches = [torch.arange(4 * 16, device=device, dtype=torch.int32).view(4, 16).to(dt) for dt in (torch.int8, torch.float32)]
    want = [c.clone() for c in caches]
    for w in want:
        w[3] = w[1]
    leaf = caches[1].clone().requires_grad_(True)
    pairs = i32(device, [1, -1]), i32(device, [3, 0])
    torch.ops.ascendflow_amd.copy_pages(caches, *pairs)
    assert all(torch.equal(c, w) for c, w in zip(caches, want)) and all(c._version > 0 for c in caches)
    with torch.no_grad():
        torch.ops.ascendflow_amd.copy_pages([leaf], *pairs)
    assert torch.equal(leaf, want[1])


# ---- forks -----------------------------------------------------------------------


def case(rng, *, B, W, page, blocks, shared=0.5, extra=0.1):
    """A table whose rows share prefixes, references with some of somebody else's among them, parents and lengths."""
    table = [[-1] * W for _ in range(B)]
    lengths = [rng.randint(0, W * page) for _ in range(B)]
    pool = list(range(blocks))
    rng.shuffle(pool)
    for b in range(B):
        held = -(-lengths[b] // page)
        of = rng.randrange(b) if b and rng.random() < shared else None
        prefix = rng.randint(0, -(-lengths[of] // page)) if of is not None else 0
        for c in range(held):
            if of is not None and c < prefix and table[of][c] >= 0:
                table[b][c] = table[of][c]
            elif pool:
                table[b][c] = pool.pop()
    counts = [0] * blocks
    for row in table:
        for e in row:
            if e >= 0:
                counts[e] += 1
    for p in range(blocks):
        counts[p] += rng.random() < extra
    parents = [rng.choice([b, b, rng.randrange(B), -1]) for b in range(B)]
    used = [min(W * page, max(0, lengths[p] - rng.choice([0, 0, 0, 1, page]))) if p >= 0 else 0 for p in parents]
    return table, counts, parents, used


def check_fork(device, table, counts, parents, used, page, reserve):
    t, c = i32(device, table), i32(device, counts)
    want = qr.fork(table, counts, parents, used, page, reserve)
    source, destination, missing = fork_pages(t, c, i32(device, parents), i32(device, used), PAGE=page, reserve=reserve)
    got = (t.tolist(), c.tolist(), source.tolist(), destination.tolist(), missing.item())
    for name, g, w in zip(("table", "counts", "source", "destination", "missing"), got, want):
        assert g == w, name


@pytest.mark.parametrize("seed", range(12))
@pytest.mark.parametrize("B,W,page", [(1, 1, 16), (7, 5, 16), (40, 9, 64), (64, 300, 16)])
def test_forks(device, B, W, page, seed):
    rng = random.Random(seed * 100 + B)
    blocks = B * W + rng.choice([0, 5, B])
    check_fork(device, *case(rng, B=B, W=W, page=page, blocks=blocks), page, rng.choice([0, 1, page, 3 * page + 1]))


@pytest.mark.parametrize("seed", range(6))
def test_too_few_free_pages(device, seed):
    rng = random.Random(seed)
    check_fork(device, *case(rng, B=20, W=6, page=16, blocks=70, shared=0.8), 16, 40)


@pytest.mark.parametrize("B", [1023, 1025, 2500])
def test_many_rows(device, B):
    rng = random.Random(B)
    check_fork(device, *case(rng, B=B, W=3, page=16, blocks=4 * B), 16, 5)


def test_free_pages_at_the_far_end(device):
    table, blocks = [[0, 1, -1], [0, 1, -1]], 50000
    counts = [2, 2] + [1] * (blocks - 5) + [0, 0, 0]
    check_fork(device, table, counts, [0, 1], [20, 20], 16, 16)
    check_fork(device, table, counts, [0, 0], [32, 20], 16, 40)


def test_entries_and_lengths_that_make_no_sense(device):
    table = [[9, -5, 2**31 - 1], [3, 3, 3]]
    check_fork(device, table, [1, 0, 0, 3], [1, 0], [40, 2**31 - 1], 16, 0)
    check_fork(device, table, [1, 0, 0, 3], [2**31 - 1, -(2**31)], [-5, 3], 16, 0)
    check_fork(device, [[0]] * 40, [40], [0] * 40, [2**31 - 1] * 40, 16, 2**20)


def test_parents_swap_rows(device):
    table, counts = [[0, 1], [2, 3], [4, -1]], [1, 1, 1, 1, 1, 0, 0]
    check_fork(device, table, counts, [1, 0, 0], [30, 20, 17], 16, 2)


def test_forks_in_a_graph(device):
    rng = random.Random(5)
    table, counts, parents, used = case(rng, B=24, W=6, page=16, blocks=200)
    t, c, p, u = (i32(device, x) for x in (table, counts, parents, used))
    fork_pages(t, c, p, u, PAGE=16, reserve=4)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        moves = fork_pages(t, c, p, u, PAGE=16, reserve=4)
    for seed in range(3):
        state = case(random.Random(seed), B=24, W=6, page=16, blocks=200)
        for tensor, value in zip((t, c, p, u), state):
            tensor.copy_(i32(device, value))
        graph.replay()
        torch.cuda.synchronize()
        want = qr.fork(*state, 16, 4)
        assert [t.tolist(), c.tolist(), moves[0].tolist(), moves[1].tolist(), moves[2].item()] == list(want)


def test_fork_custom_op_and_versions(device):
    state = case(random.Random(7), B=24, W=6, page=16, blocks=200)
    t, c, p, u = (i32(device, x) for x in state)
    source, destination, missing = torch.ops.ascendflow_amd.fork_pages(t, c, p, u, 16, 4)
    assert [t.tolist(), c.tolist(), source.tolist(), destination.tolist(), missing.item()] == list(qr.fork(*state, 16, 4))
    before = t._version, c._version
    fork_pages(t, c, p, u, PAGE=16)
    assert t._version > before[0] and c._version > before[1] and p._version == 0


@pytest.mark.parametrize("change", [
    dict(PAGE=24), dict(PAGE=0), dict(reserve=-1), dict(reserve=2**20 + 1), dict(parents=lambda t: t["parents"].long()),
    dict(parents=lambda t: t["parents"][1:]), dict(seqused_kv=lambda t: t["seqused_kv"].cpu()), dict(seqused_kv=lambda t: None),
    dict(block_table=lambda t: t["block_table"][0]), dict(block_table=lambda t: t["block_table"][:, ::2]),
    dict(page_counts=lambda t: t["block_table"]), dict(page_counts=lambda t: t["page_counts"][:0]),
    dict(page_counts=lambda t: t["block_table"].view(-1)), dict(parents=lambda t: t["page_counts"][:3]),
    dict(block_table=lambda t: torch.zeros((8193, 1), dtype=torch.int32, device="cuda")),
])
def test_fork_refusals(device, change):
    t = dict(block_table=i32(device, [[0, 1], [2, 3], [4, -1]]), page_counts=i32(device, [1, 1, 1, 1, 1, 0]),
             parents=i32(device, [0, 1, 2]), seqused_kv=i32(device, [5, 6, 7]), PAGE=16, reserve=0)
    with pytest.raises(ValueError):
        changed = {k: v(t) if callable(v) else v for k, v in change.items()}
        a = {**t, **changed}
        fork_pages(a.pop("block_table"), a.pop("page_counts"), a.pop("parents"), a.pop("seqused_kv"), **a)


# ---- compaction --------------------------------------------------------------------


@pytest.mark.parametrize("blocks", [1, 2, 3, 50, 4095, 4096, 4097, 9000, 70001])
@pytest.mark.parametrize("full", [0.0, 0.3, 0.9, 1.0])
def test_compaction(device, blocks, full):
    rng = random.Random(blocks)
    counts = [rng.randint(1, 3) if rng.random() < full else 0 for _ in range(blocks)]
    used = [p for p in range(blocks) if counts[p]]
    table = [[rng.choice(used) if used and rng.random() < 0.8 else rng.choice([-1, blocks, 2**31 - 1]) for _ in range(17)] for _ in range(9)]
    t, c = i32(device, table), i32(device, counts)
    want_table, want_counts, moves = qr.compact(table, counts)
    source, destination = compact_pages(t, c)
    assert t.tolist() == want_table and c.tolist() == want_counts
    half = blocks // 2
    assert source.tolist() == [a for a, _ in moves] + [-1] * (half - len(moves))
    assert destination.tolist() == [b for _, b in moves] + [-1] * (half - len(moves))


def test_compaction_keeps_what_rows_hold(device):
    gen = torch.Generator(device=device).manual_seed(0)
    cache = torch.randn((100, 16, 2, 8), generator=gen, device=device)
    table = torch.randperm(100, generator=gen, device=device)[:40].view(8, 5).to(torch.int32)
    counts = torch.zeros(100, dtype=torch.int32, device=device)
    counts[table.flatten().long()] = 1
    before = cache[table.long()].clone()
    copy_pages(cache, *compact_pages(table, counts))
    assert torch.equal(cache[table.long()], before) and table.max() == 39 and counts[:40].all() and not counts[40:].any()


def test_compaction_in_a_graph_and_as_custom_op(device):
    t, c = i32(device, [[0, 1]]), i32(device, [1, 1, 0, 0, 0, 0, 0, 0])
    compact_pages(t, c)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        moves = compact_pages(t, c)
    for table, counts in (([[7, 2]], [0, 0, 1, 0, 0, 0, 0, 1]), ([[5, -1]], [0, 0, 0, 1, 1, 1, 0, 0]), ([[0, 1]], [1] * 8)):
        t.copy_(i32(device, table))
        c.copy_(i32(device, counts))
        graph.replay()
        torch.cuda.synchronize()
        want_table, want_counts, want = qr.compact(table, counts)
        assert t.tolist() == want_table and c.tolist() == want_counts
        assert [m for m in zip(moves[0].tolist(), moves[1].tolist()) if m[0] >= 0] == want
        a, b = i32(device, table), i32(device, counts)
        source, _ = torch.ops.ascendflow_amd.compact_pages(a, b)
        assert torch.equal(a, t) and torch.equal(b, c) and torch.equal(source, moves[0])


@pytest.mark.parametrize("change", [
    lambda t, c: (t.long(), c), lambda t, c: (t[0], c), lambda t, c: (t, c.float()), lambda t, c: (t, c.cpu()),
    lambda t, c: (t, t.view(-1)), lambda t, c: (t[:0], c), lambda t, c: (t, None),
])
def test_compaction_refusals(device, change):
    with pytest.raises(ValueError):
        compact_pages(*change(i32(device, [[0, 1]]), i32(device, [1, 1, 0])))
