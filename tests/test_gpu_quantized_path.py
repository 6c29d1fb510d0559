"""The operators of the 8-bit paged cache together, as a decode loop with several samples a prompt uses them: prompts
appended, forked, steps of append and attention, forks again, rows that end, a compaction; against the same sequences each on
pages of its own, bit for bit, and against float64. And one whole step captured in a graph."""

import pytest
import torch

from ascendflow_amd.flash_attention import quantized_attention
from ascendflow_amd.sparse_attention import append_quantized_kv, compact_pages, copy_pages, fork_pages
from oracle import quantized_reference as qr

pytestmark = pytest.mark.gpu
HQ, HKV, D, PAGE, GROUP, SCALE = 8, 2, 64, 16, 16, 64 ** -0.5


class Cache:
    def __init__(self, device, rows, width, blocks, codes):
        self.device = device
        self.caches = [torch.zeros((blocks, PAGE, HKV, D), dtype=codes, device=device) for _ in range(2)]
        self.scales = [torch.zeros((blocks, PAGE // GROUP, HKV), device=device) for _ in range(2)]
        self.table = torch.full((rows, width), -1, dtype=torch.int32, device=device)
        self.counts = torch.zeros(blocks, dtype=torch.int32, device=device)

    def fork(self, parents, lengths, reserve):
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=self.device)
        source, destination, missing = fork_pages(self.table, self.counts, i32(parents), i32(lengths), PAGE=PAGE, reserve=reserve)
        assert missing.item() == 0
        copy_pages(self.caches + self.scales, source, destination)

    def step(self, k, v, q, counts, lengths):
        """Appends counts[b] tokens to row b, which then has lengths[b], and attends them."""
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=self.device)
        cu, used = i32([sum(counts[:i]) for i in range(len(counts) + 1)]), i32(lengths)
        append_quantized_kv(k, v, *self.caches, *self.scales, self.table, cu, used)
        return quantized_attention(q, *self.caches, *self.scales, self.table, cu, used, SCALE=SCALE)

    def rows(self, b, length):
        ids = self.table[b, :-(-length // PAGE)].long()
        return [qr.values(c[ids].cpu(), s[ids].cpu()).flatten(0, 1)[:length] for c, s in zip(self.caches, self.scales)]


@pytest.mark.parametrize("codes", [torch.float8_e4m3fn, torch.int8])
def test_samples_of_prompts(device, codes):
    gen = torch.Generator(device=device).manual_seed(4)
    normal = lambda *shape: (torch.randn(shape, generator=gen, device=device) * torch.exp(torch.randn((*shape[:2], 1), generator=gen, device=device))).bfloat16()
    rows, width = 6, 8
    shared, own = Cache(device, rows, width, 40, codes), Cache(device, rows, width, rows * width, codes)
    own.table.copy_(torch.arange(rows * width, device=device).view(rows, width))
    # Two prompts, in rows 0 and 3; rows 1, 2 continue the first, 4, 5 the second.
    lengths = [37, 0, 0, 50, 0, 0]
    k, v, q = normal(87, HKV, D), normal(87, HKV, D), normal(87, HQ, D)
    shared.fork([0, -1, -1, 3, -1, -1], [0] * 6, 64)
    first = shared.step(k, v, q, lengths, lengths)
    parts = lambda x: torch.cat([x[:37]] * 3 + [x[37:]] * 3)
    all_lengths = [37] * 3 + [50] * 3
    own.step(parts(k), parts(v), parts(q), all_lengths, all_lengths)
    shared.fork([0, 0, 0, 3, 3, 3], all_lengths, 1)
    assert (shared.counts > 0).sum() < (own.table >= 0).sum()
    lengths, history = all_lengths, [[(k[:37], v[:37])] for _ in range(3)] + [[(k[37:], v[37:])] for _ in range(3)]
    for step in range(20):
        k, v, q = normal(6, HKV, D), normal(6, HKV, D), normal(6, HQ, D)
        lengths = [n + 1 for n in lengths]
        out = shared.step(k, v, q, [1] * 6, lengths)
        assert torch.equal(out, own.step(k, v, q, [1] * 6, lengths)), step
        for b in range(6):
            history[b].append((k[b:b + 1], v[b:b + 1]))
            for mine, theirs in zip(shared.rows(b, lengths[b]), own.rows(b, lengths[b])):
                assert torch.equal(mine, theirs)
        parents = list(range(6))
        if step % 7 == 3:  # the middle samples win
            parents = [1, 1, 2, 4, 4, 4]
        shared.fork(parents, [lengths[p] for p in parents], 1)
        for x in own.caches + own.scales:
            ids = own.table.long()
            x[ids] = x[ids[torch.tensor(parents, device=device)]]
        lengths, history = [lengths[p] for p in parents], [list(history[p]) for p in parents]
        if step == 12:
            source, destination = compact_pages(shared.table, shared.counts)
            copy_pages(shared.caches + shared.scales, source, destination)
            n = int((shared.counts > 0).sum())
            assert (shared.counts[:n] > 0).all() and not shared.counts[n:].any()
    # The cache stands for what was appended, to a rounding of each block's scale: e4m3 half a step of 2^-4 of the value (or
    # of the smallest normal code), int8 half a step of the scale, at most 2 / 127 of the block's largest; twice, where a
    # block was rounded anew.
    for b in range(6):
        for i, got in enumerate(shared.rows(b, lengths[b])):
            want = torch.cat([h[i] for h in history[b]]).double().cpu()
            for at in range(0, lengths[b], GROUP):
                w, g = want[at:at + GROUP], got[at:at + GROUP]
                largest = w.abs().amax(dim=(0, 2), keepdim=True)
                bound = 2 * (w.abs() * 2 ** -4 + largest * 2 ** -9) if codes == torch.float8_e4m3fn else largest * 2 / 127
                assert ((w - g).abs() <= bound).all()
    # Ending every row frees every page.
    shared.fork([-1] * 6, [0] * 6, 5)
    assert not shared.counts.any() and (shared.table == -1).all()
    assert torch.isfinite(first.float()).all()


def test_a_step_in_a_graph(device):
    """Fork, copy, append and attention of one step captured once and replayed, lengths counted on the device."""
    gen = torch.Generator(device=device).manual_seed(6)
    normal = lambda *shape: torch.randn(shape, generator=gen, device=device).bfloat16()
    graphed, eager = (Cache(device, 4, 6, 24, torch.float8_e4m3fn) for _ in range(2))
    k, v, q = normal(4, HKV, D), normal(4, HKV, D), normal(4, HQ, D)
    cu = torch.arange(5, dtype=torch.int32, device=device)
    state = {}
    for name, cache in (("graph", graphed), ("eager", eager)):
        state[name] = dict(parents=torch.arange(4, dtype=torch.int32, device=device),
                           used=torch.zeros(4, dtype=torch.int32, device=device))

    def one(cache, s):
        source, destination, missing = fork_pages(cache.table, cache.counts, s["parents"], s["used"], PAGE=PAGE, reserve=1)
        copy_pages(cache.caches + cache.scales, source, destination)
        s["used"] += 1
        append_quantized_kv(k, v, *cache.caches, *cache.scales, cache.table, cu, s["used"])
        return quantized_attention(q, *cache.caches, *cache.scales, cache.table, cu, s["used"], SCALE=SCALE), missing

    one(graphed, state["graph"])
    one(eager, state["eager"])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, missing = one(graphed, state["graph"])
    for step in range(40):
        for x in (k, v, q):
            x.copy_(normal(*x.shape))
        if step % 9 == 5:
            for s in state.values():
                s["parents"].copy_(torch.tensor([2, 1, 2, 2], dtype=torch.int32, device=device))
        graph.replay()
        want, lacks = one(eager, state["eager"])
        torch.cuda.synchronize()
        assert torch.equal(out, want) and missing.item() == lacks.item() == 0, step
        assert torch.equal(graphed.table, eager.table) and torch.equal(graphed.counts, eager.counts)
        for s in state.values():
            s["parents"].copy_(torch.arange(4, dtype=torch.int32, device=device))
