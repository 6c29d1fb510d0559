"""Copies of long lists of pairs over many caches: a call that is refused has copied nothing, and every list that a compaction
returns is taken."""

import pytest
import torch

from ascendflow_amd.sparse_attention import compact_pages, copy_pages

pytestmark = pytest.mark.gpu


def test_a_refused_call_copies_nothing(device):
    """More caches than a launch takes, of which the last has pages too large for so many pairs."""
    caches = [torch.tensor([[1], [2]], dtype=torch.uint8, device=device) for _ in range(64)]
    caches.append(torch.zeros((2, 5 << 20), dtype=torch.uint8, device=device))
    source = torch.full(((1 << 24) - 1,), -1, dtype=torch.int32, device=device)
    destination = source.clone()
    source[0], destination[0] = 0, 1
    with pytest.raises(ValueError):
        copy_pages(caches, source, destination)
    assert all(c.tolist() == [[1], [2]] for c in caches[:64]) and all(c._version == 0 for c in caches)


@pytest.mark.parametrize("page", [1, 16])
def test_lists_of_a_compaction_of_many_pages(device, page):
    """2^25 pages and more: the list has half as many entries, which no single launch counts the threads of."""
    blocks = (1 << 25) + 6
    cache = torch.zeros((blocks, page), dtype=torch.uint8, device=device)
    table = torch.tensor([[blocks - 1, 3, blocks - 2]], dtype=torch.int32, device=device)
    counts = torch.zeros(blocks, dtype=torch.int32, device=device)
    counts[table[0].long()] = 1
    cache[table[0].long()] = torch.tensor([[7], [8], [9]], dtype=torch.uint8, device=device)
    source, destination = compact_pages(table, counts)
    assert source.shape[0] == blocks // 2 > (1 << 24) and table.max() == 2
    copy_pages(cache, source, destination)
    assert cache[table[0].long()].tolist() == [[x] * page for x in (7, 8, 9)]


@pytest.mark.parametrize("n", [1, 70])
def test_pairs_of_several_launches(device, n):
    """Pairs at both ends of each launch's range and at the list's: pages of 64 parts, 2^18 pairs and a few a launch."""
    page, blocks, pairs = 64 * 16384, 16, 5 << 17
    gen = torch.Generator(device=device).manual_seed(3)
    caches = [torch.randint(0, 255, (blocks, page) if i == n - 1 else (blocks, 3), generator=gen, device=device, dtype=torch.uint8) for i in range(n)]
    want = [c.clone() for c in caches]
    each = ((1 << 24) - 1) // 64
    source = torch.full((pairs,), -1, dtype=torch.int32, device=device)
    destination = source.clone()
    for k, at in enumerate((0, each - 1, each, 2 * each - 1, 2 * each, pairs - 1)):
        source[at], destination[at] = k, 15 - k
        for w in want:
            w[15 - k] = w[k]
    copy_pages(caches, source, destination)
    assert all(torch.equal(c, w) for c, w in zip(caches, want)) and all(c._version == 1 for c in caches)
