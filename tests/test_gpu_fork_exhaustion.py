"""What a fork leaves where pages run out, and how a caller gets back."""

import pytest
import torch

from ascendflow_amd.sparse_attention import copy_pages, fork_pages

pytestmark = pytest.mark.gpu


def i32(device, x):
    return torch.tensor(x, dtype=torch.int32, device=device)


def test_a_page_that_could_not_be_copied(device):
    """Three rows on two pages of 16, 20 tokens each, and one free page: the lowest row keeps the last page, the second gets
    the free one, the third loses its tokens 16 to 19. The next call wants none of that again."""
    table, counts = i32(device, [[0, 1, -1]] * 3), i32(device, [3, 3, 0])
    used = i32(device, [20] * 3)
    source, destination, missing = fork_pages(table, counts, i32(device, [0, 1, 2]), used, PAGE=16)
    assert table.tolist() == [[0, 1, -1], [0, 2, -1], [0, -1, -1]] and counts.tolist() == [3, 1, 1]
    assert source.tolist() == [-1, 1, -1] and destination.tolist() == [-1, 2, -1] and missing.item() == 1
    *_, missing = fork_pages(table, counts, i32(device, [0, 1, 2]), used, PAGE=16, reserve=1)
    assert table.tolist() == [[0, 1, -1], [0, 2, -1], [0, -1, -1]] and missing.item() == 0


def test_tables_saved_before_the_call_undo_it(device):
    gen = torch.Generator(device=device).manual_seed(1)
    cache = torch.randn((3, 16, 2, 8), generator=gen, device=device)
    table, counts, used = i32(device, [[0, 1, -1]] * 3), i32(device, [3, 3, 0]), i32(device, [20] * 3)
    saved, before = (table.clone(), counts.clone()), cache.clone()
    *_, missing = fork_pages(table, counts, i32(device, [0, 1, 2]), used, PAGE=16)
    assert missing.item() == 1 and torch.equal(cache, before)
    table.copy_(saved[0])
    counts.copy_(saved[1])
    # The last row ends instead; the others go on with all of their tokens.
    source, destination, missing = fork_pages(table, counts, i32(device, [0, 1, -1]), i32(device, [20, 20, 0]), PAGE=16)
    copy_pages(cache, source, destination)
    assert missing.item() == 0 and table.tolist() == [[0, 1, -1], [0, 2, -1], [-1, -1, -1]] and counts.tolist() == [2, 1, 1]
    rows = cache[table[:2, :2].long()].flatten(1, 2)[:, :20]
    assert torch.equal(rows, before[:2].flatten(0, 1)[:20].expand_as(rows))
