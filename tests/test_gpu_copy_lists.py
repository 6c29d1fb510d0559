"""Copies of long lists of pairs over many caches: a call that is refused has copied nothing, and every list that a compaction
returns is taken."""

import pytest
import torch

from ascendflow_amd.sparse_attention import copy_pages

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
