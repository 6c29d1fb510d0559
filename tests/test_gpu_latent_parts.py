"""A request in as many parts as workgroups, none of which can go missing unnoticed."""

import pytest
import torch

from oracle import latent_reference as lr
from tests.latent_helpers import compare, paged
from tests.test_gpu_latent_forms import form_of
from tests.test_gpu_latent_shares import run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("H,keys,workers", [(16, 32, 512), (100, 64, 256)])
def test_every_part_of_a_long_request_matters(device, H, keys, workers):
    """Head h attends the parts h, h + H, ... alone, each with values of its own: a part left out, or another one in its
    place, takes a column of that head beyond its bound, which is asserted before the kernel runs."""
    length, L = 70000, 128
    t = paged(device, [1], [length], H=H, L=L, R=0, page=128)
    assert form_of(t) == [16 * keys // 8, workers]
    # Keys of each part: chunks and the weight of the tile's start, shared evenly.
    chunks, start = -(-length // keys), 64 // keys
    cuts = [max(0, (chunks + start) * w // workers - start) for w in range(workers + 1)]
    part = torch.repeat_interleave(torch.arange(workers), torch.tensor(cuts).diff() * keys)[:length].to(device)
    assert part.numel() == length and part.unique().numel() == workers
    gen = torch.Generator(device=device).manual_seed(H)
    rows = torch.zeros((length, L), device=device)
    rows[torch.arange(length, device=device), part % H] = 1
    own = torch.randn((workers, L - H), generator=gen, device=device)
    rows[:, H:] = own[part] + 0.1 * torch.randn((length, L - H), generator=gen, device=device)
    rows = rows.bfloat16()
    table = t["block_table"][0].long()
    at = torch.arange(length, device=device)
    t["kv_cache"][table[at // 128], at % 128, 0] = rows
    t["q"].zero_()
    t["q"][0, :, :H] = 12 * torch.eye(H, device=device).bfloat16()

    expected = lr.latent_attention(t["q"], None, t["kv_cache"], t["block_table"].cpu(), t["cu_seqlens_q"].cpu(),
                                   t["seqused_kv"].cpu(), 1.0)
    want, want_lse, spread, reach = expected
    bound = lr.attention_bound(want, spread, reach, torch.bfloat16, length, rows.abs().max().item())[0]
    weight = (torch.matmul(t["q"][0].double(), rows.double().t()) - want_lse[0, :, None]).exp()  # [H, length]
    shares = torch.stack([torch.matmul(weight[:, part == p], rows[part == p].double()) for p in range(workers)])
    assert torch.allclose(shares.sum(0), want[0], rtol=0, atol=1e-9)
    beyond = lambda change: (change.abs() > 2 * bound).flatten(1).any(1)
    assert beyond(shares).all(), "a part could be left out"
    assert beyond(shares - shares.roll(1, 0)).all(), "a part could stand in for its neighbour"
    assert beyond(shares + shares.roll(1, 0)).all(), "two parts could be left out"
    for shift in range(16, H, 16):
        assert beyond((want[0] - want[0].roll(shift, 0))[None]).all(), "a group of rows could stand in for another"

    out, lse, shared = run(t, 1.0)
    assert shared == -(-H // (16 * keys // 8))
    compare(out, lse, expected, torch.bfloat16, length, rows.abs().max().item())
