"""The causal limit of absorbed latent attention where a request is longer than its table: it goes by the length itself, as
the places of the append do, and every token still sees its own row."""

import pytest
import torch

from oracle import latent_reference as lr
from tests.latent_helpers import call, check, paged

pytestmark = pytest.mark.gpu


def beyond(device, counts, over, *, H, L=128, page=16, pages=4, **kw):
    """Requests that fill their tables and count ``over`` rows more."""
    lengths = [pages * page] * len(counts)
    t = paged(device, counts, lengths, H=H, L=L, R=64, page=page, **kw)
    t["seqused_kv"] = torch.tensor([n + o for n, o in zip(lengths, over)], dtype=torch.int32, device=device)
    return t, lengths


@pytest.mark.parametrize("H,L", [(4, 128), (16, 512), (128, 512), (65, 256)])
@pytest.mark.parametrize("counts,over", [
    ([4], [2]), ([4], [4]), ([1], [1]), ([5, 3, 0, 2], [4, 1, 3, 2**31 - 1 - 64]), ([70], [66]), ([150, 9], [40, 0]),
])
def test_lengths_beyond_the_table(device, counts, over, H, L):
    t, lengths = beyond(device, counts, over, H=H, L=L, spare_tokens=2)
    check(device, counts, lengths, tensors=t)
    check(device, counts, lengths, tensors=t, causal=False)


@pytest.mark.parametrize("counts,over", [([230], [100]), ([600, 1, 500], [300, 1, 77])])
def test_a_tile_per_workgroup(device, counts, over):
    t, lengths = beyond(device, counts, over, H=128, pages=17)
    check(device, counts, lengths, tensors=t)


def test_the_same_as_under_a_wider_table_whose_pages_hold_no_keys(device):
    counts, over = [4, 20], [2, 30]
    t, lengths = beyond(device, counts, over, H=16)
    wide = dict(t, block_table=torch.cat([t["block_table"], torch.full((2, 2), -1, dtype=torch.int32, device=device)], 1))
    _, narrow_out, narrow_lse = check(device, counts, lengths, tensors=t)
    _, wide_out, wide_lse = check(device, counts, [n + o for n, o in zip(lengths, over)], tensors=wide)
    # Two results of one definition: each within its own bound, so within twice the larger apart.
    want, want_lse, spread, reach = lr.latent_attention(*(x.cpu() for x in (
        t["q"], t["q_rope"], t["kv_cache"], t["block_table"], t["cu_seqlens_q"], t["seqused_kv"])), 192 ** -0.5)
    bound = lr.attention_bound(want, spread, reach, torch.bfloat16, 96, 8.0)
    assert ((narrow_out.cpu().double() - wide_out.cpu().double()).abs() <= 2 * bound).all()
    assert ((narrow_lse - wide_lse).cpu().double().abs() <= 2 * lr.lse_bound(want_lse, reach, 96)).all()


def test_a_token_sees_the_row_that_the_append_gave_it(device):
    """Token 0 of 4, of a request two rows longer than its table, takes row 62 and is the row's only large score."""
    from ascendflow_amd.sparse_attention import append_paged_kv

    t, _ = beyond(device, [4], [2], H=16)
    t["q"].fill_(1.0)
    t["q_rope"].zero_()
    t["kv_cache"].zero_()
    rows = torch.zeros((4, 1, 192), dtype=torch.bfloat16, device=device)
    rows[0, 0, :128] = 2.0
    append_paged_kv(rows, t["kv_cache"], t["block_table"], t["cu_seqlens_q"], t["seqused_kv"])
    out = call(t, 1.0)
    assert (out == 2.0).all()  # a score of 256 against zeros
