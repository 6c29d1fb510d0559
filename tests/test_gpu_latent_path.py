"""The operators together, as a latent model uses them: prompt in the expanded form, its latents appended, then steps of
tokens in the absorbed form over the cache, against one dense float64 attention of the whole sequence; and the rotation
and the append around ``sparse_mla``'s caches."""

import pytest
import torch

from ascendflow_amd.flash_attention import latent_attention_expanded
from ascendflow_amd.sparse_attention import append_paged_kv, apply_rotary, latent_attention, rotary_frequencies
from oracle import latent_reference as lr

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_prompt_then_tokens(device, layout):
    H, L, page, prompts, steps = 8, 512, 64, [37, 70], 3
    b16, scale = torch.bfloat16, 192 ** -0.5
    gen = torch.Generator(device=device).manual_seed(1)
    normal = lambda *shape: torch.randn(shape, generator=gen, device=device)
    w_k, w_v = (normal(H, L, 128) * L ** -0.5 for _ in range(2))  # expansion of a latent into keys and values
    frequencies = rotary_frequencies(64, scaling="yarn", factor=4.0, device=device)
    total = [p + steps for p in prompts]
    latent = [normal(n, L).to(b16) for n in total]
    rope = [normal(n, 64).to(b16) for n in total]
    query = [normal(n, H, 192).to(b16) for n in total]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=device)
    table = i32([[3, 0], [4, 1]])
    cache = torch.full((5, page, 1, L + 64), float("nan"), dtype=b16, device=device)

    def rotated(x, at):
        return apply_rotary(x, at, frequencies, layout=layout, offset=x.shape[-1] - 64)

    def step(begin, end):
        """New tokens begin[b] .. end[b] of each request: query rows, and their latents into the cache."""
        counts = [e - b for b, e in zip(begin, end)]
        cu = i32([0, counts[0], sum(counts)])
        cut = lambda xs: torch.cat([x[b:e] for x, b, e in zip(xs, begin, end)])
        at = torch.cat([torch.arange(b, e, device=device) for b, e in zip(begin, end)])
        append_paged_kv(cut(latent)[:, None], cache, table, cu, i32(end), rope=cut(rope)[:, None], frequencies=frequencies,
                        layout=layout)
        return cu, rotated(cut(query), at), cut(latent), at, cut(rope)

    # What the whole sequence gives, all in float64 from the same 16-bit inputs.
    want = []
    for b, n in enumerate(total):
        at = torch.arange(n, device=device)
        q = lr.rotate(query[b], at, frequencies, layout, 128)
        k_rope = lr.rotate(rope[b][:, None], at, frequencies, layout)
        k = torch.matmul(latent[b].double(), w_k.double()).transpose(0, 1)
        v = torch.matmul(latent[b].double(), w_v.double()).transpose(0, 1)
        score = torch.matmul(q.transpose(0, 1), torch.cat([k, k_rope.expand(n, H, 64)], -1).permute(1, 2, 0).contiguous())
        score = (score * scale).masked_fill(torch.ones(n, n, device=device).triu(1).bool(), -torch.inf)
        want.append(torch.matmul(score.softmax(-1), v.transpose(0, 1).contiguous()).transpose(0, 1))

    # 16-bit roundings on the way (queries, rotations, projections, weights, outputs): eight or so half steps
    # in the scores, whose exponentials they multiply by |score| (under 8 here), and in the values.
    u = torch.finfo(b16).eps / 2
    bound = lambda x: 40 * u * x.abs().max().item()
    cu, q, c, at, r = step([0, 0], prompts)
    k = torch.matmul(c.float(), w_k).transpose(0, 1).to(b16).contiguous()
    v = torch.matmul(c.float(), w_v).transpose(0, 1).to(b16).contiguous()
    k_rope = rotated(r[:, None], at)[:, 0]
    out = latent_attention_expanded(q, k, k_rope, v, cu, cu, SCALE=scale)
    start = 0
    for b, n in enumerate(prompts):
        assert (out[start:start + n].double() - want[b][:n]).abs().max() <= bound(want[b])
        start += n
    for i in range(steps):
        begin, end = [p + i for p in prompts], [p + i + 1 for p in prompts]
        cu, q, *_ = step(begin, end)
        absorbed = torch.matmul(q[..., :128].transpose(0, 1).float(), w_k.transpose(1, 2).contiguous()).to(b16).transpose(0, 1)
        o = latent_attention(absorbed, cache, table, cu, i32(end), SCALE=scale, q_rope=q[..., 128:])
        out = torch.matmul(o.transpose(0, 1).float(), w_v).transpose(0, 1)
        for b in range(2):
            assert (out[b].double() - want[b][prompts[b] + i]).abs().max() <= bound(want[b])


def test_rotation_and_append_feed_the_sparse_operator(device):
    """``ori_kv`` filled by the append equals a cache filled by hand, and so does ``sparse_mla`` over it."""
    from ascendflow_amd.sparse_attention import sparse_mla
    from ascendflow_amd.sparse_attention.inputs import make_inputs, measurement_policy

    policy = measurement_policy(batch=2, query_tokens=3, context=300)
    inputs = make_inputs(policy, 300, device=device, scale=1.0)
    t = inputs.tensors
    frequencies = rotary_frequencies(64, device=device)
    rows = torch.randn((6, 1, 512), device=device).bfloat16()
    by_hand = t["ori_kv"].clone()
    for b in range(2):
        for j in range(3):
            p = 300 - 3 + j
            at = torch.tensor([p], dtype=torch.int32, device=device)
            by_hand[t["ori_block_table"][b, p // 128].long(), p % 128] = apply_rotary(
                rows[3 * b + j][None], at, frequencies, offset=448)[0]
    append_paged_kv(rows, t["ori_kv"], t["ori_block_table"], t["cu_seqlens_q"], t["seqused_ori_kv"],
                    frequencies=frequencies, offset=448)
    assert torch.equal(t["ori_kv"], by_hand)
    first = sparse_mla(*inputs.call_args(), **inputs.call_kwargs()).clone()
    t["ori_kv"].copy_(by_hand)
    assert torch.equal(first, sparse_mla(*inputs.call_args(), **inputs.call_kwargs()))
    positions = torch.cat([torch.arange(297, 300, device=device)] * 2)
    back = apply_rotary(first, positions, frequencies, offset=448, inverse=True)
    assert torch.isfinite(back.float()).all() and torch.equal(back[..., :448], first[..., :448])


@pytest.mark.parametrize("H", [16, 128])
def test_tokens_ahead_of_the_first_request_stay_as_they_were(device, H):
    from tests import test_gpu_latent_expanded as expanded
    from tests.latent_helpers import call, paged

    t = paged(device, [1, 2], [90, 300], H=H, spare_tokens=3)
    shifted = {**t, "cu_seqlens_q": t["cu_seqlens_q"] + 3,
               "q": torch.cat([t["q"][3:], t["q"][:3]]), "q_rope": torch.cat([t["q_rope"][3:], t["q_rope"][:3]])}
    want, got = torch.full_like(t["q"], 7.0), torch.full_like(t["q"], 7.0)
    call(t, 0.07, True, want)
    call(shifted, 0.07, True, got)
    assert torch.equal(got[3:], want[:3]) and (got[:3] == 7).all()

    t = expanded.inputs(device, [1, 2], [900, 700], H=4, spare=3)  # split keys, joined by a second launch
    shifted = {**t, "cu_q": t["cu_q"] + 3, "q": torch.cat([t["q"][3:], t["q"][:3]])}
    want, got = (torch.full((6, 4, 128), 7.0, dtype=torch.bfloat16, device=device) for _ in range(2))
    expanded.call(t, out=want)
    expanded.call(shifted, out=got)
    assert torch.equal(got[3:], want[:3]) and (got[:3] == 7).all()
