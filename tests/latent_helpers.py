"""Paged latent-attention inputs of the tests, and their comparison against the float64 definitions."""

import math

import torch

from oracle import latent_reference as lr

B16 = {"bf16": torch.bfloat16, "f16": torch.float16}


def paged(device, counts, lengths, *, H=4, L=128, R=64, page=16, dtype="bf16", seed=0, spare_tokens=0, spare_pages=3,
          width=None, heads_first=False):
    """Inputs of one ``latent_attention`` call: a cache of NaN whose rows below each request's length are finite."""
    gen = torch.Generator().manual_seed(seed)
    b16 = B16[dtype]
    T = sum(counts) + spare_tokens
    need = [-(-s // page) for s in lengths]
    width = max(1, max(need)) if width is None else width
    blocks = sum(need) + spare_pages
    order = torch.randperm(blocks, generator=gen)
    table = torch.full((len(counts), width), -1, dtype=torch.int32)
    cache = torch.full((blocks, page, 1, L + R), math.nan)
    at = 0
    for b, (s, pages) in enumerate(zip(lengths, need)):
        ids = order[at:at + pages]
        table[b, :pages] = ids.to(torch.int32)
        rows = torch.randn((pages * page, L + R), generator=gen)
        rows[s:] = math.nan  # behind the request's last row
        cache[ids] = rows.view(pages, page, 1, L + R)
        at += pages
    cu = torch.tensor([0] + [sum(counts[:i + 1]) for i in range(len(counts))], dtype=torch.int32)

    def rows_of(columns):
        shape = (H, T, columns) if heads_first else (T, H, columns)
        x = torch.randn(shape, generator=gen).to(b16).to(device)
        return x.transpose(0, 1) if heads_first else x

    return dict(q=rows_of(L), q_rope=rows_of(R) if R else None, kv_cache=cache.to(b16).to(device),
                block_table=table.to(device), cu_seqlens_q=cu.to(device),
                seqused_kv=torch.tensor(lengths, dtype=torch.int32).to(device))


def call(t, scale, causal=True, out=None, lse=None):
    from ascendflow_amd.sparse_attention import latent_attention

    return latent_attention(t["q"], t["kv_cache"], t["block_table"], t["cu_seqlens_q"], t["seqused_kv"], SCALE=scale,
                            q_rope=t["q_rope"], CAUSAL=causal, out=out, softmax_lse=lse)


def compare(out, lse, expected, dtype, keys, values):
    """Every element within the derived bound; tokens of no request are left out."""
    want, want_lse, spread, reach = expected
    mine = ~torch.isnan(want_lse).any(dim=1)
    want, want_lse, spread, reach = want[mine], want_lse[mine], spread[mine], reach[mine]
    got = out[mine].double()
    assert torch.isfinite(got).all()
    excess = (got - want).abs() - lr.attention_bound(want, spread, reach, dtype, keys, values)
    assert excess.max() <= 0, f"out beyond its bound by {excess.max().item():.3e}"
    empty = torch.isinf(want_lse)
    assert torch.equal(torch.isinf(lse[mine]) & (lse[mine] < 0), empty)
    assert (got[empty] == 0).all()
    off = (lse[mine].double() - want_lse).abs()[~empty] - lr.lse_bound(want_lse, reach, keys)[~empty]
    assert off.numel() == 0 or off.max() <= 0, f"lse beyond its bound by {off.max().item():.3e}"


def check(device, counts, lengths, *, causal=True, scale=None, sentinel=7.0, tensors=None, **kw):
    """One call on seeded inputs against the definition; returns (tensors, out, lse)."""
    dtype = B16[kw.get("dtype", "bf16")]
    t = paged(device, counts, lengths, **kw) if tensors is None else tensors
    T, H, L = t["q"].shape
    scale = (L + (0 if t["q_rope"] is None else t["q_rope"].shape[2])) ** -0.5 if scale is None else scale
    out = torch.full((T, H, L), sentinel, dtype=dtype, device=device)
    lse = torch.full((T, H), sentinel, dtype=torch.float32, device=device)
    assert call(t, scale, causal, out, lse) is out
    torch.cuda.synchronize()
    cpu = {k: None if v is None else v.cpu() for k, v in t.items()}
    expected = lr.latent_attention(cpu["q"], cpu["q_rope"], cpu["kv_cache"], cpu["block_table"], cpu["cu_seqlens_q"],
                                   cpu["seqused_kv"], scale, causal)
    finite = cpu["kv_cache"].double()
    values = finite[torch.isfinite(finite)].abs().max().item() if torch.isfinite(finite).any() else 0.0
    compare(out.cpu(), lse.cpu(), expected, dtype, max(1, *lengths) if len(lengths) > 1 else max(1, lengths[0]), values)
    padding = sum(counts)
    assert (out[padding:] == sentinel).all() and (lse[padding:] == sentinel).all()
    return t, out, lse
