"""Inputs of the tests of the 8-bit paged cache, and the comparison of its attention against the float64 definition."""

import math

import torch

from oracle import latent_reference as lr
from oracle import quantized_reference as qr

B16 = {"bf16": torch.bfloat16, "f16": torch.float16}
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}


def codes_of(x, codes):
    """float32 values in units of their scale as codes."""
    top = qr.TOP[CODES[codes]]
    x = x.clamp(-top, top)
    return x.to(CODES[codes]) if codes == "e4m3" else x.round().to(torch.int8)


def paged(device, counts, lengths, *, HQ=8, HKV=2, D=128, page=32, group=None, codes="e4m3", dtype="bf16", seed=0,
          spare_tokens=0, spare_pages=3, width=None, heads_first=False, plain_scales=False):
    """Inputs of one ``quantized_attention`` call. Rows behind each request's last are codes of no number (e4m3) or large
    (int8), blocks without a row have a scale of NaN; scales vary by head and block and are powers of two or not."""
    gen = torch.Generator().manual_seed(seed)
    group = page if group is None else group
    need = [-(-s // page) for s in lengths]
    width = max(1, max(need)) if width is None else width
    blocks = sum(need) + spare_pages
    order = torch.randperm(blocks, generator=gen)
    table = torch.full((len(counts), width), -1, dtype=torch.int32)
    t = {}
    written = torch.zeros((blocks, page), dtype=torch.bool)
    at = 0
    for b, (s, pages) in enumerate(zip(lengths, need)):
        ids = order[at:at + pages]
        table[b, :pages] = ids.to(torch.int32)
        rows = torch.zeros(pages * page, dtype=torch.bool)
        rows[:s] = True
        written[ids] = rows.view(pages, page)
        at += pages
    for which in ("k", "v"):
        x = torch.randn((blocks, page, HKV, D), generator=gen) * (30.0 if codes == "e4m3" else 40.0)
        bytes_ = codes_of(x, codes).view(torch.uint8)
        bytes_[~written] = 0x7f
        t[which + "_cache"] = bytes_.view(CODES[codes]).to(device)
        exponent = torch.randint(-9, -3, (blocks, page // group, HKV), generator=gen)
        scale = torch.exp2(exponent.float())
        if not plain_scales:
            scale *= 1 + torch.rand(scale.shape, generator=gen) * (torch.rand(scale.shape, generator=gen) < 0.5)
        scale[~written.view(blocks, page // group, group).any(-1)] = math.nan
        t[which + "_scale"] = scale.to(device)
    T = sum(counts) + spare_tokens
    q = torch.randn((HQ, T, D) if heads_first else (T, HQ, D), generator=gen).to(B16[dtype]).to(device)
    t.update(q=q.transpose(0, 1) if heads_first else q, block_table=table.to(device),
             cu_seqlens_q=torch.tensor([0] + [sum(counts[:i + 1]) for i in range(len(counts))], dtype=torch.int32).to(device),
             seqused_kv=torch.tensor(lengths, dtype=torch.int32).to(device))
    return t


def call(t, scale, causal=True, out=None, lse=None):
    from ascendflow_amd.flash_attention import quantized_attention

    return quantized_attention(t["q"], t["k_cache"], t["v_cache"], t["k_scale"], t["v_scale"], t["block_table"],
                               t["cu_seqlens_q"], t["seqused_kv"], SCALE=scale, CAUSAL=causal, out=out, softmax_lse=lse)


def expected(t, scale, causal):
    """The definition's (out, lse, spread, reach), and the two figures of its bound that the scales give."""
    cpu = {k: v.cpu() for k, v in t.items()}
    k, v = (qr.values(cpu[w + "_cache"], cpu[w + "_scale"].clamp(min=2.0 ** -80)) for w in ("k", "v"))
    result = qr.attention(cpu["q"], k, v, cpu["block_table"], cpu["cu_seqlens_q"], cpu["seqused_kv"], scale, causal)
    used = cpu["v_scale"][torch.isfinite(cpu["v_scale"])].clamp(min=2.0 ** -80)
    exponents = used.log2().abs().max().item() if used.numel() else 0.0
    largest = used.max().item() * qr.TOP[cpu["v_cache"].dtype] if used.numel() else 0.0
    return result, largest, exponents


def compare(out, lse, want_all, dtype, keys):
    """Every element within the derived bound; tokens of no request are left out."""
    (want, want_lse, spread, reach), largest, exponents = want_all
    mine = ~torch.isnan(want_lse).any(dim=1)
    want, want_lse, spread, reach = want[mine], want_lse[mine], spread[mine], reach[mine]
    got = out[mine].double()
    assert torch.isfinite(got).all()
    excess = (got - want).abs() - qr.attention_bound(want, spread, reach, dtype, keys, largest, exponents)
    assert excess.numel() == 0 or excess.max() <= 0, f"out beyond its bound by {excess.max().item():.3e}"
    empty = torch.isinf(want_lse)
    assert torch.equal(torch.isinf(lse[mine]) & (lse[mine] < 0), empty)
    assert (got[empty] == 0).all()
    # lse = (m + log2 sum) ln 2 with |m| up to reach + exponents: two roundings more than the other attentions'.
    off = (lse[mine].double() - want_lse).abs()[~empty]
    bound = (lr.lse_bound(want_lse, reach, keys) + 8 * 2.0 ** -24 * (reach + exponents))[~empty]
    assert off.numel() == 0 or (off - bound).max() <= 0, f"lse beyond its bound by {(off - bound).max().item():.3e}"


def check(device, counts, lengths, *, causal=True, scale=None, sentinel=7.0, tensors=None, **kw):
    """One call on seeded inputs against the definition; returns (tensors, out, lse)."""
    t = paged(device, counts, lengths, **kw) if tensors is None else tensors
    dtype, (T, HQ, D) = t["q"].dtype, t["q"].shape
    scale = D ** -0.5 if scale is None else scale
    out = torch.full((T, HQ, D), sentinel, dtype=dtype, device=device)
    lse = torch.full((T, HQ), sentinel, dtype=torch.float32, device=device)
    assert call(t, scale, causal, out, lse) is out
    torch.cuda.synchronize()
    compare(out.cpu(), lse.cpu(), expected(t, scale, causal), dtype, max(1, *lengths) if len(lengths) > 1 else max(1, lengths[0]))
    padding = int(t["cu_seqlens_q"][-1])
    assert (out[padding:] == sentinel).all() and (lse[padding:] == sentinel).all()
    return t, out, lse
