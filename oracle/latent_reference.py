"""Float64 definitions of the latent-attention path: rotation, append to a paged cache, absorbed and expanded attention.

Plain torch on any device. Every attention result comes with what a bound on a
16-bit implementation's error needs: ``spread`` = sum_j w_j |v_j| of each output
element and ``reach`` = the largest SCALE * sum |q_i k_i| of each row.
"""

from __future__ import annotations

import math

import torch


def rotate(x, positions, frequencies, layout="half", offset=0, magnitude=1.0, inverse=False):
    """x [..., T, H, D] with positions [..., T]: float64 result."""
    R = 2 * frequencies.numel()
    y = x.double().clone()
    angle = positions.double()[..., None, None] * frequencies.double()
    angle = -angle if inverse else angle
    part = y[..., offset:offset + R]
    u, v = (part[..., :R // 2], part[..., R // 2:]) if layout == "half" else (part[..., 0::2], part[..., 1::2])
    a = magnitude * (u * angle.cos() - v * angle.sin())
    b = magnitude * (u * angle.sin() + v * angle.cos())
    turned = torch.cat([a, b], -1) if layout == "half" else torch.stack([a, b], -1).flatten(-2)
    y[..., offset:offset + R] = turned
    return y


def rows_of(cu, used, table, page, blocks, b):
    """(token, block, slot) of the new tokens of request b that have a cache row."""
    start, end = int(cu[b]), int(cu[b + 1])
    out = []
    for t in range(start, end):
        p = int(used[b]) - end + t
        if p < 0 or p // page >= table.shape[1]:
            continue
        block = int(table[b, p // page])
        if 0 <= block < blocks:
            out.append((t, p, block, p % page))
    return out


def _attend(q, k, v, scale, limit):
    """q [n, H, Dk] over k [s, H or 1, Dk], v [s, H or 1, Dv]; row i sees the first limit[i] keys."""
    n, H, _ = q.shape
    s = k.shape[0]
    k, v = k.expand(s, H, -1), v.expand(s, H, -1)
    score = torch.matmul(q.transpose(0, 1), k.permute(1, 2, 0).contiguous()) * scale       # [H, n, s]
    reach = torch.matmul(q.abs().transpose(0, 1), k.abs().permute(1, 2, 0).contiguous()) * scale
    hidden = torch.arange(s, device=q.device)[None, :] >= torch.as_tensor(limit, device=q.device)[:, None]
    score = score.masked_fill(hidden, -math.inf)
    reach = reach.masked_fill(hidden, 0.0)
    lse = torch.logsumexp(score, -1) if s else torch.full((H, n), -math.inf, dtype=torch.float64, device=q.device)
    w = torch.exp(score - lse.clamp(min=-1e300)[..., None])
    values = v.transpose(0, 1).contiguous()
    out, spread = torch.matmul(w, values), torch.matmul(w, values.abs())
    top = reach.amax(-1) if s else torch.zeros((H, n), dtype=torch.float64, device=q.device)
    return out.transpose(0, 1), lse.t(), spread.transpose(0, 1), top.t()


def _empty(T, H, D, device):
    f64 = dict(dtype=torch.float64, device=device)
    return (torch.full((T, H, D), math.nan, **f64), torch.full((T, H), math.nan, **f64), torch.zeros((T, H, D), **f64),
            torch.zeros((T, H), **f64))


def latent_attention(q, q_rope, cache, table, cu, used, scale, causal=True):
    """(out, lse, spread, reach); tokens of no request are NaN."""
    T, H, L = q.shape
    page, blocks = cache.shape[1], cache.shape[0]
    result = _empty(T, H, L, q.device)
    whole = q.double() if q_rope is None else torch.cat([q.double(), q_rope.double()], -1)
    for b in range(table.shape[0]):
        start, end = int(cu[b]), int(cu[b + 1])
        n, length = end - start, max(0, int(used[b]))
        s = min(length, table.shape[1] * page)  # rows that the table holds; the tokens' places go by the length itself
        if n == 0:
            continue
        ids = table[b].tolist()
        there = [j for j in range(s) if 0 <= ids[j // page] < blocks]
        block = torch.tensor([ids[j // page] for j in there], dtype=torch.long, device=q.device)
        slot = torch.tensor([j % page for j in there], dtype=torch.long, device=q.device)
        rows = cache[block, slot].double()  # [keys, 1, L + R]
        limit = [sum(1 for j in there if j < (length - n + i + 1 if causal else s)) for i in range(n)]
        part = _attend(whole[start:end], rows, rows[..., :L], scale, limit)
        for whole_result, piece in zip(result, part):
            whole_result[start:end] = piece
    return result


def latent_attention_expanded(q, k_nope, k_rope, v, cu_q, cu_k, scale, causal=True):
    """(out, lse, spread, reach); queries of no request are NaN."""
    Tq, H, _ = q.shape
    result = _empty(Tq, H, v.shape[-1], q.device)
    for b in range(len(cu_q) - 1):
        qs, qe, ks, ke = int(cu_q[b]), int(cu_q[b + 1]), int(cu_k[b]), int(cu_k[b + 1])
        n, s = qe - qs, ke - ks
        if n == 0:
            continue
        k = torch.cat([k_nope[ks:ke].double(), k_rope[ks:ke, None].double().expand(s, H, -1)], -1)
        limit = [max(0, min(s, s - n + i + 1)) if causal else s for i in range(n)]
        part = _attend(q[qs:qe].double(), k, v[ks:ke].double(), scale, limit)
        for whole_result, piece in zip(result, part):
            whole_result[qs:qe] = piece
    return result


def rotation_bound(x, positions, frequencies, dtype, magnitude=1.0):
    """Largest error of a rotation computed in float32 and rounded once: u |y| (half a step of the storage type, or half its
    smallest subnormal) and, per pair, the float32 errors of cosine, sine, products and sum: the reduced angle is off by at
    most pi 2^-24 and float64 turns by |p f| 2^-51, cosine and sine by 4 steps of 2^-24, each product and the sum by one:
    together under 16 2^-24 + |p f| 2^-51 of |u| + |v| <= 2 max |x|."""
    info = torch.finfo(dtype)
    turns = (positions.double().abs().max() * frequencies.abs().max()).item() if positions.numel() else 0.0
    absolute = 2 * abs(magnitude) * x.double().abs().max().item() * (16 * 2.0 ** -24 + turns * 2.0 ** -51)
    return absolute + info.smallest_normal * info.eps / 2, info.eps / 2 * (1 + 1e-3)


def attention_bound(out, spread, reach, dtype, keys, values):
    """Largest error of an attention with products of 16-bit operands accumulated in float32 and P rounded to ``dtype``.

    With u half a step: P = p (1 + d), |d| <= u, in the products only, the denominator being the sum of the p, moves
    out = sum P v / sum p by at most u spread; a score summed in float32 over blocks of 32 columns, at most 18 of them, is
    off by at most (18 + 5) 2^-24 reach, its exponent (scale, difference, exp2) by 4 2^-24 (reach + |m|) more,
    |m| <= reach: 64 2^-24 reach covers both, which moves w by twice that and out by as much of spread + |out|; sums of P v
    over `keys` in float32 add (keys / 32 + 8) 2^-24 spread, the sum of the p, a quarter of them one after the other,
    (keys / 4 + 8) 2^-24 |out|; float16's P below 2^-14 is off by 2^-25 (all of it where it becomes 0), next to a sum of
    at least 1 (the maximum's own weight, or more where the running maximum lags); the result rounds once more.
    """
    u = torch.finfo(dtype).eps / 2
    score = 2 * 64 * 2.0 ** -24 * reach[..., None]
    bound = (u * spread + score * (spread + out.abs())) * (1 + 1e-2)
    bound = bound + 2.0 ** -24 * ((keys / 32 + 8) * spread + (keys / 4 + 8) * out.abs())
    if dtype == torch.float16:
        bound = bound + keys * 2.0 ** -25 * values
    return bound * (1 + u) + u * out.abs() + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def lse_bound(lse, reach, keys):
    """The scores' error, the float32 sum of `keys` weights and the logarithm's own 2^-20."""
    return 64 * 2.0 ** -24 * reach + (keys / 8 + 16) * 2.0 ** -24 + 2.0 ** -20 + 2.0 ** -22 * lse.abs()
