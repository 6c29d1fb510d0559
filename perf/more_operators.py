"""Measured calls of the 8-bit paged cache: append, the attention that reads it, and the upkeep of its pages.

Keys and values of several heads lie in pages as e4m3 or int8 codes, with a float32 scale for each block of ``group``
tokens and head. ``listed()`` gives the fixed cases, ``draw(rng)`` another one of the same ranges, ``prepare`` what a
serving program has in hand before the call, ``run`` one call, in the plain form (elementary torch operations) or, where
``own`` is true, through the framework's entry points, ``exact`` its result in float64.
"""

from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

B16 = {"bf16": torch.bfloat16, "f16": torch.float16}
CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
TOP = {"e4m3": 448.0, "int8": 127.0}      # the largest code
LEAST = -80                               # exponent of the least scale that an append writes


def listed():
    return [
        # A batched decode step: one token of each of 64 requests, 8 heads, into blocks that mostly hold tokens already.
        _append("append8_decode_64x1", B=64, n=1, context=2000, HKV=8),
        # Prompts of a few unequal requests behind earlier tokens, int8, blocks of 32 tokens.
        _append("append8_prompt_3x1987", B=3, n=1987, context=2600, HKV=8, page=128, group=32, codes="int8", dtype="f16",
                ragged=True),
        # One user's single-token step at 4K: latency bound.
        _attention("attention8_decode_1x1_4k", B=1, n=1, context=4096, HQ=32, HKV=8),
        # Batched single-token decode over long, unequal contexts, bound by the cache's bytes.
        _attention("attention8_decode_64x1_16k", B=64, n=1, context=16384, HQ=64, HKV=8, ragged=True),
        # Verification of three draft tokens a request on a model of narrow heads, int8, small pages.
        _attention("attention8_verify_48x4", B=48, n=4, context=5000, HQ=32, HKV=4, D=64, page=16, group=16, codes="int8",
                   dtype="f16", ragged=True),
        # A chunk of a long prompt behind 18K tokens of its own: bound by the matrix products.
        _attention("attention8_chunk_1x2000", B=1, n=2000, context=20011, HQ=32, HKV=8, page=128, group=128),
        # Copies of the last pages of four beams of a small model: latency bound.
        _copy("copy_pages_4", pairs=4, layers=1, HKV=2, page=16, group=16, blocks=64),
        # 500 pages, an eighth of the list empty, in the caches and scales of eight layers.
        _copy("copy_pages_500x8", pairs=500, layers=8, HKV=8, blocks=1200, empty=0.125),
        # A beam search step: four beams of each of eight requests continue from the best of them.
        _fork("fork_beams_8x4", B=32, W=64, context=1500, blocks=2048, kept=0.4, ended=0.0),
        # A serving step over many rows: most go on as they are, some end, some start as samples of another.
        _fork("fork_serving_256", B=256, W=1024, context=16000, page=16, blocks=300000, kept=0.8, ended=0.1, reserve=8),
        # A small cache half empty.
        _compact("compact_2048", B=32, W=64, context=2000, blocks=2048),
        # A large cache of small pages.
        _compact("compact_300000", B=256, W=1024, context=12000, page=16, blocks=300000),
    ]


def _append(name, *, B, n, context, HKV, D=128, page=64, group=64, codes="e4m3", dtype="bf16", ragged=False):
    return {"name": name, "kind": "append", "B": B, "n": n, "context": context, "HKV": HKV, "D": D, "page": page,
            "group": group, "codes": codes, "dtype": dtype, "ragged": ragged}


def _attention(name, *, B, n, context, HQ, HKV, D=128, page=64, group=64, codes="e4m3", dtype="bf16", ragged=False):
    return {"name": name, "kind": "attention", "B": B, "n": n, "context": context, "HQ": HQ, "HKV": HKV, "D": D,
            "page": page, "group": group, "codes": codes, "dtype": dtype, "ragged": ragged}


def _copy(name, *, pairs, layers, HKV, blocks, D=128, page=64, group=64, codes="e4m3", empty=0.0):
    return {"name": name, "kind": "copy", "pairs": pairs, "layers": layers, "HKV": HKV, "D": D, "page": page,
            "group": group, "blocks": blocks, "codes": codes, "empty": empty}


def _fork(name, *, B, W, context, blocks, kept, ended, page=64, reserve=1):
    return {"name": name, "kind": "fork", "B": B, "W": W, "context": context, "page": page, "blocks": blocks,
            "kept": kept, "ended": ended, "reserve": reserve}


def _compact(name, *, B, W, context, blocks, page=64):
    return {"name": name, "kind": "compact", "B": B, "W": W, "context": context, "page": page, "blocks": blocks}


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(max(low, high))))))


def draw(rng):
    kind = rng.choice(["append", "append", "attention", "attention", "attention", "attention", "copy", "fork", "compact"])
    page = rng.choice([16, 32, 64, 64, 128])
    group = rng.choice([g for g in (16, 32, 64, 128) if g <= page] + [page])
    codes, dtype = rng.choice(["e4m3", "e4m3", "int8"]), rng.choice(["bf16", "bf16", "f16"])
    if kind == "append":
        B = _log_int(rng, 1, 256)
        n = _log_int(rng, 1, 8 if rng.random() < 0.5 else max(8, 8192 // B))
        case = _append("", B=B, n=n, context=min(_log_int(rng, 2 * n, 8 * n + 2000), max(2 * n, 400000 // B)),
                       HKV=rng.choice([1, 2, 4, 5, 8, 8]), D=rng.choice([64, 128, 128, 256]), page=page, group=group,
                       codes=codes, dtype=dtype, ragged=rng.random() < 0.6)
    elif kind == "attention":
        HQ, HKV = rng.choice([(8, 1), (16, 2), (32, 8), (32, 4), (64, 8), (40, 8), (12, 4), (8, 8), (16, 1)])
        D = rng.choice([64, 128, 128, 128, 256])
        B = _log_int(rng, 1, 128)
        n = 1 if rng.random() < 0.5 else _log_int(rng, 2, 8 if rng.random() < 0.6 else max(8, 2000 // B))
        # At most the cache bytes and the products of the largest listed cases.
        context = min(_log_int(rng, max(30, 2 * n), 131072), int(1.6e9 / (2 * HKV * D * B)),
                      int(5.5e11 / (4 * HQ * D * B * n)))
        case = _attention("", B=B, n=n, context=max(2 * n, context), HQ=HQ, HKV=HKV, D=D, page=page, group=group,
                          codes=codes, dtype=dtype, ragged=rng.random() < 0.6)
    elif kind == "copy":
        HKV, D, layers = rng.choice([1, 2, 8]), rng.choice([64, 128, 256]), _log_int(rng, 1, 16)
        pairs = min(_log_int(rng, 1, 2000), max(1, 500 * 8 * 64 * 8 * 128 // (layers * page * HKV * D)))
        case = _copy("", pairs=pairs, layers=layers, HKV=HKV, D=D, page=page, group=group,
                     blocks=2 * pairs + _log_int(rng, 1, 200), codes=codes, empty=rng.choice([0.0, 0.3, 0.6]))
    else:
        B = _log_int(rng, 2, 512)
        context = min(_log_int(rng, 20, 100000), 8000 * 512 // B)
        W = -(-(context + 64) // page) + rng.randint(0, 8)
        blocks = B * W + _log_int(rng, 64, 4096)
        if kind == "fork":
            case = _fork("", B=B, W=W, context=context, page=page, blocks=blocks, kept=rng.uniform(0.2, 0.9),
                         ended=rng.choice([0.0, 0.1]), reserve=rng.choice([0, 1, 4, 64]))
        else:
            case = _compact("", B=B, W=W, context=context, page=page, blocks=blocks)
    del case["name"]
    return case


# ---- sizes -----------------------------------------------------------------------


def _requests(case):
    """(new tokens, length with them) of each request; the same for every seed."""
    B, n, length = case["B"], case["n"], case["context"]
    if not case["ragged"]:
        return [n] * B, [length] * B
    rng = random.Random(B * 1000003 + n * 1009 + length)
    counts = [max(1, rng.randint(n // 2, n)) for _ in range(B)]
    return counts, [max(c, rng.randint(length // 2, length)) for c in counts]


def work(case):
    kind = case["kind"]
    if kind == "append":
        counts, lengths = _requests(case)
        T, G = sum(counts), case["group"]
        blocks = sum((s - 1) // G - (s - c) // G + 1 for c, s in zip(counts, lengths))
        return {"bytes": 2 * (3 * T * case["HKV"] * case["D"] + 4 * blocks * case["HKV"]) + 8 * case["B"],
                "flops": 4 * T * case["HKV"] * case["D"]}
    if kind == "attention":
        counts, lengths = _requests(case)
        T, HQ, HKV, D, G = sum(counts), case["HQ"], case["HKV"], case["D"], case["group"]
        pairs = sum(c * s - c * (c - 1) // 2 for c, s in zip(counts, lengths))
        return {"bytes": 2 * HKV * sum(D * s + 4 * -(-s // G) for s in lengths) + T * HQ * (4 * D + 4),
                "flops": 4 * HQ * D * pairs}
    if kind == "copy":
        row = 2 * case["HKV"] * (case["page"] * case["D"] + 4 * (case["page"] // case["group"]))
        full = case["pairs"] - int(case["pairs"] * case["empty"])
        return {"bytes": 2 * full * case["layers"] * row + 8 * case["pairs"], "flops": 0}
    # The table and the counts once; a fork writes rows anew, a compaction both.
    table, counts = 4 * case["B"] * case["W"], 4 * case["blocks"]
    return {"bytes": 2 * table + (counts if kind == "fork" else 2 * counts), "flops": 0}


# ---- inputs ----------------------------------------------------------------------


def _power(top, codes):
    """The least power of two that ``top`` is at most the largest code of, from 2^LEAST on, as float32."""
    fraction, exponent = torch.frexp(top.float())
    limit, shift = (0.875, 9) if codes == "e4m3" else (127 / 128, 7)
    exponent = torch.where(top > 0, exponent - shift + (fraction > limit).int(), torch.full_like(exponent, LEAST))
    return ((exponent.clamp(min=LEAST) + 127) << 23).view(torch.float32)


def _encode(x, codes):
    """x (in units of its scale, float32) rounded to codes: to nearest, ties to even."""
    x = x.clamp(-TOP[codes], TOP[codes])
    return x.to(CODES[codes]) if codes == "e4m3" else x.nan_to_num(0.0).round().to(torch.int8)


def _offsets(counts, device):
    total = [0]
    for c in counts:
        total.append(total[-1] + c)
    return torch.tensor(total, dtype=torch.int32, device=device)


def _filled(case, blocks, gen, device):
    """A cache of normal rows whose size varies by head and block, as codes, and its scales."""
    HKV, D, page, G, codes = case["HKV"], case["D"], case["page"], case["group"], case["codes"]
    cache = torch.empty((blocks, page, HKV, D), dtype=CODES[codes], device=device)
    scale = torch.empty((blocks, page // G, HKV), dtype=torch.float32, device=device)
    size = torch.exp(0.5 * torch.randn((HKV,), generator=gen, device=device))
    step = max(1, (1 << 27) // (page * HKV * D))
    for at in range(0, blocks, step):
        m = min(step, blocks - at)
        x = torch.randn((m, page // G, G, HKV, D), generator=gen, device=device)
        x *= (size * torch.exp(0.3 * torch.randn((m, page // G, HKV), generator=gen, device=device)))[:, :, None, :, None]
        s = _power(x.abs().amax(dim=(2, 4)), codes)
        cache[at:at + m] = _encode(x / s[:, :, None, :, None], codes).view(m, page, HKV, D)
        scale[at:at + m] = s
    return cache, scale


def _rows(case, gen, device):
    """Tables of requests that share full pages in groups, as samples of one prompt do, and the references of each page."""
    B, W, page, blocks = case["B"], case["W"], case["page"], case["blocks"]
    lengths = torch.randint(case["context"] // 2, case["context"] + 1, (-(-B // 4),), generator=gen, device=device)
    lengths = lengths.repeat_interleave(4)[:B]
    held = (lengths + page - 1) // page
    column = torch.arange(W, device=device)
    order = torch.randperm(blocks, generator=gen, device=device)[:B * W].view(B, W)
    shared = column[None, :] < (lengths // page // 2)[:, None]          # the first half of them
    first = (torch.arange(B, device=device) // 4 * 4)[:, None].expand(B, W)
    table = torch.where(shared, order.gather(0, first), order)
    table = torch.where(column[None, :] < held[:, None], table, torch.full_like(table, -1)).to(torch.int32)
    counts = torch.zeros(blocks + 1, dtype=torch.int32, device=device)
    counts.index_add_(0, torch.where(table >= 0, table, blocks).flatten().long(), torch.ones(B * W, dtype=torch.int32, device=device))
    return table, counts[:blocks].clone(), lengths.to(torch.int32)


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device)
    gen.manual_seed(seed)
    kind = case["kind"]
    state = {"case": case}
    if kind in ("fork", "compact"):
        table, counts, lengths = _rows(case, gen, device)
        state.update(table=table, counts=counts)
        if kind == "fork":
            # Rows that go on as they are, rows that end, and rows that continue from one of the first kind.
            B = case["B"]
            u = torch.rand((B,), generator=gen, device=device)
            row = torch.arange(B, device=device)
            stay = (u < case["kept"]) | (row % 4 == 0)
            from_ = torch.where(stay, row, row // 4 * 4)
            from_ = torch.where((u >= 1 - case["ended"]) & ~stay, torch.full_like(row, -1), from_)
            state["parents"] = from_.to(torch.int32)
            state["used"] = torch.where(from_ >= 0, lengths[from_.clamp(min=0)], torch.zeros_like(lengths)).to(torch.int32)
        return state
    if kind == "copy":
        P, blocks = case["pairs"], case["blocks"]
        state["caches"] = [t for _ in range(case["layers"]) for _ in range(2) for t in _filled(case, blocks, gen, device)]
        order = torch.randperm(blocks, generator=gen, device=device).to(torch.int32)
        source, destination = order[:P].clone(), order[P:2 * P].clone()
        off = torch.randperm(P, generator=gen, device=device)[:int(P * case["empty"])]
        source[off], destination[off] = -1, -1
        state.update(source=source, destination=destination)
        return state

    counts, lengths = _requests(case)
    T, HKV, D, page, b16 = sum(counts), case["HKV"], case["D"], case["page"], B16[case["dtype"]]
    pages = [-(-s // page) for s in lengths]
    order = torch.randperm(sum(pages), generator=gen, device=device).to(torch.int32).cpu()
    table = torch.full((case["B"], max(pages)), -1, dtype=torch.int32)
    at = 0
    for b, p in enumerate(pages):
        table[b, :p] = order[at:at + p]
        at += p
    state.update(counts=counts, lengths=lengths, cu_q=_offsets(counts, device), table=table.to(device),
                 used=torch.tensor(lengths, dtype=torch.int32, device=device))
    state["k_cache"], state["k_scale"] = _filled(case, sum(pages), gen, device)
    state["v_cache"], state["v_scale"] = _filled(case, sum(pages), gen, device)
    if kind == "append":
        both = torch.randn((T, 2, HKV, D), generator=gen, device=device).to(b16)  # one projection
        state["k"], state["v"] = both[:, 0], both[:, 1]
    else:
        state["q"] = torch.randn((T, case["HQ"], D), generator=gen, device=device).to(b16)
        state["scale"] = D ** -0.5
    return state


# ---- one call ----------------------------------------------------------------------


def _append_one(state, x, cache, scale):
    """New rows x [T, HKV, D] into one cache, block by block."""
    case = state["case"]
    page, G, codes = case["page"], case["group"], case["codes"]
    cu, used = state["cu_q"].long(), state["used"].long()
    token = torch.arange(x.shape[0], device=x.device)
    request = torch.searchsorted(cu[1:], token, right=True)
    position = used[request] - cu[request + 1] + token
    slot = state["table"][request, position // page].long() * page + position % page
    block, inside = slot // G, slot % G
    flat = scale.view(-1, scale.shape[-1])
    blocks, HKV = flat.shape
    x = x.float()
    top = torch.where(x.isfinite(), x.abs(), torch.zeros_like(x)).amax(dim=-1)
    most = torch.zeros_like(flat).index_reduce_(0, block, top, "amax")
    start = torch.full((blocks,), G, device=x.device).index_reduce_(0, block, inside, "amin")
    need = _power(most, codes)
    scale_now = torch.where((start < G)[:, None], torch.where((start > 0)[:, None], torch.maximum(need, flat), need), flat)
    # Rows that a block held before its new ones: only the first block of a request has any.
    first = block[cu[:-1]]
    rows = cache.view(blocks, G, HKV, -1)
    old = rows[first]
    again = _encode(old.float() * flat[first][:, None, :, None] * (1.0 / scale_now[first])[:, None, :, None], codes)
    before = torch.arange(G, device=x.device)[None, :] < start[first][:, None]
    rows[first] = torch.where(before[:, :, None, None], again.float(), old.float()).to(old.dtype)
    cache.view(-1, HKV, cache.shape[-1])[slot] = _encode(x * (1.0 / scale_now[block])[:, :, None], codes)
    flat.copy_(scale_now)


def _rows_of(state, b, s, which):
    """The first s rows of request b as the values they stand for, float32 [HKV, s, D]."""
    case = state["case"]
    page = case["page"]
    block = state["table"][b, :-(-s // page)].long()
    x = state[which + "_cache"][block].float().view(-1, case["group"], case["HKV"], case["D"])
    x = x * state[which + "_scale"][block].view(-1, 1, case["HKV"], 1)
    return x.view(-1, case["HKV"], case["D"])[:s].transpose(0, 1).contiguous()


def _run_attention(state):
    case = state["case"]
    HQ, HKV, D = case["HQ"], case["HKV"], case["D"]
    g = HQ // HKV
    out = torch.empty_like(state["q"])
    lse = torch.empty(out.shape[:2], dtype=torch.float32, device=out.device)
    t = 0
    for b, (n, s) in enumerate(zip(state["counts"], state["lengths"])):
        k, v = _rows_of(state, b, s, "k"), _rows_of(state, b, s, "v")
        key = torch.arange(s, device=out.device)
        step = max(1, (1 << 29) // (HQ * s))
        for i in range(0, n, step):
            m = min(step, n - i)
            q = state["q"][t + i:t + i + m].float().view(m, HKV, g, D).transpose(0, 1).reshape(HKV, m * g, D)
            score = torch.bmm(q, k.transpose(1, 2).contiguous()) * state["scale"]
            if n > 1:
                last = torch.arange(s - n + i, s - n + i + m, device=out.device).repeat_interleave(g)
                score.masked_fill_(key > last[:, None], -math.inf)
            top = score.amax(dim=-1, keepdim=True)
            p = torch.exp(score - top)
            total = p.sum(dim=-1, keepdim=True)
            out[t + i:t + i + m] = torch.bmm(p / total, v).view(HKV, m, g, D).transpose(0, 1).reshape(m, HQ, D)
            lse[t + i:t + i + m] = (total.log() + top).view(HKV, m, g).transpose(0, 1).reshape(m, HQ)
        t += n
    return out, lse


def _run_fork(state):
    case = state["case"]
    table, counts, parents = state["table"], state["counts"], state["parents"].long()
    B, W = table.shape
    blocks, page = counts.shape[0], case["page"]
    used = state["used"].long()
    column = torch.arange(W, device=table.device)[None, :]
    lives = ((parents >= 0) & (parents < B))[:, None]
    held = (used + page - 1) // page
    rows = torch.where(lives & (column < held[:, None]), table[parents.clamp(0, B - 1)], torch.full_like(table, -1))

    def add(entries, by):  # references of the pages that `entries` names
        valid = (entries >= 0) & (entries < blocks)
        wide = torch.zeros(blocks + 1, dtype=torch.int32, device=table.device)
        index = torch.where(valid, entries, torch.full_like(entries, blocks)).flatten().long()
        counts.add_(wide.index_add_(0, index, torch.full(index.shape, by, dtype=torch.int32, device=table.device))[:blocks])

    add(table, -1)
    add(rows, 1)
    # A page that a row will go on writing to, and that others hold too: all but the lowest row get a page of their own,
    # all of them where somebody holds it who will not write to it.
    at = (used // page).clamp(max=W - 1)
    tail = rows.gather(1, at[:, None])[:, 0]
    tail = torch.where((used % page > 0) & (used < W * page) & (tail < blocks), tail, torch.full_like(tail, -1)).long()
    same = (tail[:, None] == tail[None, :]) & (tail >= 0)[:, None]
    lowest = ~(same & (torch.arange(B, device=table.device)[None, :] < torch.arange(B, device=table.device)[:, None])).any(1)
    alone = counts[tail.clamp(min=0)] == same.sum(1)
    copied = (tail >= 0) & ~(lowest & alone)
    add(torch.where(copied, tail, torch.full_like(tail, -1)).to(torch.int32), -1)
    # The k-th page wanted, row by row, is the k-th free one.
    most = (used + case["reserve"] + page - 1) // page
    fresh = lives & (column >= held[:, None]) & (column < most[:, None])
    want = fresh | (copied[:, None] & (column == at[:, None]))
    kth = (want.flatten().cumsum(0) - 1).view(B, W)
    free = torch.nonzero(counts == 0)[:, 0]
    over = (lives[:, 0].long() * (most - W).clamp(min=0)).sum()  # beyond the table
    given = torch.cat([free, free.new_full((1,), -1)])[kth.clamp(max=free.shape[0])].to(torch.int32)
    table.copy_(torch.where(want, given, rows))
    add(torch.where(want, given, torch.full_like(given, -1)), 1)
    source = torch.where(copied, tail, torch.full_like(tail, -1)).to(torch.int32)
    destination = torch.where(copied, table.gather(1, at[:, None])[:, 0], torch.full_like(table[:, 0], -1))
    missing = ((want & (given < 0)).sum() + over).to(torch.int32).view(1)
    return table, counts, torch.where(destination >= 0, source, destination), destination, missing


def _run_compact(state):
    table, counts = state["table"], state["counts"]
    blocks = counts.shape[0]
    page = torch.arange(blocks, device=table.device)
    in_use = counts > 0
    n = in_use.sum()
    from_, to = torch.nonzero(in_use & (page >= n))[:, 0], torch.nonzero(~in_use & (page < n))[:, 0]
    name = page.clone()
    name[from_] = to
    valid = (table >= 0) & (table < blocks)
    table.copy_(torch.where(valid, name[table.clamp(0, blocks - 1).long()].to(torch.int32), table))
    counts[to] = counts[from_]
    counts[from_] = 0
    source = torch.full((blocks // 2,), -1, dtype=torch.int32, device=table.device)
    destination = source.clone()
    source[:from_.shape[0]], destination[:to.shape[0]] = from_.to(torch.int32), to.to(torch.int32)
    return table, counts, source, destination


def run(state):
    case = state["case"]
    kind = case["kind"]
    if kind == "append":
        if own:
            from ascendflow_amd.sparse_attention import append_quantized_kv

            append_quantized_kv(state["k"], state["v"], state["k_cache"], state["v_cache"], state["k_scale"],
                                state["v_scale"], state["table"], state["cu_q"], state["used"])
        else:
            _append_one(state, state["k"], state["k_cache"], state["k_scale"])
            _append_one(state, state["v"], state["v_cache"], state["v_scale"])
        return state["k_cache"], state["v_cache"], state["k_scale"], state["v_scale"]
    if kind == "attention":
        if not own:
            return _run_attention(state)
        from ascendflow_amd.flash_attention import quantized_attention

        lse = torch.empty(state["q"].shape[:2], dtype=torch.float32, device=state["q"].device)
        out = quantized_attention(state["q"], state["k_cache"], state["v_cache"], state["k_scale"], state["v_scale"],
                                  state["table"], state["cu_q"], state["used"], SCALE=state["scale"], softmax_lse=lse)
        return out, lse
    if kind == "copy":
        if own:
            from ascendflow_amd.sparse_attention import copy_pages

            copy_pages(state["caches"], state["source"], state["destination"])
        else:
            full = (state["source"] >= 0) & (state["destination"] >= 0)
            source, destination = state["source"][full].long(), state["destination"][full].long()
            for cache in state["caches"]:
                part = cache.view(torch.uint8)
                part[destination] = part[source]
        return state["caches"]
    if kind == "fork":
        if not own:
            return _run_fork(state)
        from ascendflow_amd.sparse_attention import fork_pages

        source, destination, missing = fork_pages(state["table"], state["counts"], state["parents"], state["used"],
                                                  PAGE=case["page"], reserve=case["reserve"])
        return state["table"], state["counts"], source, destination, missing
    if not own:
        return _run_compact(state)
    from ascendflow_amd.sparse_attention import compact_pages

    source, destination = compact_pages(state["table"], state["counts"])
    return state["table"], state["counts"], source, destination


# ---- the same in float64, from the definitions ----------------------------------------


def _exact_append(case, state):
    """Request by request and block by block; e4m3 rows before they are rounded, in units of their scales."""
    page, G, HKV, codes = case["page"], case["group"], case["HKV"], case["codes"]
    table = state["table"].cpu().numpy()
    out = []
    for which in ("k", "v"):
        x = state[which].double().cpu().numpy()
        cache = state[which + "_cache"].float().double().cpu().numpy()
        scale = state[which + "_scale"].double().cpu().numpy()
        t = 0
        for b, (n, s) in enumerate(zip(state["counts"], state["lengths"])):
            first = s - n
            for g in range(first // G, (s - 1) // G + 1):
                low, high = max(first, g * G), min(s, (g + 1) * G)
                new = x[t + low - first:t + high - first]
                block, at = table[b, g * G // page], g * G % page
                top = np.maximum(np.abs(new).max(axis=(0, 2)), 2.0 ** LEAST)
                need = np.maximum(np.exp2(np.ceil(np.log2(top / TOP[codes]))), 2.0 ** LEAST)
                had = scale[block, at // G].copy()
                now = np.maximum(need, had) if low > g * G else need
                scale[block, at // G] = now
                cache[block, at:at + low - g * G] *= (had / now)[None, :, None]
                cache[block, at + low - g * G:at + high - g * G] = new / now[None, :, None]
            t += n
        out.append((cache if codes == "e4m3" else None, scale))
    device = state["k"].device
    as_tensor = [None if a is None else torch.from_numpy(a).to(device) for a in (out[0][0], out[1][0], out[0][1], out[1][1])]
    return tuple(as_tensor)


def exact(case, seed):
    kind = case["kind"]
    if kind in ("copy", "fork", "compact"):
        return None
    state = prepare(case, seed)
    if kind == "append":
        return _exact_append(case, state) if sum(_requests(case)[0]) * case["HKV"] * case["D"] <= 1 << 25 else None
    HQ, HKV, D, page, G = case["HQ"], case["HKV"], case["D"], case["page"], case["group"]
    q = state["q"].double()
    out = torch.empty(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.empty(q.shape[:2], dtype=torch.float64, device=q.device)
    t = 0
    for b, (n, s) in enumerate(zip(state["counts"], state["lengths"])):
        position = torch.arange(s, device=q.device)
        block = state["table"][b].long()[position // page]
        for h in range(HKV):
            k = state["k_cache"][block, position % page, h].double() * state["k_scale"][block, position % page // G, h].double()[:, None]
            v = state["v_cache"][block, position % page, h].double() * state["v_scale"][block, position % page // G, h].double()[:, None]
            for j in range(h * (HQ // HKV), (h + 1) * (HQ // HKV)) if n > 1 else (slice(h * (HQ // HKV), (h + 1) * (HQ // HKV)),):
                mine = q[t:t + n, j] if n > 1 else q[t, j]
                score = mine @ k.t() * state["scale"]
                if n > 1:
                    seen = s - n + torch.arange(n, device=q.device)
                    score.masked_fill_(position[None, :] > seen[:, None], -math.inf)
                total = torch.logsumexp(score, dim=1)
                rows = torch.exp_(score.sub_(total[:, None])) @ v
                if n > 1:
                    out[t:t + n, j], lse[t:t + n, j] = rows, total
                else:
                    out[t, j], lse[t, j] = rows, total
        t += n
    return out, lse
