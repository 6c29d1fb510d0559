"""Definitions of the 8-bit paged cache: the codes and scales of an append, attention over them in float64, and the upkeep of
pages, all written as plain loops over requests, blocks and pages."""

from __future__ import annotations

import math

import numpy as np
import torch

from . import latent_reference as lr

TOP = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def e4m3_values():
    """The finite magnitudes of e4m3 by code 0 .. 126: exponent bits 1 .. 15 of bias 7 with three bits, and the subnormals."""
    return np.array([(m / 8) * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7) for e in range(16) for m in range(8)][:127])


def nearest(x, dtype):
    """float64 values rounded to the values of codes: to nearest, ties to the even code, held inside the range."""
    x = np.asarray(x, dtype=np.float64)
    top = TOP[dtype]
    if dtype == torch.int8:
        return np.rint(np.clip(np.where(np.isnan(x), 0.0, x), -top, top))
    table = e4m3_values()
    a = np.minimum(np.abs(np.where(np.isnan(x), 0.0, x)), top)
    high = np.searchsorted(table, a)                 # first value at or above
    low = np.maximum(high - 1, 0)
    below, above = a - table[low], table[high] - a
    code = np.where((below < above) | ((below == above) & (low % 2 == 0)), low, high)
    return np.where(np.isnan(x), np.nan, np.copysign(table[code], x))


def needed_scale(rows, dtype):
    """2^max(ceil(log2(A / C)), -80), A the largest finite magnitude of rows: by doubling, without a logarithm."""
    a = np.abs(rows[np.isfinite(rows)])
    top = a.max() if a.size else 0.0
    s = 2.0 ** -80
    while top > s * TOP[dtype]:
        s *= 2
    return s


def append(x, cache, scale, table, cu, used):
    """New rows x [T, HKV, D] into values of codes ``cache`` [BLOCKS, PAGE, HKV, D] (float64 numpy, in place; codes of type
    ``dtype``) and ``scale`` [BLOCKS, S, HKV]; ``cache`` is (array, dtype)."""
    codes, dtype = cache
    blocks, page, HKV, _ = codes.shape
    G = page // scale.shape[1]
    x = x.double().numpy()
    for b in range(table.shape[0]):
        touched = {}
        for t, _, block, slot in lr.rows_of(cu, used, table, page, blocks, b):
            touched.setdefault((block, slot // G), []).append((slot % G, t))
        for (block, part), rows in touched.items():
            first = min(slot for slot, _ in rows)
            for h in range(HKV):
                new = np.stack([x[t, h] for _, t in rows])
                s, had = needed_scale(new, dtype), float(scale[block, part, h])
                if first > 0:
                    s = max(s, had)
                    if s != had:
                        old = slice(part * G, part * G + first)
                        codes[block, old, h] = nearest(codes[block, old, h] * had / s, dtype)
                for (slot, _), row in zip(rows, new):
                    codes[block, part * G + slot, h] = nearest(row / s, dtype)
                scale[block, part, h] = s


def values(codes, scale):
    """What codes [BLOCKS, PAGE, HKV, D] with scales [BLOCKS, S, HKV] stand for, float64."""
    G = codes.shape[1] // scale.shape[1]
    return codes.float().double() * scale.double().repeat_interleave(G, dim=1)[..., None]


def attention(q, k, v, table, cu, used, scale, causal=True):
    """(out, lse, spread, reach) over caches of float64 values k and v [BLOCKS, PAGE, HKV, D]; tokens of no request are NaN."""
    T, HQ, D = q.shape
    blocks, page, HKV, _ = k.shape
    result = lr._empty(T, HQ, D, q.device)
    for b in range(table.shape[0]):
        start, end = int(cu[b]), int(cu[b + 1])
        n, length = end - start, max(0, int(used[b]))
        s = min(length, table.shape[1] * page)
        if n == 0:
            continue
        ids = table[b].tolist()
        there = [j for j in range(s) if 0 <= ids[j // page] < blocks]
        block = torch.tensor([ids[j // page] for j in there], dtype=torch.long, device=q.device)
        slot = torch.tensor([j % page for j in there], dtype=torch.long, device=q.device)
        limit = [sum(1 for j in there if j < (length - n + i + 1 if causal else s)) for i in range(n)]
        keys, rows = (x[block, slot].repeat_interleave(HQ // HKV, dim=1) for x in (k, v))
        for whole, piece in zip(result, lr._attend(q[start:end].double(), keys, rows, scale, limit)):
            whole[start:end] = piece
    return result


def attention_bound(out, spread, reach, dtype, keys, largest, exponents):
    """``latent_reference.attention_bound`` and what the scales add. The exponent of a weight is fma(s, a, log2 b - m): the
    logarithm is off by a step of 2^-23 |log2 b| and the two roundings by 2^-24 (reach + 2 |log2 b|) more, with
    |log2 b| <= ``exponents``: together under 8 2^-24 (reach + exponents), of which w moves by as much and out, whose
    denominator takes b itself, by that of spread + |out|. ``largest``: the largest code times the largest value scale,
    against which float16's weights below 2^-14 are rounded (the weight that contributes most is at least 1 in units of its
    own scale)."""
    more = 2 * 8 * 2.0 ** -24 * (reach[..., None] + exponents) * (spread + out.abs())
    return lr.attention_bound(out, spread, reach, dtype, keys, largest) + more * (1 + 1e-2)


def fork(table, counts, parents, used, page, reserve):
    """(table, counts, source, destination, missing) as lists; ``missing`` counts entries wanted and not had."""
    B, W, blocks = len(table), len(table[0]), len(counts)
    valid = lambda e: 0 <= e < blocks
    counts = list(counts)
    rows = []
    for b in range(B):
        held = -(-max(used[b], 0) // page)
        lives = 0 <= parents[b] < B
        rows.append([table[parents[b]][c] if lives and c < held else -1 for c in range(W)])
    for row in table:
        for e in row:
            if valid(e):
                counts[e] -= 1
    for row in rows:
        for e in row:
            if valid(e):
                counts[e] += 1
    writers = {}  # page: rows that will go on writing to it
    for b in range(B):
        if 0 <= parents[b] < B and used[b] > 0 and used[b] % page and used[b] // page < W and valid(rows[b][used[b] // page]):
            writers.setdefault(rows[b][used[b] // page], []).append(b)
    copied = {}
    for e, mine in writers.items():
        for b in mine[1:] if counts[e] == len(mine) else mine:
            copied[b] = e
    for e in copied.values():
        counts[e] -= 1
    free = [p for p in range(blocks) if counts[p] == 0]
    source, destination, missing = [-1] * B, [-1] * B, 0
    for b in range(B):
        if not 0 <= parents[b] < B:
            continue
        length = max(used[b], 0)
        held, most = -(-length // page), -(-(length + reserve) // page)
        wanted = ([held - 1] if b in copied else []) + list(range(held, min(most, W)))
        missing += max(0, most - W)  # beyond the table
        for c in wanted:
            got = free.pop(0) if free else -1
            rows[b][c] = got
            if got >= 0:
                counts[got] = 1
            else:
                missing += 1
            if b in copied and c == held - 1 and got >= 0:
                source[b], destination[b] = copied[b], got
    return rows, counts, source, destination, min(missing, 2**31 - 1)


def compact(table, counts):
    """(table, counts, moves) as lists."""
    counts = list(counts)
    n = sum(c > 0 for c in counts)
    moves = list(zip([p for p in range(n, len(counts)) if counts[p] > 0], [p for p in range(n) if counts[p] <= 0]))
    name = dict(moves)
    for a, b in moves:
        counts[a], counts[b] = 0, counts[a]
    return [[name.get(e, e) for e in row] for row in table], counts, moves


__all__ = ["append", "attention", "attention_bound", "compact", "e4m3_values", "fork", "needed_scale", "nearest", "values"]
assert math.isclose(e4m3_values()[-1], 448.0)
