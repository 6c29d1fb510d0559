"""Measured calls of the latent-attention path: rotary positions, append to the paged cache, attention in its two forms.

``listed()`` gives the fixed cases, ``draw(rng)`` another one of the same ranges,
``prepare`` what a serving program has in hand before the call, ``run`` one call,
in the plain form (elementary torch operations in float32) or, where ``own`` is
true, through the framework's entry points, ``exact`` its result in float64.
"""

from __future__ import annotations

import math
import random

import torch

own = False

B16 = {"bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # The smallest call: the queries of one request with five draft tokens at a far position, the last 64 of 512 columns.
        _rotary("rotary_decode_6", T=6, H=64, D=512, R=64, offset=448, start=131000),
        # A prompt's query heads, the 64 rotary columns of 192, scaled for long contexts, as a strided view.
        _rotary("rotary_prompt_8k", T=8192, H=64, D=192, R=64, offset=128, view=True, layout="interleaved", factor=40.0),
        # A training step's forward and gradient over whole heads of an odd length.
        _rotary("rotary_train_1987", T=1987, H=32, D=128, R=128, offset=0, dtype="f16", gradient=True),
        # Batched decode with five draft tokens: latent and rotary key of each token into 64 requests' pages.
        _append("append_decode_64x6", B=64, n=6, context=2000, L=512, R=64, layout="interleaved", split=True),
        # Keys and values of a few unequal prompts, 8 heads, part of each head rotated, views of one projection.
        _append("append_prompt_3x1987", B=3, n=1987, context=2600, HKV=8, L=128, R=64, offset=0, value=128, page=64,
                dtype="f16", ragged=True),
        # One user's single-token step at 4K: latency bound.
        _latent("latent_decode_1x1_4k", B=1, n=1, context=4096),
        # Batched single-token decode of unequal requests with all 128 heads on the GPU.
        _latent("latent_decode_64x1_h128", B=64, n=1, context=8000, H=128, ragged=True),
        # The same step where eight GPUs share the heads: 16 of them, long contexts, bound by the cache's bytes.
        _latent("latent_decode_32x1_h16", B=32, n=1, context=32768, H=16),
        # Verification of five draft tokens a request over cache rows that hold keys and values in all 512 columns.
        _latent("latent_verify_16x6_f16", B=16, n=6, context=16000, R=0, dtype="f16", ragged=True),
        # A chunk of a long prompt over a smaller latent.
        _latent("latent_chunk_1x1000", B=1, n=1000, context=20011, H=32, L=256),
        # A whole prompt, causal, in the expanded form.
        _expanded("expanded_prompt_8k", B=1, nq=8192, nk=8192, H=32),
        # Ragged chunks behind earlier context on a small f16 model.
        _expanded("expanded_5x470_f16", B=5, nq=470, nk=2000, H=16, dtype="f16", ragged=True),
    ]


def _rotary(name, *, T, H, D, R, offset, start=0, layout="half", factor=1.0, dtype="bf16", view=False, gradient=False):
    return {"name": name, "kind": "rotary", "T": T, "H": H, "D": D, "R": R, "offset": offset, "start": start,
            "layout": layout, "factor": factor, "dtype": dtype, "view": view, "gradient": gradient}


def _append(name, *, B, n, context, L, R, HKV=1, layout="half", split=False, offset=0, value=0, page=128, dtype="bf16",
            ragged=False):
    return {"name": name, "kind": "append", "B": B, "n": n, "context": context, "HKV": HKV, "L": L, "R": R,
            "layout": layout, "split": split, "offset": offset, "value": value, "page": page, "dtype": dtype,
            "ragged": ragged}


def _latent(name, *, B, n, context, H=64, L=512, R=64, page=128, dtype="bf16", ragged=False):
    return {"name": name, "kind": "latent", "B": B, "n": n, "context": context, "H": H, "L": L, "R": R, "page": page,
            "dtype": dtype, "ragged": ragged}


def _expanded(name, *, B, nq, nk, H, dtype="bf16", causal=True, ragged=False):
    return {"name": name, "kind": "expanded", "B": B, "nq": nq, "nk": nk, "H": H, "dtype": dtype, "causal": causal,
            "ragged": ragged}


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(max(low, high))))))


def draw(rng):
    kind = rng.choice(["rotary", "append", "latent", "latent", "latent", "expanded", "expanded"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if kind == "rotary":
        H = rng.choice([1, 8, 16, 32, 64, 128])
        D, R, offset = rng.choice([(512, 64, 448), (192, 64, 128), (128, 128, 0), (128, 64, 0), (64, 64, 0)])
        T = _log_int(rng, 1, min(131072, 8192 * 64 * 192 // (H * D)))
        view = offset > 0 and rng.random() < 0.5
        case = _rotary("", T=T, H=H, D=D, R=R, offset=offset, start=_log_int(rng, 1, 1000000), dtype=dtype, view=view,
                       layout=rng.choice(["half", "interleaved"]), factor=rng.choice([1.0, 4.0, 40.0]),
                       gradient=rng.random() < 0.3)
    elif kind == "append":
        B = _log_int(rng, 1, 128)
        n = _log_int(rng, 1, 8 if rng.random() < 0.5 else max(8, 8192 // B))
        context = min(_log_int(rng, 2 * n, 8 * n + 2000), max(2 * n, 200000 // B))
        if rng.random() < 0.5:
            L = rng.choice([512, 512, 256])
            case = _append("", B=B, n=n, context=context, L=L, R=64, split=True)
        else:
            D = rng.choice([64, 128, 128])
            R = rng.choice([D // 2, D])
            case = _append("", B=B, n=n, context=context, L=D, R=R, HKV=rng.choice([1, 2, 8]), value=D,
                           offset=rng.choice([0, D - R]))
        case.update(dtype=dtype, page=rng.choice([16, 64, 128]), layout=rng.choice(["half", "interleaved"]),
                    ragged=rng.random() < 0.6)
    elif kind == "latent":
        H = rng.choice([8, 16, 32, 64, 64, 128, 128])
        L, R = rng.choice([(512, 64), (512, 64), (512, 64), (512, 0), (256, 64)])
        B = _log_int(rng, 1, 128)
        n = 1 if rng.random() < 0.5 else _log_int(rng, 2, 8 if rng.random() < 0.6 else max(8, 2000 // B))
        # At most the cache bytes and the products of the largest listed cases.
        context = min(_log_int(rng, max(100, 2 * n), 131072), 1400000 // B, int(6e11 / (2 * H * (2 * L + R) * B * n)))
        case = _latent("", B=B, n=n, context=max(2 * n, context), H=H, L=L, R=R, page=rng.choice([16, 64, 128, 128]),
                       dtype=dtype, ragged=rng.random() < 0.6)
    else:
        H = rng.choice([4, 8, 16, 32, 64, 128])
        B = _log_int(rng, 1, 16)
        nk = _log_int(rng, 64, 8192)
        nq = nk if rng.random() < 0.6 else _log_int(rng, 1, nk)
        B = max(1, min(B, int(1.2e12 / (2 * H * 320 * nq * nk * 1.5))))
        H = H if 2 * H * 320 * nq * nk * B < 1.4e12 else 8
        case = _expanded("", B=B, nq=nq, nk=nk, H=H, dtype=dtype, causal=rng.random() < 0.7, ragged=rng.random() < 0.6)
    del case["name"]
    return case


# ---- sizes -----------------------------------------------------------------------


def _requests(case):
    """(new tokens, length with them) of each request; the same for every seed."""
    B, n, length = (case["B"], case["n"], case["context"]) if "n" in case else (case["B"], case["nq"], case["nk"])
    if not case["ragged"]:
        return [n] * B, [length] * B
    rng = random.Random(B * 1000003 + n * 1009 + length)
    counts = [max(1, rng.randint(n // 2, n)) for _ in range(B)]
    return counts, [max(c, rng.randint(length // 2, length)) for c in counts]


def _visible(count, length, causal=True):
    """(token, key) pairs of one request."""
    return count * length - (count * (count - 1) // 2 if causal else 0)


def work(case):
    kind = case["kind"]
    if kind == "rotary":
        T, H, R = case["T"], case["H"], case["R"]
        columns = R if case["view"] else case["D"]
        passes = 2 if case["gradient"] else 1
        return {"bytes": passes * (4 * T * H * columns + 8 * T + 4 * R), "flops": passes * 3 * T * H * R}
    if kind == "append":
        counts, _ = _requests(case)
        T = sum(counts)
        row = case["L"] + (case["R"] if case["split"] else 0) + case["value"]
        pages = sum(c // case["page"] + 1 for c in counts)
        return {"bytes": 4 * T * case["HKV"] * row + 4 * pages + 8 * case["B"] + 4 * case["R"],
                "flops": 3 * T * case["HKV"] * case["R"]}
    counts, lengths = _requests(case)
    T, H = sum(counts), case["H"]
    if kind == "latent":
        L, R = case["L"], case["R"]
        pairs = sum(_visible(c, s) for c, s in zip(counts, lengths))
        keys = sum(lengths)
        return {"bytes": 2 * keys * (L + R) + 2 * T * H * (2 * L + R) + 4 * T * H, "flops": 2 * H * (2 * L + R) * pairs}
    pairs = sum(_visible(c, s, case["causal"]) for c, s in zip(counts, lengths))
    keys = sum(lengths)
    return {"bytes": 2 * T * H * (192 + 128) + 2 * keys * (H * 256 + 64) + 4 * T * H, "flops": 2 * H * 320 * pairs}


# ---- inputs ----------------------------------------------------------------------


def _frequencies(R, factor, device):
    """Radians per position of each pair: base 10000, scaled by parts for ``factor`` times a context of 4096."""
    plain = 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / R)
    if factor != 1.0:
        turn = [R * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(10000.0)) for turns in (32.0, 1.0)]
        low, high = max(0, math.floor(turn[0])), min(R - 1, math.ceil(turn[1]))
        ramp = ((torch.arange(R // 2, dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0, 1)
        plain = plain / factor * ramp + plain * (1 - ramp)
    return plain.to(device)


def _offsets(counts, device):
    total = [0]
    for c in counts:
        total.append(total[-1] + c)
    return torch.tensor(total, dtype=torch.int32, device=device)


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device)
    gen.manual_seed(seed)
    kind, b16 = case["kind"], B16[case["dtype"]]

    def normal(*shape):
        out = torch.empty(shape, dtype=b16, device=device)
        flat = out.view(-1)
        for i in range(0, flat.numel(), 1 << 28):  # bounded float32 temporaries
            part = flat[i:i + (1 << 28)]
            part.copy_(torch.randn(part.numel(), generator=gen, device=device))
        return out

    state = {"case": case}
    if kind == "rotary":
        T, H, D, R = case["T"], case["H"], case["D"], case["R"]
        x = normal(T, H, D)
        state["x"] = x[..., case["offset"]:case["offset"] + R] if case["view"] else x
        state["offset"] = 0 if case["view"] else case["offset"]
        first = torch.randint(0, case["start"] + 1, (1,), generator=gen, device=device)
        state["positions"] = (first + torch.arange(T, device=device)).to(torch.int32)
        state["frequencies"] = _frequencies(R, case["factor"], device)
        state["magnitude"] = 1.0 if case["factor"] == 1.0 else 0.1 * math.log(case["factor"]) + 1.0
        if case["gradient"]:
            state["x"] = state["x"].detach().requires_grad_(True)
            state["grad"] = normal(*state["x"].shape)
        return state

    counts, lengths = _requests(case)
    T = sum(counts)
    state["counts"], state["lengths"] = counts, lengths
    state["cu_q"] = _offsets(counts, device)
    if kind == "expanded":
        H, K = case["H"], sum(lengths)
        state["cu_k"] = _offsets(lengths, device)
        state["q"] = normal(T, H, 192)
        expanded = normal(K, H, 256)  # one projection of the latents: keys, then values
        state["k"], state["v"] = expanded[..., :128], expanded[..., 128:]
        state["k_rope"] = normal(K, 64)
        return state

    page = case["page"]
    pages = [-(-s // page) for s in lengths]
    width = max(pages)
    order = torch.randperm(sum(pages), generator=gen, device=device).to(torch.int32).cpu()
    table = torch.zeros((case["B"], width), dtype=torch.int32)
    at = 0
    for b, p in enumerate(pages):
        table[b, :p] = order[at:at + p]
        at += p
    state["table"] = table.to(device)
    state["used"] = torch.tensor(lengths, dtype=torch.int32, device=device)
    if kind == "append":
        HKV, L, R = case["HKV"], case["L"], case["R"]
        state["frequencies"] = _frequencies(R, 1.0, device)
        if case["split"]:
            both = normal(T, HKV, L + R)  # one projection: the latent, then the rotary key
            state["k"], state["rope"] = both[..., :L], both[..., L:]
            state["k_cache"] = torch.zeros((sum(pages), page, HKV, L + R), dtype=b16, device=device)
        else:
            both = normal(T, 2, HKV, L)
            state["k"], state["v"] = both[:, 0], both[:, 1]
            state["k_cache"] = torch.zeros((sum(pages), page, HKV, L), dtype=b16, device=device)
            state["v_cache"] = torch.zeros((sum(pages), page, HKV, L), dtype=b16, device=device)
        return state
    H, L, R = case["H"], case["L"], case["R"]
    state["cache"] = normal(sum(pages), page, 1, L + R)
    q = normal(T, H, L + R)
    state["q"], state["q_rope"] = q[..., :L], (q[..., L:] if R else None)
    state["scale"] = 192 ** -0.5 if R else 512 ** -0.5
    return state


# ---- one call ----------------------------------------------------------------------


def _rotate(x, positions, frequencies, layout, magnitude=1.0, inverse=False, wide=torch.float32):
    """x [T, H, R] rotated, in ``wide``; the angles of far positions need 64 bits."""
    angle = positions.double()[:, None, None] * frequencies
    cos, sin = (magnitude * angle.cos()).to(wide), (magnitude * angle.sin()).to(wide)
    sin = -sin if inverse else sin
    x = x.to(wide)
    half = x.shape[-1] // 2
    a, b = (x[..., :half], x[..., half:]) if layout == "half" else (x[..., 0::2], x[..., 1::2])
    y = (a * cos - b * sin, a * sin + b * cos)
    return torch.cat(y, dim=-1) if layout == "half" else torch.stack(y, dim=-1).flatten(-2)


def _run_rotary(state, x, inverse=False):
    case = state["case"]
    at, R = state["offset"], case["R"]
    y = x.clone()
    y[..., at:at + R] = _rotate(x[..., at:at + R], state["positions"], state["frequencies"], case["layout"],
                                state["magnitude"], inverse).to(x.dtype)
    return y


def _slots(state):
    """(position, cache row) of each new token."""
    cu, used, page = state["cu_q"].long(), state["used"].long(), state["case"]["page"]
    token = torch.arange(state["k"].shape[0], device=cu.device)
    request = torch.searchsorted(cu[1:], token, right=True)
    position = used[request] - cu[request + 1] + token
    return position, state["table"][request, position // page].long() * page + position % page


def _run_append(state):
    case = state["case"]
    position, slot = _slots(state)
    R, L = case["R"], case["L"]
    keys = state["k_cache"].flatten(0, 1)
    if case["split"]:
        keys[slot, :, :L] = state["k"]
        keys[slot, :, L:] = _rotate(state["rope"], position, state["frequencies"], case["layout"]).to(keys.dtype)
        return state["k_cache"]
    at = case["offset"]
    k = state["k"].clone()
    k[..., at:at + R] = _rotate(k[..., at:at + R], position, state["frequencies"], case["layout"]).to(k.dtype)
    keys[slot] = k
    state["v_cache"].flatten(0, 1)[slot] = state["v"]
    return state["k_cache"], state["v_cache"]


def _softmax_rows(s, hidden):
    """(weights, log of the sum) of scores s with the entries ``hidden`` left out; a row with none left has weights 0."""
    if hidden is not None:
        s = s.masked_fill(hidden, -math.inf)
    top = s.amax(dim=-1, keepdim=True).clamp(min=-1e30)
    p = torch.exp(s - top)
    total = p.sum(dim=-1, keepdim=True)
    return p / total.clamp(min=1e-30), (total.log() + top)[..., 0]


def _run_latent(state):
    case = state["case"]
    H, L, R, page = case["H"], case["L"], case["R"], case["page"]
    T = state["q"].shape[0]
    out = torch.empty((T, H, L), dtype=state["q"].dtype, device=state["q"].device)
    lse = torch.empty((T, H), dtype=torch.float32, device=out.device)
    t = 0
    for b, (n, s) in enumerate(zip(state["counts"], state["lengths"])):
        rows = state["cache"][state["table"][b, :-(-s // page)].long()].view(-1, L + R)[:s].float()
        key = torch.arange(s, device=out.device)
        step = max(1, (1 << 29) // (H * s))
        for i in range(0, n, step):
            m = min(step, n - i)
            q = state["q"][t + i:t + i + m].float()
            if R:
                q = torch.cat([q, state["q_rope"][t + i:t + i + m].float()], dim=-1)
            score = (q.reshape(m * H, L + R) @ rows.t()) * state["scale"]
            last = torch.arange(s - n + i, s - n + i + m, device=out.device).repeat_interleave(H)[:, None]
            p, total = _softmax_rows(score, key > last if n > 1 else None)
            out[t + i:t + i + m] = (p @ rows[:, :L]).view(m, H, L)
            lse[t + i:t + i + m] = total.view(m, H)
        t += n
    return out, lse


def _run_expanded(state):
    case = state["case"]
    H = case["H"]
    out = torch.empty((state["q"].shape[0], H, 128), dtype=state["q"].dtype, device=state["q"].device)
    lse = torch.empty(out.shape[:2], dtype=torch.float32, device=out.device)
    t = u = 0
    for n, s in zip(state["counts"], state["lengths"]):
        rope = state["k_rope"][u:u + s].float()
        hidden = None
        if case["causal"]:
            last = torch.arange(s - n, s, device=out.device)[:, None]
            hidden = torch.arange(s, device=out.device) > last
        for h in range(H):
            k = torch.cat([state["k"][u:u + s, h].float(), rope], dim=-1)
            score = (state["q"][t:t + n, h].float() @ k.t()) * 192 ** -0.5
            p, total = _softmax_rows(score, hidden)
            out[t:t + n, h] = (p @ state["v"][u:u + s, h].float()).to(out.dtype)
            lse[t:t + n, h] = total
        t, u = t + n, u + s
    return out, lse


def run(state):
    case = state["case"]
    kind = case["kind"]
    if kind == "rotary":
        if own:
            from ascendflow_amd.sparse_attention import apply_rotary

            y = apply_rotary(state["x"], state["positions"], state["frequencies"], layout=case["layout"],
                             offset=state["offset"], magnitude=state["magnitude"])
            return (y, torch.autograd.grad(y, state["x"], state["grad"])[0]) if case["gradient"] else y
        if case["gradient"]:
            return _run_rotary(state, state["x"].detach()), _run_rotary(state, state["grad"], inverse=True)
        return _run_rotary(state, state["x"])
    if kind == "append":
        if not own:
            return _run_append(state)
        from ascendflow_amd.sparse_attention import append_paged_kv

        args = (state["k"], state["k_cache"], state["table"], state["cu_q"], state["used"])
        if case["split"]:
            append_paged_kv(*args, rope=state["rope"], frequencies=state["frequencies"], layout=case["layout"])
            return state["k_cache"]
        append_paged_kv(*args, v=state["v"], v_cache=state["v_cache"], frequencies=state["frequencies"],
                        layout=case["layout"], offset=case["offset"])
        return state["k_cache"], state["v_cache"]
    if kind == "latent":
        if not own:
            return _run_latent(state)
        from ascendflow_amd.sparse_attention import latent_attention

        lse = torch.empty(state["q"].shape[:2], dtype=torch.float32, device=state["q"].device)
        out = latent_attention(state["q"], state["cache"], state["table"], state["cu_q"], state["used"],
                               q_rope=state["q_rope"], SCALE=state["scale"], softmax_lse=lse)
        return out, lse
    if not own:
        return _run_expanded(state)
    from ascendflow_amd.flash_attention import latent_attention_expanded

    lse = torch.empty(state["q"].shape[:2], dtype=torch.float32, device=state["q"].device)
    out = latent_attention_expanded(state["q"], state["k"], state["k_rope"], state["v"], state["cu_q"], state["cu_k"],
                                    SCALE=192 ** -0.5, CAUSAL=case["causal"], softmax_lse=lse)
    return out, lse


# ---- the same in float64, from the definitions ----------------------------------------


def _turned(x, position, frequencies, layout, magnitude):
    """Each pair (u, v) as the complex number u + iv times magnitude e^(i angle)."""
    x = x.double()
    half = x.shape[-1] // 2
    z = torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous()) if layout == "half" else \
        torch.view_as_complex(x.reshape(*x.shape[:-1], half, 2).contiguous())
    angle = position.double().view(-1, 1, 1) * frequencies
    z = z * torch.polar(torch.full_like(angle, magnitude), angle)
    return torch.cat([z.real, z.imag], dim=-1) if layout == "half" else torch.view_as_real(z).flatten(-2)


def _exact_append(case, state):
    R, L, page = case["R"], case["L"], case["page"]
    key = state["k_cache"].double()
    value = state["v_cache"].double() if case["value"] else None
    t = 0
    for b, (n, s) in enumerate(zip(state["counts"], state["lengths"])):
        position = torch.arange(s - n, s, device=key.device)
        block, slot = state["table"][b].long()[position // page], position % page
        row = state["k"][t:t + n].double()
        if case["split"]:
            row = torch.cat([row, _turned(state["rope"][t:t + n], position, state["frequencies"], case["layout"], 1.0)], -1)
        else:
            at = case["offset"]
            row[..., at:at + R] = _turned(row[..., at:at + R], position, state["frequencies"], case["layout"], 1.0)
            value[block, slot] = state["v"][t:t + n].double()
        key[block, slot] = row
        t += n
    return key if case["split"] else (key, value)


def _attend(q, k, v, scale, first):
    """softmax(q k^T scale) v in float64; query row i sees keys up to first + i, or all of them where first is None."""
    s = torch.matmul(q, k.t()) * scale
    if first is not None:
        rows = first + torch.arange(q.shape[0], device=q.device)
        s.masked_fill_(torch.arange(k.shape[0], device=q.device)[None, :] > rows[:, None], -math.inf)
    total = torch.logsumexp(s, dim=1)
    return torch.exp_(s.sub_(total[:, None])) @ v, total


def exact(case, seed):
    kind = case["kind"]
    state = prepare(case, seed)
    if kind == "rotary":
        at, R = state["offset"], case["R"]

        def turned(x, position):
            y = x.detach().double().clone()
            y[..., at:at + R] = _turned(y[..., at:at + R], position, state["frequencies"], case["layout"],
                                        state["magnitude"])
            return y

        y = turned(state["x"], state["positions"])
        return (y, turned(state["grad"], -state["positions"])) if case["gradient"] else y
    if kind == "append":
        return _exact_append(case, state)
    H = case["H"]
    q = state["q"]
    width = case["L"] if kind == "latent" else 128
    out = torch.empty((q.shape[0], H, width), dtype=torch.float64, device=q.device)
    lse = torch.empty((q.shape[0], H), dtype=torch.float64, device=q.device)
    t = u = 0
    for b, (n, s) in enumerate(zip(state["counts"], state["lengths"])):
        if kind == "latent":
            position = torch.arange(s, device=q.device)
            rows = state["cache"][state["table"][b].long()[position // case["page"]], position % case["page"], 0].double()
            if n == 1:  # all heads at once
                whole = q[t] if state["q_rope"] is None else torch.cat([q[t], state["q_rope"][t]], dim=-1)
                out[t], lse[t] = _attend(whole.double(), rows, rows[:, :width], state["scale"], None)
                t += n
                continue
        for h in range(H):
            if kind == "latent":
                mine = q[t:t + n, h] if state["q_rope"] is None else torch.cat([q[t:t + n, h], state["q_rope"][t:t + n, h]], -1)
                part = _attend(mine.double(), rows, rows[:, :width], state["scale"], s - n)
            else:
                keys = torch.cat([state["k"][u:u + s, h], state["k_rope"][u:u + s]], dim=-1).double()
                part = _attend(q[t:t + n, h].double(), keys, state["v"][u:u + s, h].double(), 192 ** -0.5,
                               s - n if case["causal"] else None)
            out[t:t + n, h], lse[t:t + n, h] = part
        t, u = t + n, u + s
    return out, lse
