"""Cases, plain forms and 64-bit definitions of the serving operators beside sdpa: rotary
positions on q and k, the write into a paged 8-bit key/value cache, and attention over that
cache.

With ``own`` false, ``run`` computes an operator from elementary torch operations in 32 bits;
with ``own`` true it makes the calls a user makes of tiledattention_b200.

The cache: pages [P, Hkv, page, D] of float8_e4m3fn for keys and for values, with one float32
scale, a power of two, for each (page, head). A sequence's token i lives in page
page_table[b, i // page] at row i % page.
"""

import math

import torch

own = False

E4M3_MAX = 448.0
# Scale exponents are held in this range, so that products of scales stay far from the ends
# of float32.
SCALE_EXP_MIN, SCALE_EXP_MAX = -50, 50

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------------------ the cases


def listed():
    return [
        # One decoding step's rotation: a batch of single tokens at far positions, with the
        # frequencies of a long-context scaling.
        {"name": "rotary decode b32", "op": "rotary", "batch": 32, "heads": 32, "kv_heads": 8,
         "tokens": 1, "dim": 128, "rotary_dim": 128, "interleaved": False, "dtype": "bf16",
         "scaling": "yarn", "far": 1 << 20, "grad": False},
        # The prefill configuration of the attention benchmark (B=8, H=32, S=4096, D=128).
        {"name": "rotary prefill 8x4096", "op": "rotary", "batch": 8, "heads": 32,
         "kv_heads": 32, "tokens": 4096, "dim": 128, "rotary_dim": 128, "interleaved": False,
         "dtype": "bf16", "scaling": "none", "far": 0, "grad": False},
        # Part of each head rotated, neighbouring pairs, an odd number of tokens, fp16.
        {"name": "rotary partial interleaved", "op": "rotary", "batch": 3, "heads": 20,
         "kv_heads": 5, "tokens": 1777, "dim": 80, "rotary_dim": 32, "interleaved": True,
         "dtype": "fp16", "scaling": "linear", "far": 30000, "grad": False},
        # A training step's rotation: outputs and the gradients of q and k.
        {"name": "rotary train 4x2048", "op": "rotary", "batch": 4, "heads": 32, "kv_heads": 8,
         "tokens": 2048, "dim": 128, "rotary_dim": 128, "interleaved": False, "dtype": "bf16",
         "scaling": "none", "far": 0, "grad": True},
        # One decoding step's write: one token for each of 64 sequences, wherever its page is.
        {"name": "append decode b64", "op": "append", "batch": 64, "kv_heads": 8, "tokens": 1,
         "dim": 128, "page": 64, "context": 4096, "ragged": False, "dtype": "bf16"},
        # Prompts of different lengths written in one padded batch.
        {"name": "append prompts 8x4096", "op": "append", "batch": 8, "kv_heads": 8,
         "tokens": 4096, "dim": 128, "page": 64, "context": 0, "ragged": True, "dtype": "bf16"},
        # A chunk that begins inside a page; small pages, an odd head dim, fp16.
        {"name": "append odd chunk", "op": "append", "batch": 5, "kv_heads": 3, "tokens": 333,
         "dim": 80, "page": 16, "context": 1001, "ragged": False, "dtype": "fp16"},
        # The smallest decoding step: one short sequence, where latency counts.
        {"name": "decode b1 777", "op": "attend", "batch": 1, "heads": 8, "kv_heads": 2,
         "tokens": 1, "dim": 64, "page": 16, "length": 777, "ragged": False, "dtype": "fp16",
         "lse": False},
        # A serving batch of uneven lengths with an unused last row.
        {"name": "decode b32 ragged 4096", "op": "attend", "batch": 32, "heads": 32,
         "kv_heads": 8, "tokens": 1, "dim": 128, "page": 64, "length": 4096, "ragged": True,
         "dtype": "bf16", "lse": True},
        # The largest: long contexts in a large batch, bound by the cache's bytes.
        {"name": "decode b64 16384", "op": "attend", "batch": 64, "heads": 64, "kv_heads": 8,
         "tokens": 1, "dim": 128, "page": 64, "length": 16384, "ragged": False,
         "dtype": "bf16", "lse": False},
        # A few drafted tokens checked at once; head dim 256.
        {"name": "verify 5 tokens d256", "op": "attend", "batch": 8, "heads": 16, "kv_heads": 4,
         "tokens": 5, "dim": 256, "page": 32, "length": 2999, "ragged": False, "dtype": "fp16",
         "lse": False},
        # A prompt's chunk against the context before it.
        {"name": "chunk 1024 of 8192", "op": "attend", "batch": 2, "heads": 32, "kv_heads": 8,
         "tokens": 1024, "dim": 128, "page": 128, "length": 8192, "ragged": False,
         "dtype": "bf16", "lse": False},
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("rotary", "append", "attend", "attend"))
    kv_heads = rng.choice((1, 2, 3, 4, 5, 8))
    case = {"op": op, "kv_heads": kv_heads, "dtype": rng.choice(("bf16", "fp16"))}
    if op == "rotary":
        dim = rng.choice((64, 80, 96, 128, 192, 256))
        case.update(heads=kv_heads * rng.choice((1, 2, 4, 6)), dim=dim,
                    rotary_dim=rng.choice((dim, dim, dim // 2, 32)),
                    interleaved=rng.random() < 0.4, grad=rng.random() < 0.3,
                    scaling=rng.choice(("none", "linear", "ntk", "yarn")),
                    far=rng.choice((0, 5000, 1 << 17, 1 << 20)), batch=_log(rng, 1, 64))
        row = case["batch"] * (case["heads"] + kv_heads) * dim
        case["tokens"] = _log(rng, 1, max(1, min(8192, (120 << 20) // row)))
        return case
    case.update(batch=_log(rng, 1, 64), dim=rng.choice((64, 64, 80, 96, 128, 128, 192, 256)),
                page=rng.choice((16, 32, 64, 128)), ragged=rng.random() < 0.5)
    row = case["batch"] * kv_heads * case["dim"]
    if op == "append":
        case["tokens"] = 1 if rng.random() < 0.4 else _log(rng, 2, max(2, min(6000, (30 << 20) // row)))
        case["context"] = rng.choice((0, _log(rng, 1, 5000)))
        return case
    group = rng.choice((1, 2, 4, 5, 8, 16))
    kind = rng.choice(("one", "one", "few", "chunk"))
    case.update(heads=kv_heads * group, lse=rng.random() < 0.5)
    if kind == "chunk":
        case["batch"] = _log(rng, 1, 4)
        case["tokens"] = _log(rng, 17, 1500)
        row = case["batch"] * case["heads"] * case["tokens"] * case["dim"]
        case["length"] = case["tokens"] + _log(rng, 1, max(2, min(9000, (40 << 30) // row)))
    else:
        case["tokens"] = 1 if kind == "one" else rng.randint(2, 16)
        case["length"] = case["tokens"] + _log(rng, 1, max(2, min(40000, (200 << 20) // row)))
    return case


def _lengths(case):
    """Tokens in the cache for each sequence once this call's tokens are written, and how many
    of them this call brings."""
    batch, tokens = case["batch"], case["tokens"]
    if case["op"] == "append":
        if not case["ragged"]:
            return [case["context"] + tokens] * batch, [tokens] * batch
        counts = [1 + (tokens - 1) * ((7 * b + 3) % batch) // max(1, batch - 1) for b in range(batch)]
        return [c + case["context"] * ((3 * b + 1) % batch + 1) // batch for b, c in enumerate(counts)], counts
    if not case["ragged"]:
        return [case["length"]] * batch, [tokens] * batch
    lengths = [tokens + (case["length"] - tokens) * ((7 * b + 3) % batch + 1) // batch
               for b in range(batch)]
    counts = [1 + (5 * b) % tokens for b in range(batch)]
    if batch > 8:  # an unused row of the batch
        lengths[-1], counts[-1] = 0, 0
    return lengths, counts


# ------------------------------------------------------------------------------ the inputs


def _inverse_frequencies(rotary_dim, scaling):
    """Radians per position of each pair, in 64 bits, and the factor on cos and sin."""
    i = torch.arange(rotary_dim // 2, dtype=torch.float64)
    base, factor, original = 10000.0, 8.0, 8192.0
    if scaling == "ntk":
        base *= factor ** (rotary_dim / max(1.0, rotary_dim - 2.0))
    freq = base ** (-2.0 * i / rotary_dim)
    if scaling == "linear":
        return freq / factor, 1.0
    if scaling == "yarn":
        turns = original * freq / (2 * math.pi)  # turns over the original context
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0, 1)
        return freq * keep + freq / factor * (1 - keep), 0.1 * math.log(factor) + 1.0
    return freq, 1.0


def _pow2_scale(amax):
    """The least power of two s with amax <= 448 s, in the range of scales (float32)."""
    mantissa, exponent = torch.frexp(amax)  # amax = mantissa * 2^exponent, mantissa in [0.5, 1)
    e = exponent - 9 + (mantissa > 0.875).int()
    e = torch.where(amax > 0, e, torch.full_like(e, SCALE_EXP_MIN)).clamp(SCALE_EXP_MIN, SCALE_EXP_MAX)
    return torch.ldexp(torch.ones_like(amax), e)


def _filled_pages(pages, heads, page, dim, gen, spread):
    """Codes and scales of a cache of random tokens; `spread` is the channels' spread."""
    x = torch.randn(pages, heads, page, dim, device="cuda", generator=gen, dtype=torch.bfloat16)
    x *= torch.exp(spread * torch.randn(1, heads, 1, dim, device="cuda", generator=gen)).bfloat16()
    scale = _pow2_scale(x.abs().amax((2, 3)).float())
    x /= scale[:, :, None, None].bfloat16()
    return x.to(torch.float8_e4m3fn), scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, batch, tokens, dim = DTYPES[case["dtype"]], case["batch"], case["tokens"], case["dim"]

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=gen, dtype=torch.float32).to(dtype)

    if case["op"] == "rotary":
        freq, magnitude = _inverse_frequencies(case["rotary_dim"], case["scaling"])
        start = torch.randint(0, case["far"] + 1, (batch, 1), device="cuda", generator=gen)
        state = {"q": normal(batch, case["heads"], tokens, dim),
                 "k": normal(batch, case["kv_heads"], tokens, dim),
                 "positions": (start + torch.arange(tokens, device="cuda")).int(),
                 "inv_freq": freq.cuda(), "magnitude": magnitude,
                 "interleaved": case["interleaved"], "op": "rotary"}
        if case["grad"]:
            state.update(op="rotary_grad", gq=normal(*state["q"].shape), gk=normal(*state["k"].shape),
                         q=state["q"].requires_grad_(), k=state["k"].requires_grad_())
        return state

    page, heads = case["page"], case["kv_heads"]
    lengths, counts = _lengths(case)
    width = max(1, -(-max(lengths) // page))
    pages = batch * width + 3
    table = torch.randperm(pages, device="cuda", generator=gen)[: batch * width].view(batch, width).int()
    k_pages, k_scale = _filled_pages(pages, heads, page, dim, gen, 0.5)
    v_pages, v_scale = _filled_pages(pages, heads, page, dim, gen, 0.2)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    state = {"op": case["op"], "k_pages": k_pages, "v_pages": v_pages, "k_scale": k_scale,
             "v_scale": v_scale, "table": table, "lengths": ints(lengths),
             "counts": ints(counts) if case["ragged"] else None}
    if case["op"] == "append":
        # Some tokens are far larger than what their page held before, so that scales grow.
        loud = torch.exp2(torch.randint(-2, 4, (batch, 1, tokens, 1), device="cuda", generator=gen).float())
        state.update(k=(normal(batch, heads, tokens, dim) * loud).to(dtype),
                     v=(normal(batch, heads, tokens, dim) * loud).to(dtype),
                     starts=ints([n - c for n, c in zip(lengths, counts)]))
    else:
        state.update(q=normal(batch, case["heads"], tokens, dim), lse=case["lse"])
    return state


# ------------------------------------------------------------------------------ the plain forms


def _rotate(x, cos, sin, interleaved):
    half = cos.shape[-1]
    x = x.float()
    turned, rest = x[..., : 2 * half], x[..., 2 * half:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = turned[..., :half], turned[..., half:]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, rest), -1)


def _rotary(s):
    angle = s["positions"].double()[:, None, :, None] * s["inv_freq"]
    cos, sin = (angle.cos() * s["magnitude"]).float(), (angle.sin() * s["magnitude"]).float()
    dtype = s["q"].dtype
    out = [_rotate(s[n].detach(), cos, sin, s["interleaved"]).to(dtype) for n in ("q", "k")]
    if s["op"] == "rotary_grad":  # the transpose of a rotation turns the other way
        out += [_rotate(s[n], cos, -sin, s["interleaved"]).to(dtype) for n in ("gq", "gk")]
    return out


def _append_to(pages, scales, x, page_ids, t, new, kept, touched):
    ids = page_ids[touched]
    held = pages.view(torch.uint8)[ids].view(torch.float8_e4m3fn).float()  # [n, H, page, D]
    before = scales[ids]
    rows = torch.arange(x.shape[0], device=x.device)[:, None, None].expand_as(t)[touched]
    fresh = x.permute(0, 2, 1, 3)[rows, t[touched].clamp(0, x.shape[2] - 1)].permute(0, 2, 1, 3).float()
    new, kept = new[touched][:, None, :, None], kept[touched][:, None, :, None]
    scale = _pow2_scale((fresh.abs() * new).amax((2, 3)))
    scale = torch.where(kept.any(2).flatten(1), torch.maximum(scale, before), scale)
    whole = scale[:, :, None, None]
    codes = torch.where(new, (fresh / whole).clamp(-E4M3_MAX, E4M3_MAX),
                        torch.where(kept, held * (before[:, :, None, None] / whole), held))
    pages.view(torch.uint8)[ids] = codes.to(torch.float8_e4m3fn).view(torch.uint8)
    scales[ids] = scale


def _append(s):
    page, tokens = s["k_pages"].shape[2], s["k"].shape[2]
    starts = s["starts"].long()
    counts = s["counts"].long() if s["counts"] is not None else torch.full_like(starts, tokens)
    slots = (starts // page)[:, None] + torch.arange((tokens + page - 2) // page + 1, device="cuda")
    place = slots[..., None] * page + torch.arange(page, device="cuda")  # [B, slots, page]
    t = place - starts[:, None, None]
    new = (t >= 0) & (t < counts[:, None, None])
    touched = new.any(-1)
    page_ids = s["table"].long().gather(1, slots.clamp(max=s["table"].shape[1] - 1))
    for kind in ("k", "v"):
        _append_to(s[kind + "_pages"], s[kind + "_scale"], s[kind], page_ids, t, new, t < 0, touched)
    return [s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"]]


def _sequences(pages, scales, table):
    """[B, Hkv, tokens, D] in 32 bits from the cache's pages."""
    x = pages.view(torch.uint8)[table].view(torch.float8_e4m3fn).float()
    x *= scales[table][..., None, None]
    return x.permute(0, 2, 1, 3, 4).flatten(2, 3)


def _attend(s):
    q, table = s["q"], s["table"].long()
    batch, heads, tokens, dim = q.shape
    kv_heads = s["k_pages"].shape[1]
    lengths = s["lengths"].long()
    counts = s["counts"].long() if s["counts"] is not None else torch.full_like(lengths, tokens)
    k = _sequences(s["k_pages"], s["k_scale"], table)
    scores = q.float().view(batch, kv_heads, -1, dim) @ k.transpose(-1, -2)
    del k
    scores = scores.view(batch, heads, tokens, -1).mul_(dim ** -0.5)
    t = torch.arange(tokens, device="cuda")
    last = (lengths - counts)[:, None] + t  # the newest key that row t sees
    last = torch.where(t < counts[:, None], last, -1)
    hidden = torch.arange(scores.shape[-1], device="cuda") > last[..., None]
    scores.masked_fill_(hidden[:, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = scores.sub_(top.clamp(min=-1e30)).exp_()
    total = weights.sum(-1, keepdim=True)
    v = _sequences(s["v_pages"], s["v_scale"], table)
    out = (weights.view(batch, kv_heads, -1, weights.shape[-1]) @ v).view(q.shape)
    out = (out / total.clamp(min=1e-30)).to(q.dtype)
    return [out, (top + total.log()).squeeze(-1)] if s["lse"] else [out]


# ------------------------------------------------------------------------------ one pass


def run(state):
    op = state["op"]
    if not own:
        return _rotary(state) if op.startswith("rotary") else _append(state) if op == "append" else _attend(state)
    import tiledattention_b200 as ta

    if op.startswith("rotary"):
        q, k = ta.rotary(state["q"], state["k"], state["positions"], state["inv_freq"],
                         interleaved=state["interleaved"], magnitude=state["magnitude"])
        if op == "rotary":
            return [q, k]
        grads = torch.autograd.grad((q, k), (state["q"], state["k"]), (state["gq"], state["gk"]))
        return [q.detach(), k.detach(), *grads]
    cache = ta.KVCache8(state["k_pages"], state["v_pages"], state["k_scale"], state["v_scale"])
    if op == "append":
        ta.kv_cache_append(state["k"], state["v"], cache, state["table"], state["starts"],
                           counts=state["counts"])
        return list(cache)
    out = ta.sdpa_kv_cache(state["q"], cache, state["table"], state["lengths"],
                           counts=state["counts"], return_lse=state["lse"])
    return list(out) if state["lse"] else [out]


def work(case):
    batch, tokens, dim, kv_heads = case["batch"], case["tokens"], case["dim"], case["kv_heads"]
    if case["op"] == "rotary":
        values = batch * tokens * (case["heads"] + kv_heads) * dim * (2 if case["grad"] else 1)
        turned = values // dim * case["rotary_dim"]
        return {"bytes": 4 * values + 4 * batch * tokens, "flops": 3 * turned}
    lengths, counts = _lengths(case)
    page = case["page"]
    if case["op"] == "append":
        values = 2 * sum(counts) * kv_heads * dim
        touched = sum(-(-n // page) - (n - c) // page for n, c in zip(lengths, counts) if c)
        return {"bytes": 3 * values + 8 * touched * kv_heads + 4 * touched, "flops": 2 * values}
    rows = sum(counts) * case["heads"]
    seen = sum(c * (n - c) + c * (c + 1) // 2 for n, c in zip(lengths, counts)) * case["heads"]
    pages = sum(-(-n // page) for n in lengths)
    return {"bytes": 2 * sum(lengths) * kv_heads * dim + pages * (8 * kv_heads + 4) + 4 * rows * dim
            + (4 * rows if case["lse"] else 0), "flops": 4 * seen * dim}


# ------------------------------------------------------------------------------ 64 bits


def _exact_rotation(x, turn, interleaved):
    """The pairs as complex numbers, times `turn`."""
    half = turn.shape[-1]
    x = x.detach().double().clone()
    view = x[..., : 2 * half]
    pairs = (view.unflatten(-1, (half, 2)) if interleaved
             else view.unflatten(-1, (2, half)).transpose(-1, -2)).contiguous()
    turned = torch.view_as_real(torch.view_as_complex(pairs) * turn)
    view.copy_(turned.flatten(-2) if interleaved else turned.transpose(-1, -2).flatten(-2))
    return x


def _exact_codes(x):
    """x rounded to the nearest e4m3 value, ties to even, in 64 bits."""
    x = x.clamp(-E4M3_MAX, E4M3_MAX)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def _exact_append(case, s):
    lengths, counts = _lengths(case)
    page = case["page"]
    out = []
    for kind in ("k", "v"):
        pages, scales = s[kind + "_pages"].double(), s[kind + "_scale"].double()
        for b, (n, c) in enumerate(zip(lengths, counts)):
            start = n - c
            for slot in range(start // page, -(-n // page) if c else 0):
                lo, hi = max(start, slot * page), min(n, (slot + 1) * page)
                at, off = int(s["table_list"][b][slot]), lo - slot * page
                x = s[kind][b, :, lo - start: hi - start].double()
                amax = x.abs().amax((1, 2))
                e = torch.ceil(torch.log2(amax.clamp(min=2.0 ** -80) / E4M3_MAX))
                scale = torch.exp2(e.clamp(SCALE_EXP_MIN, SCALE_EXP_MAX))
                if off:
                    scale = torch.maximum(scale, scales[at])
                    held = pages[at, :, :off] * (scales[at] / scale)[:, None, None]
                    pages[at, :, :off] = _exact_codes(held)
                pages[at, :, off: off + hi - lo] = _exact_codes(x / scale[:, None, None])
                scales[at] = scale
        out.append((pages, scales))
    return [out[0][0], out[1][0], out[0][1], out[1][1]]


def _exact_attend(case, s):
    lengths, counts = _lengths(case)
    batch, heads, tokens, dim = s["q"].shape
    group, page = heads // case["kv_heads"], case["page"]
    out = torch.zeros(batch, heads, tokens, dim, device="cuda", dtype=torch.float64)
    lse = torch.full((batch, heads, tokens), -math.inf, device="cuda", dtype=torch.float64)
    for b, (n, c) in enumerate(zip(lengths, counts)):
        if not c:
            continue
        ids = s["table"][b, : -(-n // page)].long()
        k, v = (
            (s[x + "_pages"].view(torch.uint8)[ids].view(torch.float8_e4m3fn).double()
             * s[x + "_scale"][ids].double()[..., None, None]).transpose(0, 1).flatten(1, 2)[:, :n]
            for x in ("k", "v"))
        for h in range(case["kv_heads"]):
            own_heads = slice(h * group, (h + 1) * group)
            q = s["q"][b, own_heads, :c].double()
            scores = torch.einsum("gtd,nd->gtn", q, k[h]) / math.sqrt(dim)
            if c > 1:
                seen = torch.ones(c, n, device="cuda", dtype=torch.bool).tril(n - c)
                scores = torch.where(seen, scores, -math.inf)
            lse[b, own_heads, :c] = torch.logsumexp(scores, -1)
            out[b, own_heads, :c] = torch.einsum("gtn,nd->gtd", torch.softmax(scores, -1), v[h])
    return [out, lse] if case["lse"] else [out]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        angle = s["positions"].double()[:, None, :, None] * s["inv_freq"]
        turn = torch.polar(torch.full_like(angle, s["magnitude"]), angle)
        out = [_exact_rotation(s[n], turn, s["interleaved"]) for n in ("q", "k")]
        if case["grad"]:
            out += [_exact_rotation(s[n], turn.conj(), s["interleaved"]) for n in ("gq", "gk")]
        return out
    if case["op"] == "append":
        s["table_list"] = s["table"].tolist()
        return _exact_append(case, s)
    return _exact_attend(case, s)
