"""Plain 64-bit forms of the serving operators for the GPU tests, with the error bounds that
the kernels' arithmetic allows."""

import math

import torch

E4M3_MAX = 448.0


def half_step(dtype):
    """Largest relative error of one rounding to dtype."""
    return torch.finfo(dtype).eps / 2


# ------------------------------------------------------------------------------ rotary


def rotary64(x, positions, inv_freq, interleaved=False, magnitude=1.0, inverse=False):
    """(result, bound): the rotation in 64 bits and how far an fp32 kernel with one rounding may
    be from it."""
    half = inv_freq.shape[0]
    batch, _, seq, _ = x.shape
    pos = positions.double().expand(batch, seq) if positions.ndim < 2 or positions.shape[0] == 1 else positions.double()
    angle = pos[:, None, :, None] * inv_freq
    c, s = angle.cos() * magnitude, angle.sin() * magnitude * (-1 if inverse else 1)
    v = x.double()
    if interleaved:
        a, b = v[..., 0:2 * half:2], v[..., 1:2 * half:2]
        join = lambda p, q: torch.stack((p, q), -1).flatten(-2)  # noqa: E731
    else:
        a, b = v[..., :half], v[..., half:2 * half]
        join = lambda p, q: torch.cat((p, q), -1)  # noqa: E731
    rest = v[..., 2 * half:]
    out = torch.cat((join(a * c - b * s, b * c + a * s), rest), -1)
    # The turn's fraction, at most 1/2, is rounded to fp32 (2^-26 turns = 2^-23.3 radians), cos
    # and sin are off by 2 units (2^-23), the magnitude and the two products and the sum round
    # once each (4 * 2^-24): together below 2^-21 of |m| (|a| + |b|). Positions below 2^31 leave
    # less than 2^-20 turns' share of double rounding: 2^31 * 2^-53 * 2 pi < 2^-19 radians at the
    # far end, added in proportion.
    far = pos.abs().amax().item() * float(inv_freq.abs().amax()) * 2.0 ** -51
    size = (a.abs() + b.abs()) * abs(magnitude)
    arith = torch.cat((join(size, size) * (2.0 ** -21 + far), torch.zeros_like(rest)), -1)
    return out, arith + half_step(x.dtype) * (out.abs() + arith) + torch.finfo(x.dtype).tiny * half_step(x.dtype) * 2


# ------------------------------------------------------------------------------ the cache


def e4m3(x):
    """x (float64) to the nearest e4m3 value, ties to even, saturating; NaN stays."""
    y = x.clamp(-E4M3_MAX, E4M3_MAX)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step


def scale_of(amax):
    """The least power of two s >= 2^-50 with amax <= 448 s, at most 2^50."""
    e = -50
    while e < 50 and E4M3_MAX * 2.0 ** e < amax:
        e += 1
    return 2.0 ** e


def values(codes):
    return codes.view(torch.uint8).cpu().view(torch.float8_e4m3fn).double()


def append64(x, pages, scales, table, starts, counts):
    """What append leaves in `pages` (float64 code values) and `scales` (float64), token by
    token and page by page; both are changed in place. Bad page ids are skipped."""
    num, heads, page, _ = pages.shape
    for b, start in enumerate(starts):
        n = start + counts[b]
        for slot in range(start // page, -(-n // page) if n > start else 0):
            at = table[b][slot] if slot < len(table[b]) else -1
            if not 0 <= at < num:
                continue
            lo, hi = max(start, slot * page), min(n, (slot + 1) * page)
            off = lo - slot * page
            for h in range(heads):
                new = x[b, h, lo - start:hi - start].double().cpu()
                finite = new[torch.isfinite(new)]
                s = scale_of(float(finite.abs().max()) if finite.numel() else 0.0)
                if off:
                    s = max(s, float(scales[at, h]))
                    pages[at, h, :off] = e4m3(pages[at, h, :off] * (float(scales[at, h]) / s))
                pages[at, h, off:off + hi - lo] = e4m3(new / s)
                scales[at, h] = s


def attend64(q, k_pages, v_pages, k_scale, v_scale, table, lengths, counts=None, causal=True,
             scale=None):
    """(out, lse, out bound, lse bound) in 64 bits on q's device."""
    batch, heads, tokens, dim = q.shape
    kv_heads, page = k_pages.shape[1:3]
    group = heads // kv_heads
    scale = dim ** -0.5 if scale is None else scale
    dev = q.device
    out = torch.zeros(q.shape, dtype=torch.float64, device=dev)
    lse = torch.full(q.shape[:3], -math.inf, dtype=torch.float64, device=dev)
    tol, lse_tol = torch.zeros_like(out), torch.zeros_like(lse)
    whole = [values(p) for p in (k_pages, v_pages)]
    for b in range(batch):
        n, c = int(lengths[b]), tokens if counts is None else int(counts[b])
        if n == 0 or c == 0:
            continue
        ids = table[b, :-(-n // page)].long().cpu()
        k, v = ((p[ids] * s.double().cpu()[ids][..., None, None]).transpose(0, 1)
                .flatten(1, 2)[:, :n].to(dev) for p, s in zip(whole, (k_scale, v_scale)))
        qq = q[b, :, :c].double().view(kv_heads, group, c, dim)
        s = torch.einsum("hgtd,hnd->hgtn", qq, k) * scale
        size = torch.einsum("hgtd,hnd->hgtn", qq.abs(), k.abs()) * scale
        pos = torch.arange(n, device=dev)
        last = n - c + torch.arange(c, device=dev) if causal else torch.full((c,), n - 1, device=dev)
        seen = pos <= last[:, None]
        s = torch.where(seen, s, -math.inf)
        top = s.amax(-1, keepdim=True)
        p = torch.where(seen, torch.exp(s - top.clamp(min=-1e300)), torch.zeros_like(s))
        total = p.sum(-1, keepdim=True)
        has = total > 0
        p = torch.where(has, p / total, torch.zeros_like(p))
        r = torch.einsum("hgtn,hnd->hgtd", p, torch.nan_to_num(v))
        absr = torch.einsum("hgtn,hnd->hgtd", p, torch.nan_to_num(v).abs())
        out[b, :, :c] = r.reshape(heads, c, dim)
        lse[b, :, :c] = (top + total.log()).squeeze(-1).reshape(heads, c)
        # Scores: products of fp16-exact factors summed in fp32 (each of D terms may lose a unit
        # of the sum's size), then the scale, the shift and exp2, in magnitudes up to |s| log2 e.
        ds = dim * 2.0 ** -23 * torch.where(seen, size, torch.zeros_like(size)).amax(-1, keepdim=True)
        ds = ds + (torch.nan_to_num(top.abs(), posinf=0.0) * 1.45 + 110) * 2.0 ** -22
        # Weights: 2^-12 of rounding each (fp16), or 2^-25 absolutely at its lower end against a
        # largest weight of 2^7 or more, on codes up to 448, of which the largest value v shows at
        # least half: per key 448 * 2^-25 / 2^7 <= 2 v * 2^-32. And fp32 sums over n keys.
        e = (2.0 ** -12 + 2 * ds + n * 2.0 ** -23)
        t = e * absr + n * 2.0 ** -31 * torch.nan_to_num(v).abs().amax((1, 2))[:, None, None, None]
        t = t + half_step(q.dtype) * (r.abs() + t) + torch.finfo(q.dtype).tiny * half_step(q.dtype) * 2
        tol[b, :, :c] = t.reshape(heads, c, dim)
        lse_tol[b, :, :c] = (ds + n * 2.0 ** -23).squeeze(-1).reshape(heads, c)
    return out, lse, tol, lse_tol


def make_cache(pages, heads, page, dim, seed, device, v_spread=0):
    """Random cache: (k, v, k_scale, v_scale); scales vary by page, those of V over 2^+-v_spread
    more."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for spread in (1, 1 + v_spread):
        codes = (torch.randn(pages, heads, page, dim, generator=g) * 100).clamp(-448, 448)
        out.append(codes.to(torch.float8_e4m3fn).to(device))
        e = torch.randint(-spread, spread + 1, (pages, heads), generator=g) - 7
        out.append(torch.exp2(e.float()).to(device))
    return out[0], out[2], out[1], out[3]
