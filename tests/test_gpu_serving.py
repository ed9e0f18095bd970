"""Rotary positions, the 8-bit cache and attention over it on the GPU, against plain 64-bit
forms (serving_plain.py) with bounds derived there."""

import math

import pytest
import torch

import serving_plain as plain

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF16, FP16 = torch.bfloat16, torch.float16


def _randn(*shape, dtype=BF16, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(DEV)


def _ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device=DEV)


def _within(got, want, tol):
    """got within tol of want; an infinity only where want, give or take tol, rounds to one:
    from the largest finite value and half a step on (fp16: 65520)."""
    edge = torch.finfo(got.dtype).max * (1 + plain.half_step(got.dtype) / 2)
    over = torch.isinf(got) & (torch.sign(want) == torch.sign(got)) & (want.abs() + tol >= edge)
    bad = ~over & ~((got.double() - want).abs() <= tol)
    if bad.any():
        i = tuple(int(x) for x in bad.nonzero()[0])
        raise AssertionError(f"{int(bad.sum())} of {bad.numel()} off; first at {i}: got {float(got[i])}, "
                             f"want {float(want[i])}, bound {float(tol[i])}")


# ------------------------------------------------------------------------------ rotary


@pytest.mark.parametrize("B,H,Hk,S,D,R,inter,dtype", [
    (1, 1, 1, 1, 64, 64, False, BF16),
    (2, 4, 2, 1, 128, 128, False, FP16),
    (3, 5, 1, 37, 80, 32, True, FP16),
    (2, 3, 3, 130, 256, 256, True, BF16),
    (1, 32, 8, 300, 128, 64, False, BF16),
    (2, 2, 1, 19, 96, 48, False, FP16),
    (2, 3, 2, 9, 7, 6, False, BF16),      # element by element
    (2, 3, 2, 9, 50, 10, True, FP16),
    (1, 2, 1, 5, 64, 24, False, BF16),    # 24 rotated dims: not whole vectors of the half layout
    (70, 9, 2, 1, 128, 128, False, BF16),
])
def test_rotary_matches_64_bits(B, H, Hk, S, D, R, inter, dtype):
    import tiledattention_b200 as ta

    q, k = _randn(B, H, S, D, dtype=dtype, seed=1), _randn(B, Hk, S, D, dtype=dtype, seed=2)
    freq, mag = ta.rotary_frequencies(R, scaling="yarn", factor=8.0, device=DEV)
    for inverse, pos in ((False, torch.arange(S, device=DEV)),
                         (True, _ints([[7 * b + s + (1 << 20) for s in range(S)] for b in range(B)]))):
        got = ta.rotary(q, k, pos, freq, interleaved=inter, magnitude=mag, inverse=inverse)
        for x, y in zip((q, k), got):
            want, tol = plain.rotary64(x, pos, freq, inter, mag, inverse)
            assert y.is_contiguous() and y.dtype == dtype
            _within(y, want, tol)
            assert torch.equal(y[..., R:], x[..., R:])
    alone, none = ta.rotary(q, None, pos, freq, interleaved=inter, magnitude=mag, inverse=True)
    assert none is None and torch.equal(alone, got[0])


def test_rotary_far_and_negative_positions():
    import tiledattention_b200 as ta

    q = _randn(1, 2, 6, 64, dtype=FP16, seed=3)
    freq, _ = ta.rotary_frequencies(64, device=DEV)
    pos = torch.tensor([0, -1, 12345678, 2 ** 31 - 1, -(2 ** 31), 2 ** 30], device=DEV)
    want, tol = plain.rotary64(q, pos, freq)
    _within(ta.rotary(q, None, pos, freq)[0], want, tol)
    _within(ta.rotary(q, None, pos.int(), freq)[0], want, tol)


def test_rotary_strides_and_layouts():
    import tiledattention_b200 as ta

    freq, _ = ta.rotary_frequencies(64, device=DEV)
    pos = torch.arange(11, device=DEV)
    base = _randn(2, 11, 6, 64, seed=4)
    qkv = _randn(2, 11, 3, 4, 64, seed=5)
    cases = [
        (base.transpose(1, 2), qkv[:, :, 1].transpose(1, 2)),           # [B,S,H,D] storage
        (_randn(2, 6, 11, 65, seed=6)[..., 1:], base.transpose(1, 2)),   # rows not 16-byte aligned
        (_randn(2, 6, 64, 11, seed=7).transpose(2, 3), None),             # dim stride 11
        (_randn(2, 1, 11, 64, seed=8).expand(2, 6, 11, 64), None),        # shared heads
        (_randn(2, 6, 1, 64, seed=9).expand(2, 6, 11, 64), None),
        (_randn(2, 12, 22, 64, seed=10)[:, ::2, ::2], None),
    ]
    for q, k in cases:
        for p in (pos, pos.expand(2, 11), torch.arange(22, device=DEV)[::2]):
            got = ta.rotary(q, k, p, freq)
            for x, y in ((q, got[0]), (k, got[1])):
                if x is not None:
                    want, tol = plain.rotary64(x, p, freq)
                    _within(y, want, tol)
    wide = torch.stack((freq, freq), -1)[:, 0]
    assert torch.equal(ta.rotary(q, None, pos, wide)[0], ta.rotary(q, None, pos, freq)[0])


@pytest.mark.parametrize("shape", [(0, 2, 3, 64), (2, 0, 3, 64), (2, 2, 0, 64)])
def test_rotary_empty(shape):
    import tiledattention_b200 as ta

    freq, _ = ta.rotary_frequencies(64, device=DEV)
    q = torch.empty(shape, dtype=BF16, device=DEV)
    k = _randn(shape[0], 1, shape[2], 64) if shape[0] and shape[2] else q[:, :1]
    a, b = ta.rotary(q, k, torch.arange(shape[2], device=DEV), freq)
    assert a.shape == q.shape and b.shape == k.shape
    if b.numel():
        want, tol = plain.rotary64(k, torch.arange(3, device=DEV), freq)
        _within(b, want, tol)


@pytest.mark.parametrize("inter", [False, True])
def test_rotary_gradient(inter):
    """Against the formula, and against differences of the function itself."""
    import tiledattention_b200 as ta

    freq, mag = ta.rotary_frequencies(48, scaling="yarn", factor=4.0, device=DEV)
    pos = _ints([[3, 100, 5000, 9, 9], [0, 1, 2, 3, 70000]])
    q = _randn(2, 6, 5, 64, dtype=FP16, seed=1).requires_grad_()
    shared = _randn(2, 1, 5, 64, dtype=FP16, seed=2).requires_grad_()
    k = shared.expand(2, 3, 5, 64)  # one head for three
    gq, gk = _randn(2, 6, 5, 64, dtype=FP16, seed=3), _randn(2, 3, 5, 64, dtype=FP16, seed=4)
    oq, ok = ta.rotary(q, k, pos, freq, interleaved=inter, magnitude=mag)
    torch.autograd.backward((oq, ok), (gq, gk))
    want, tol = plain.rotary64(gq, pos, freq, inter, mag, True)
    _within(q.grad, want, tol)
    want, tol = plain.rotary64(gk, pos, freq, inter, mag, True)
    want, tol = want.sum(1, keepdim=True), tol.sum(1, keepdim=True)
    # torch adds the three heads' fp16 gradients: at most three roundings of partial sums
    _within(shared.grad, want, tol + 3 * plain.half_step(FP16) * (want.abs() + 12.0))
    # differences: the map is linear, f(q + e) - f(q) = J e, so <g, J e> = <J^T g, e>
    e = _randn(2, 6, 5, 64, dtype=FP16, seed=5)
    f = lambda x: plain.rotary64(x, pos, freq, inter, mag)[0]  # noqa: E731
    diff = (f(q.detach().double() + e.double() * 1e-3) - f(q.detach().double() - e.double() * 1e-3)) / 2e-3
    lhs, rhs = (gq.double() * diff).sum(), (q.grad.double() * e.double()).sum()
    assert abs(float(lhs - rhs)) <= float((tol.new_tensor(plain.half_step(FP16)) * 2 * (q.grad.double().abs() * e.double().abs()).sum())) + 1e-3

    # only one of the outputs used, only one input wanting a gradient
    (g,) = torch.autograd.grad(ta.rotary(q, k.detach(), pos, freq, interleaved=inter, magnitude=mag)[0],
                               q, gq)
    assert torch.equal(g, q.grad)
    (g,) = torch.autograd.grad(ta.rotary(q.detach(), shared, pos, freq, interleaved=inter, magnitude=mag)[1],
                               shared, gk[:, :1])
    want, tol = plain.rotary64(gk[:, :1], pos, freq, inter, mag, True)
    _within(g, want, tol)
    (g,) = torch.autograd.grad(ta.rotary(q, None, pos, freq, interleaved=inter, magnitude=mag)[0], q, gq)
    assert torch.equal(g, q.grad)
    with torch.no_grad():
        assert not ta.rotary(q, None, pos, freq)[0].requires_grad
    # a gradient that is one value everywhere comes without strides
    (g,) = torch.autograd.grad(ta.rotary(q, None, pos, freq, interleaved=inter)[0].sum(), q)
    want, tol = plain.rotary64(torch.ones_like(q), pos, freq, inter, 1.0, True)
    _within(g, want, tol)


@pytest.mark.parametrize("fast", [True, False])
def test_rotary_second_gradient_and_both_launchers(fast, monkeypatch):
    """The gradient is differentiable too: turning there and back gives the gradient's own."""
    import tiledattention_b200 as ta
    from tiledattention_b200 import _native

    freq, _ = ta.rotary_frequencies(64, device=DEV)
    pos = torch.arange(5, device=DEV)
    q = _randn(2, 3, 5, 64, dtype=FP16, seed=1).requires_grad_()
    k = _randn(2, 1, 5, 64, dtype=FP16, seed=2).requires_grad_()
    ta.rotary(q, k, pos, freq)
    if not fast:
        monkeypatch.setattr(_native, "_fast", None)
    gq = _randn(2, 3, 5, 64, dtype=FP16, seed=3).requires_grad_()
    gk = _randn(2, 1, 5, 64, dtype=FP16, seed=4)
    oq, ok = ta.rotary(q, k, pos, freq, magnitude=1.5)
    dq, dk = torch.autograd.grad((oq, ok), (q, k), (gq, gk), create_graph=True)
    for d, g in ((dq, gq), (dk, gk)):
        want, tol = plain.rotary64(g.detach(), pos, freq, False, 1.5, True)
        _within(d, want, tol)
    u = _randn(2, 3, 5, 64, dtype=FP16, seed=5)
    (dd,) = torch.autograd.grad(dq, gq, u)
    want, tol = plain.rotary64(u, pos, freq, False, 1.5, False)
    _within(dd, want, tol)
    (only,) = torch.autograd.grad(ta.rotary(q.detach(), k, pos, freq)[1], k, gk)
    want, tol = plain.rotary64(gk, pos, freq, False, 1.0, True)
    _within(only, want, tol)


def test_rotary_stream_graph_and_python_path(monkeypatch):
    import tiledattention_b200 as ta
    from tiledattention_b200.rotary import run_rotary

    freq, _ = ta.rotary_frequencies(128, device=DEV)
    q, k = _randn(2, 4, 9, 128, seed=1), _randn(2, 2, 9, 128, seed=2)
    pos = torch.arange(9, device=DEV)
    want = ta.rotary(q, k, pos, freq)
    assert all(torch.equal(a, b) for a, b in zip(want, run_rotary(q, k, pos, freq, False, 1.0, False)))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ta.rotary(q, k, pos, freq)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = ta.rotary(q, k, pos, freq)
    q.copy_(q.flip(2))
    pos.copy_(pos.flip(0))
    g.replay()
    assert all(torch.equal(a, b) for a, b in zip(ta.rotary(q, k, pos, freq), got))
    monkeypatch.setenv("TILEDATTN_SYNC_MODE", "strict")
    assert torch.equal(ta.rotary(q, k, pos, freq)[0], got[0])
    monkeypatch.setenv("TILEDATTN_SYNC_MODE", "nonsense")
    with pytest.raises(ValueError):
        ta.rotary(q, k, pos, freq)


# ------------------------------------------------------------------------------ append


def _table(batch, width, pages, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randperm(pages, generator=g)[:batch * width].view(batch, width).int().to(DEV)


def _append_case(B, H, T, D, page, starts, counts, dtype, seed=0, k=None, v=None):
    import tiledattention_b200 as ta

    width = max(1, max(-(-(s + T) // page) for s in starts))
    pages = B * width + 2
    cache = ta.KVCache8(*plain.make_cache(pages, H, page, D, seed, DEV))
    table = _table(B, width, pages, seed + 1)
    k = _randn(B, H, T, D, dtype=dtype, seed=seed + 2, scale=3.0) if k is None else k
    v = _randn(B, H, T, D, dtype=dtype, seed=seed + 3, scale=0.02) if v is None else v
    want = []
    for codes, scale, x in ((cache.k, cache.k_scale, k), (cache.v, cache.v_scale, v)):
        pv, sv = plain.values(codes), scale.double().cpu()
        plain.append64(x, pv, sv, table.tolist(), starts, counts or [T] * B)
        want.append((pv, sv))
    ta.kv_cache_append(k, v, cache, table, _ints(starts), counts=None if counts is None else _ints(counts))
    ta.check_device_status(DEV)
    for (pv, sv), codes, scale in zip(want, (cache.k, cache.v), (cache.k_scale, cache.v_scale)):
        assert torch.equal(scale.double().cpu(), sv)
        got = plain.values(codes)
        assert torch.equal(torch.isnan(got), torch.isnan(pv))
        assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(pv))
    return cache, table


@pytest.mark.parametrize("B,H,T,D,page,starts,counts,dtype", [
    (1, 1, 1, 16, 16, [0], None, BF16),
    (3, 2, 1, 64, 16, [0, 15, 16], None, FP16),
    (4, 2, 1, 128, 64, [1, 63, 64, 200], None, BF16),
    (2, 3, 5, 80, 16, [13, 30], [5, 2], FP16),
    (3, 2, 130, 128, 64, [0, 7, 64], [130, 0, 129], BF16),
    (1, 2, 300, 256, 128, [5], None, FP16),     # more values a page than registers hold
    (2, 1, 70, 192, 32, [31, 1], [70, 1], BF16),
    (2, 5, 17, 96, 128, [127, 0], None, BF16),
])
def test_append_matches_64_bits(B, H, T, D, page, starts, counts, dtype):
    _append_case(B, H, T, D, page, starts, counts, dtype)


def test_append_extreme_values():
    """Borders of the scale, ties, infinities, NaN, zeros, subnormals."""
    for dtype in (BF16, FP16):
        x = _randn(2, 2, 40, 64, dtype=dtype, seed=9)
        x[0, 0, 0, 0] = 448.0
        x[0, 1, 3, 5] = 450.0
        x[0, 0, 17, 1] = float("inf")
        x[0, 0, 18, 2] = float("-inf")
        x[0, 1, 33, 7] = float("nan")
        x[1, 0] = 0.0
        x[1, 1, :16] = float("inf")
        x[1, 1, 16:32] = float("nan")
        x[1, 1, 32:] = torch.finfo(dtype).tiny / 4
        _append_case(2, 2, 40, 64, 16, [0, 32], None, dtype, k=x, v=x.flip(0).contiguous())
    big = torch.full((1, 1, 3, 64), 3e38, dtype=BF16, device=DEV)
    big[..., ::3] = 1e-30
    _append_case(1, 1, 3, 64, 16, [4], None, BF16, k=big, v=-big)


def test_append_one_by_one_equals_its_definition():
    """Tokens written one at a time through growing scales, page after page."""
    import tiledattention_b200 as ta

    B, H, D, page, n = 2, 2, 64, 16, 40
    cache = ta.kv_cache_alloc(2 * 3, H, page, D, device=DEV)
    table = _table(B, 3, 6, 1)
    x = _randn(B, H, n, D, seed=2) * torch.exp2((torch.arange(n, device=DEV) * 5 % 11).float() - 5)[None, None, :, None].to(BF16)
    pv, sv = plain.values(cache.k), cache.k_scale.double().cpu()
    pw, sw = pv.clone(), sv.clone()
    starts = _ints([0, 0])
    for i in range(n):
        tok = x[:, :, i:i + 1]
        plain.append64(tok, pv, sv, table.tolist(), [i, i], [1, 1])
        plain.append64(-tok, pw, sw, table.tolist(), [i, i], [1, 1])
        ta.kv_cache_append(tok, -tok, cache, table, starts)
        starts += 1
    for codes, scale, want, ws in ((cache.k, cache.k_scale, pv, sv), (cache.v, cache.v_scale, pw, sw)):
        assert torch.equal(scale.double().cpu(), ws)
        assert torch.equal(plain.values(codes), want)


def test_append_strides_graph_and_stream():
    import tiledattention_b200 as ta

    B, H, T, D, page = 2, 3, 21, 64, 16
    x = _randn(B, T, 2, H, D, seed=3)
    k, v = x[:, :, 0].transpose(1, 2), x[:, :, 1].transpose(1, 2)
    _append_case(B, H, T, D, page, [3, 16], None, BF16, k=k, v=v)
    odd = _randn(B, H, T, D + 1, seed=4)[..., 1:]          # rows not 16-byte aligned
    _append_case(B, H, T, D, page, [3, 16], None, BF16, k=odd, v=v.contiguous())
    shared = _randn(B, 1, T, D, seed=5).expand(B, H, T, D)
    _append_case(B, H, T, D, page, [3, 16], None, BF16, k=shared, v=shared)

    a, b = (ta.kv_cache_alloc(8, H, page, D, device=DEV) for _ in range(2))
    table = _table(B, 4, 8, 2)
    starts = _ints([0, 5])
    k, v = k.contiguous(), v.contiguous()
    g = torch.cuda.CUDAGraph()
    ta.kv_cache_append(k, v, a, table, starts)
    a = ta.kv_cache_alloc(8, H, page, D, device=DEV)
    with torch.cuda.graph(g):
        ta.kv_cache_append(k, v, a, table, starts)
    assert not a.k.view(torch.uint8).any()
    g.replay()
    starts += 17
    k.neg_()
    g.replay()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        ta.kv_cache_append(-k, v, b, table, starts - 17)
        ta.kv_cache_append(k, v, b, table, starts)
    s.synchronize()
    assert torch.equal(a.k.view(torch.uint8), b.k.view(torch.uint8))
    assert torch.equal(a.v_scale, b.v_scale)


def test_append_bad_pages_and_lengths_are_reported():
    """Ids and lengths out of range: skipped or held in range by the kernel's own checks, the
    rest written, and check_device_status raises once."""
    import tiledattention_b200 as ta

    B, H, T, D, page = 4, 2, 20, 64, 16
    cache = ta.kv_cache_alloc(8, H, page, D, device=DEV)
    k = _randn(B, H, T, D, seed=1)
    ta.check_device_status(DEV)
    table = _ints([[0, 1], [2, 99], [-1, 3], [4, 5]])
    ta.kv_cache_append(k, k, cache, table, _ints([0, 0, 0, 0]))
    with pytest.raises(ta.KernelError, match="page id"):
        ta.check_device_status(DEV)
    ta.check_device_status(DEV)
    pv, sv = torch.zeros(8, H, page, D, dtype=torch.float64), torch.ones(8, H, dtype=torch.float64)
    plain.append64(k, pv, sv, table.tolist(), [0] * 4, [T] * 4)
    assert torch.equal(plain.values(cache.k), pv) and torch.equal(cache.v_scale.double().cpu(), sv)
    for starts, counts in (([-1, 0, 0, 0], None), ([13, 0, 0, 0], None), ([0] * 4, [T + 1, 1, 1, 1]),
                           ([0] * 4, [-1, 0, 0, 0])):
        ta.kv_cache_append(k, k, cache, _ints([[0, 1], [2, 3], [4, 5], [6, 7]]), _ints(starts),
                           counts=None if counts is None else _ints(counts))
        with pytest.raises(ta.KernelError, match="outside its range"):
            ta.check_device_status(DEV)


# ------------------------------------------------------------------------------ attention


def _attend_case(B, Hq, Hkv, T, D, page, lengths, counts, dtype, causal=True, scale=None, seed=0,
                 v_spread=0, q_scale=1.0, q=None):
    import tiledattention_b200 as ta

    width = max(1, max(-(-n // page) for n in lengths))
    pages = B * width + 2
    cache = ta.KVCache8(*plain.make_cache(pages, Hkv, page, D, seed, DEV, v_spread))
    table = _table(B, width, pages, seed + 1)
    q = _randn(B, Hq, T, D, dtype=dtype, seed=seed + 2, scale=q_scale) if q is None else q
    n, c = _ints(lengths), None if counts is None else _ints(counts)
    got, lse = ta.sdpa_kv_cache(q, cache, table, n, counts=c, causal=causal, scale=scale, return_lse=True)
    ta.check_device_status(DEV)
    want, want_lse, tol, lse_tol = plain.attend64(q, *cache, table, lengths, counts, causal, scale)
    assert got.dtype == dtype and got.shape == q.shape and lse.dtype == torch.float32
    _within(got, want, tol)
    empty = torch.isinf(want_lse)
    assert torch.equal(torch.isinf(lse) & (lse < 0), empty)
    assert (got[empty] == 0).all()
    _within(lse.masked_fill(empty, 0), want_lse.masked_fill(empty, 0), lse_tol)
    alone = ta.sdpa_kv_cache(q, cache, table, n, counts=c, causal=causal, scale=scale)
    assert torch.equal(alone, got)  # the same bits each time, with or without the lse
    return got, lse, cache, table


@pytest.mark.parametrize("D", [16, 64, 80, 128, 176, 192, 240, 256])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_decode_head_dims(D, dtype):
    _attend_case(3, 4, 2, 1, D, 16, [1, 130, 333], None, dtype)


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("group", [1, 3, 8, 16, 17, 40])
def test_decode_pages_and_groups(page, group):
    _attend_case(2, 2 * group, 2, 1, 64, page, [page + 1, 517], None, BF16, seed=page)


@pytest.mark.parametrize("lengths", [[1], [15], [16], [17], [31], [32], [33], [63], [64], [65], [127],
                                     [128], [129], [0], [0, 0], [0, 1, 0], [5, 0, 0, 700, 0]])
def test_decode_lengths(lengths):
    _attend_case(len(lengths), 4, 1, 1, 128, 16, lengths, None, BF16)
    _attend_case(len(lengths), 2, 1, 1, 256, 64, lengths, None, FP16)


@pytest.mark.parametrize("T,causal", [(2, True), (5, True), (5, False), (16, True), (33, True), (100, False)])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_several_tokens(T, causal, D):
    n = [T, T + 1, 300, 3, 0]
    c = [T, min(T, 3), T, min(T, 3), 0]  # at most T
    _attend_case(5, 4, 2, T, D, 32, n, c, BF16, causal=causal)
    # more query rows than keys: the first rows come before the sequence's first token
    _attend_case(2, 2, 2, T, D, 32, [max(1, T - 1), 1], None, FP16, causal=causal)


def test_uneven_batches():
    """Many sequences of very different lengths: runs that are cut, shared and whole."""
    lengths = [(37 * b * b) % 1500 for b in range(70)]
    _attend_case(70, 8, 2, 1, 64, 16, lengths, None, BF16)
    _attend_case(300, 2, 1, 1, 64, 16, [(7 * b) % 40 for b in range(300)], None, FP16)
    lengths[3] = 9000
    _attend_case(70, 4, 4, 1, 128, 64, lengths, None, BF16)


def test_one_long_sequence():
    _attend_case(1, 8, 1, 1, 128, 128, [40001], None, BF16)
    _attend_case(1, 1, 1, 1, 64, 16, [20000], None, FP16)


def test_scales_queries_and_weights_of_many_sizes():
    # value pages over 2^+-20, key scores that leave one key all the weight, tiny and huge queries
    _attend_case(3, 4, 2, 1, 128, 16, [700, 33, 200], None, BF16, v_spread=20)
    _attend_case(3, 4, 2, 3, 64, 16, [700, 33, 200], None, FP16, v_spread=20, q_scale=6.0)
    _attend_case(2, 4, 2, 1, 128, 32, [500, 80], None, BF16, q_scale=30.0)
    _attend_case(2, 4, 2, 1, 128, 32, [500, 80], None, BF16, scale=1e-3, q_scale=1e4)
    _attend_case(2, 4, 2, 1, 128, 32, [500, 80], None, BF16, scale=1e9, q_scale=1e-9)
    _attend_case(2, 4, 2, 1, 128, 32, [500, 80], None, BF16, q=torch.zeros(2, 4, 1, 128, dtype=BF16, device=DEV))
    q = _randn(2, 4, 1, 128, seed=5)
    q[..., ::2] *= 1e-6  # values far below the row's largest
    _attend_case(2, 4, 2, 1, 128, 32, [500, 80], None, BF16, q=q)


def test_zero_pages_with_all_the_weight():
    """A page of zero values (the least scale, 2^-50) that holds the heaviest key still counts in
    the denominator."""
    import tiledattention_b200 as ta

    D, page = 64, 16
    cache = ta.KVCache8(*plain.make_cache(4, 1, page, D, 3, DEV))
    cache.v.view(torch.uint8)[0] = 0
    cache.v_scale[0] = 2.0 ** -50
    cache.v_scale[1] = 2.0 ** 20
    table = _ints([[0, 1, 2]])
    q = values_q = cache.k.view(torch.uint8).cpu().view(torch.float8_e4m3fn).float()[0, 0, 3].to(DEV)
    q = (values_q / values_q.norm() * 8).to(BF16).view(1, 1, 1, D)
    got, lse = ta.sdpa_kv_cache(q, cache, table, _ints([40]), return_lse=True)
    want, want_lse, tol, lse_tol = plain.attend64(q, *cache, table, [40])
    _within(got, want, tol)
    _within(lse, want_lse, lse_tol)


def test_garbage_behind_the_end_and_in_unused_rows():
    """NaN codes and NaN scales in places that no row may see, NaN queries in rows beyond counts,
    and tokens of the same call that hold NaN: they reach only the rows that see them."""
    import tiledattention_b200 as ta

    for D, page, T in ((64, 16, 1), (128, 64, 4), (80, 32, 3), (256, 16, 2), (128, 16, 40)):
        B, H = 3, 2
        cache = ta.KVCache8(*plain.make_cache(B * 4 + 2, H, page, D, D + T, DEV))
        table = _table(B, 4, B * 4 + 2, 1)
        lengths = [page + 5 + T, 3 * page + 1, T]
        counts = [T, max(1, T - 1), T]
        q = _randn(B, 4, T, D, seed=2)
        clean = ta.sdpa_kv_cache(q, cache, table, _ints(lengths), counts=_ints(counts))
        for b in range(B):
            slot, row = divmod(lengths[b], page)
            for codes, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
                raw = codes.view(torch.uint8)
                if row:
                    raw[table[b, slot].long(), :, row:] = 0x7F
                for s in range(slot + (row > 0), 4):
                    raw[table[b, s].long()] = 0xFF
                    scale[table[b, s].long()] = float("nan")
        q[1, :, counts[1]:] = float("nan")
        got = ta.sdpa_kv_cache(q, cache, table, _ints(lengths), counts=_ints(counts))
        assert torch.equal(got, clean)
        if T > 1:  # the last token's value holds a NaN in one dim: only the last row sees it
            slot, row = divmod(lengths[0] - 1, page)
            cache.v.view(torch.uint8)[table[0, slot].long(), 1, row, 7] = 0x7F
            got = ta.sdpa_kv_cache(q, cache, table, _ints(lengths), counts=_ints(counts))
            bad = torch.isnan(got)
            assert bad[0, 2:, T - 1, 7].all()
            bad[0, 2:, T - 1, 7] = False
            assert not bad.any()
            keep = ~torch.isnan(got)
            assert torch.equal(got[keep], clean[keep])
        ta.check_device_status(DEV)


def test_nan_and_infinite_queries_stay_in_their_rows():
    import tiledattention_b200 as ta

    cache = ta.KVCache8(*plain.make_cache(10, 2, 16, 64, 1, DEV))
    table = _table(2, 4, 10, 2)
    for lengths in ([50, 33], [1, 64]):
        q = _randn(2, 8, 2, 64, seed=3)
        clean = ta.sdpa_kv_cache(q, cache, table, _ints(lengths), causal=False)
        q[0, 1, 0, 3] = float("nan")
        q[1, 6, 1, 0] = float("inf")
        got = ta.sdpa_kv_cache(q, cache, table, _ints(lengths), causal=False)
        bad = torch.isnan(got).any(-1)
        assert bad[0, 1, 0] and bad[1, 6, 1] and int(bad.sum()) == 2
        assert torch.equal(got[~bad], clean[~bad])


def test_attention_bad_pages_and_lengths_are_reported():
    import tiledattention_b200 as ta

    cache = ta.KVCache8(*plain.make_cache(6, 1, 16, 64, 1, DEV))
    q = _randn(2, 2, 1, 64, seed=1)
    table = _ints([[0, 1], [2, 3]])
    ta.check_device_status(DEV)
    clean = ta.sdpa_kv_cache(q, cache, table, _ints([30, 20]))
    for bad in ([[0, 1], [2, 6]], [[0, 1], [-7, 3]], [[0, 1], [2 ** 31 - 1, 3]]):
        got = ta.sdpa_kv_cache(q, cache, _ints(bad), _ints([30, 20]))
        assert torch.equal(got[0], clean[0]) and torch.isfinite(got).all()
        with pytest.raises(ta.KernelError, match="page id"):
            ta.check_device_status(DEV)
    ta.sdpa_kv_cache(q, cache, _ints([[0, 1], [2, 6]]), _ints([30, 16]))  # not read: no report
    ta.check_device_status(DEV)
    for lengths, counts in (([33, 20], None), ([-1, 20], None), ([30, 20], [2, 1]), ([30, 20], [-1, 1])):
        got = ta.sdpa_kv_cache(q, cache, table, _ints(lengths), counts=None if counts is None else _ints(counts))
        assert torch.equal(got[1], clean[1])
        with pytest.raises(ta.KernelError, match="outside its range"):
            ta.check_device_status(DEV)


def test_attention_strides_python_path_stream_and_graph(monkeypatch):
    import tiledattention_b200 as ta
    from tiledattention_b200.kv_cache import run_sdpa_kv_cache

    B, H, T, D = 2, 4, 3, 64
    cache = ta.KVCache8(*plain.make_cache(40, 2, 16, D, 1, DEV))
    table, lengths = _table(B, 16, 40, 2), _ints([200, 77])
    q = _randn(B, T, H, D, seed=3).transpose(1, 2)
    want = ta.sdpa_kv_cache(q.contiguous(), cache, table, lengths)
    assert torch.equal(ta.sdpa_kv_cache(q, cache, table, lengths), want)
    odd = torch.cat((q[..., :1], q), -1)[..., 1:]
    assert odd.data_ptr() % 16 and torch.equal(ta.sdpa_kv_cache(odd, cache, table, lengths), want)
    wide = torch.stack((table, table), -1)[..., 0]
    assert torch.equal(ta.sdpa_kv_cache(q, cache, wide, torch.stack((lengths, lengths), -1)[:, 0]), want)
    sliced = torch.cat((table, torch.full_like(table, 10 ** 6)), 1)[:, :16]
    assert torch.equal(ta.sdpa_kv_cache(q, cache, sliced, lengths), want)
    assert torch.equal(run_sdpa_kv_cache(q, cache, table, lengths, None, True, D ** -0.5, False), want)
    assert torch.equal(ta.sdpa_kv_cache(q, tuple(cache), table, lengths), want)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = [ta.sdpa_kv_cache(q, cache, table, lengths) for _ in range(5)]
    others = [ta.sdpa_kv_cache(q, cache, table, lengths) for _ in range(5)]  # two calls at once
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(x, want) for x in got + others)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = ta.sdpa_kv_cache(q, cache, table, lengths)
    lengths.copy_(_ints([31, 0]))
    g.replay()
    assert torch.equal(got, ta.sdpa_kv_cache(q, cache, table, lengths))
    assert (got[1] == 0).all()
    empty = ta.sdpa_kv_cache(q[:0], cache, table[:0], lengths[:0], return_lse=True)
    assert empty[0].shape == (0, H, T, D) and empty[1].shape == (0, H, T)
    monkeypatch.setenv("TILEDATTN_SYNC_MODE", "post")
    assert torch.equal(ta.sdpa_kv_cache(q, cache, table, lengths), got)


def test_offsets_beyond_32_bits():
    """Pages whose byte offsets pass 2^32: written and read at the far end of a cache of
    4.3 GB a side."""
    import tiledattention_b200 as ta

    H, page, D = 8, 128, 256
    pages = (1 << 32) // (H * page * D) + 8
    cache = ta.kv_cache_alloc(pages, H, page, D, device=DEV)
    table = _ints([[pages - 1, 3, pages - 2]])
    x = _randn(1, H, 300, D, seed=1)
    ta.kv_cache_append(x, -x, cache, table, _ints([0]))
    q = _randn(1, H, 1, D, seed=2)
    got = ta.sdpa_kv_cache(q, cache, table, _ints([300]))
    ta.check_device_status(DEV)
    ids = table[0].long()
    small = ta.KVCache8(*(t[ids].contiguous() if t.ndim == 2 else
                          t.view(torch.uint8)[ids].view(torch.float8_e4m3fn) for t in cache))
    want, _, tol, _ = plain.attend64(q, *small, _ints([[0, 1, 2]]), [300])
    _within(got, want, tol)


def test_decoding_loop_over_the_operators():
    """A prompt, then tokens one by one: positions, write, attention, as a decoder runs them,
    against sdpa over all tokens so far, with the cache's own rounding as the only difference."""
    import tiledattention_b200 as ta

    B, Hq, Hkv, D, page, prompt, steps = 2, 8, 2, 128, 16, 37, 6
    total = prompt + steps
    q, k, v = (_randn(B, h, total, D, seed=i) for i, h in enumerate((Hq, Hkv, Hkv)))
    freq, mag = ta.rotary_frequencies(D, scaling="bands", factor=4.0, device=DEV)
    cache = ta.kv_cache_alloc(B * 4, Hkv, page, D, device=DEV)
    table = _table(B, 4, B * 4, 1)
    outs = []
    at = 0
    for n in [prompt] + [1] * steps:
        sl = slice(at, at + n)
        pos = torch.arange(at, at + n, device=DEV)
        qr, kr = ta.rotary(q[:, :, sl], k[:, :, sl], pos, freq, magnitude=mag)
        ta.kv_cache_append(kr, v[:, :, sl], cache, table, _ints([at] * B))
        outs.append(ta.sdpa_kv_cache(qr, cache, table, _ints([at + n] * B)))
        at += n
    got = torch.cat(outs, 2)
    ta.check_device_status(DEV)
    pos = torch.arange(total, device=DEV)
    qr, kr = ta.rotary(q, k, pos, freq, magnitude=mag)
    want = ta.sdpa(qr, kr.repeat_interleave(Hq // Hkv, 1), v.repeat_interleave(Hq // Hkv, 1), causal=True)
    # e4m3 keys and values are off by 2^-4 of themselves at most: values enter the output
    # directly, keys through scores of size |q||k|/sqrt(D) ~ 8, whose errors average over D dims.
    err = (got.float() - want.float()).abs()
    assert float(err.max()) < 0.5 and float(err.mean()) < 0.05
    # exactly: the last step is attention over what the cache now holds
    want, _, tol, _ = plain.attend64(qr[:, :, -1:], *cache, table, [total] * B)
    _within(got[:, :, -1:], want, tol)


@pytest.mark.parametrize("Hq,Hkv,T,D", [(8, 2, 1, 128), (20, 2, 2, 256), (6, 2, 5, 64), (8, 1, 4, 128),
                                        (4, 2, 40, 128), (2, 1, 70, 64)])
def test_lines_of_short_and_long_sequences(Hq, Hkv, T, D):
    """Sequences without keys, of one token and of many in one batch: runs that hold many whole
    sequences beside runs of a part of one."""
    B = 48
    lengths = [(0, 1, T, 17, 300, 64)[b % 6] for b in range(B)]
    lengths[7], lengths[20], lengths[B - 1] = 5000, 2049, 0
    counts = [min(T, n) if b % 5 else max(0, min(T, n) - 1) for b, n in enumerate(lengths)]
    _attend_case(B, Hq, Hkv, T, D, 32, lengths, counts, BF16, seed=T)
    _attend_case(B, Hq, Hkv, T, D, 32, [0] * B, [0] * B, BF16, seed=T)


@pytest.mark.parametrize("D,T", [(128, 32), (128, 33), (192, 48), (192, 49), (256, 48), (256, 49)])
def test_border_of_the_two_kernels(D, T):
    _attend_case(3, 2, 2, T, D, 64, [T, 700, 129 + T], None, FP16, seed=T)


@pytest.mark.parametrize("Hq,Hkv,T,D", [(8, 2, 1, 128), (8, 2, 8, 128), (4, 2, 60, 128), (4, 1, 30, 256)])
def test_calls_at_once_and_graphs(Hq, Hkv, T, D):
    """The same bits from calls in a row, on two streams at once, and from two captured graphs
    replayed in turn with lengths, table and queries that have changed since."""
    import tiledattention_b200 as ta

    B, page = 5, 16
    cache = ta.KVCache8(*plain.make_cache(B * 70 + 2, Hkv, page, D, 1, DEV))
    table = _table(B, 70, B * 70 + 2, 2)
    lengths = _ints([1100, T, 77 + T, 640, 1001])
    q = _randn(B, Hq, T, D, seed=3)
    want = ta.sdpa_kv_cache(q, cache, table, lengths)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = [ta.sdpa_kv_cache(q, cache, table, lengths) for _ in range(20)]
    got += [ta.sdpa_kv_cache(q, cache, table, lengths) for _ in range(20)]
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(x, want) for x in got)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = ta.sdpa_kv_cache(q, cache, table, lengths, return_lse=True)
        graphs.append((g, out))
    for n in ([T, 1100, 900, T + 1, 20 + T], [T] * 5, [1120] * 5):
        lengths.copy_(_ints(n))
        q.copy_(_randn(B, Hq, T, D, seed=sum(n)))
        table.copy_(table.roll(1, 0))
        for g, out in graphs * 2:
            out[0].fill_(7), out[1].fill_(7)
            g.replay()
            fresh = ta.sdpa_kv_cache(q, cache, table, lengths, return_lse=True)
            assert torch.equal(out[0], fresh[0]) and torch.equal(out[1], fresh[1])
    ta.check_device_status(DEV)


def test_each_call_sees_what_the_one_before_wrote():
    """Rotation, write and attention in a row over one set of buffers, eagerly and in a graph,
    against the same calls with the device idle between them."""
    import tiledattention_b200 as ta

    B, Hq, Hkv, D, page, steps = 4, 8, 2, 128, 16, 24
    freq, mag = ta.rotary_frequencies(D, device=DEV)
    q, k, v = (_randn(B, h, 1, D, seed=i) for i, h in enumerate((Hq, Hkv, Hkv)))
    table = _table(B, 4, B * 4, 1)

    def step(cache, at, x, idle):
        pos = at.view(B, 1)
        qr, kr = ta.rotary(x, k, pos, freq, magnitude=mag)
        idle()
        ta.kv_cache_append(kr, v, cache, table, at)
        idle()
        at += 1
        idle()
        out = ta.sdpa_kv_cache(qr, cache, table, at)
        idle()
        x.copy_(out)  # the next query
        idle()

    def run(idle):
        cache, at, x = ta.kv_cache_alloc(B * 4, Hkv, page, D, device=DEV), _ints([0, 3, 15, 30]), q.clone()
        for _ in range(steps):
            step(cache, at, x, idle)
        return x, cache

    want, want_cache = run(torch.cuda.synchronize)
    got, cache = run(lambda: None)
    same = lambda a, b: all(torch.equal(s.view(torch.uint8), t.view(torch.uint8)) for s, t in zip(a, b))
    assert torch.equal(got, want) and same(cache, want_cache)
    cache, at, x = ta.kv_cache_alloc(B * 4, Hkv, page, D, device=DEV), _ints([0, 3, 15, 30]), q.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for _ in range(4):
            step(cache, at, x, lambda: None)
    for _ in range(steps // 4):
        g.replay()
    assert torch.equal(x, want) and same(cache, want_cache)
    ta.check_device_status(DEV)


def test_heads_beyond_a_group_are_refused():
    import tiledattention_b200 as ta

    cache = ta.KVCache8(*plain.make_cache(2, 1, 16, 64, 1, DEV))
    with pytest.raises(ta.InvalidShapeError, match="256 query heads"):
        ta.sdpa_kv_cache(_randn(1, 257, 1, 64), cache, _ints([[0, 1]]), _ints([20]))
    _attend_case(1, 256, 1, 1, 64, 16, [20], None, BF16)


@pytest.mark.parametrize("T", [1, 40])
def test_short_workspaces_are_refused(T):
    from tiledattention_b200 import _native, _runtime

    lib = _runtime.get_native_library()
    cache = plain.make_cache(2, 2, 16, 64, 1, DEV)
    q, table, lengths = _randn(1, 4, T, 64), _ints([[0, 1]]), _ints([20])
    out = torch.full_like(q, 7)
    need = lib.ta_sdpa_kv8_workspace(1, 4, 2, T, 64)
    work = torch.empty(need + 16, dtype=torch.uint8, device=DEV)
    for at, size in ((0, need - 1), (0, 0), (0, -1), (8, need)):
        rc = lib.ta_sdpa_kv8(
            q.data_ptr(), _native.strides4(q.stride()), out.data_ptr(), _native.strides4(out.stride()), None,
            *(t.data_ptr() for t in cache), 2, 16, table.data_ptr(), 2, 2, lengths.data_ptr(), None, 1, 4, 2,
            T, 64, 1, 1, 0.1, work.data_ptr() + at, size, None, torch.cuda.current_stream().cuda_stream)
        assert rc == _native.TA_ERR_INVALID_ARGUMENT, (at, size)
    torch.cuda.synchronize()
    assert (out == 7).all()


@pytest.mark.parametrize("B,H,Hk,S,D,R,inter,dtype", [
    (1, 2, 1, 3, 2304, 2304, True, BF16),    # more slots of 16 bytes than a block has threads
    (1, 2, 1, 3, 2304, 32, False, FP16),
    (9, 6, 3, 220, 80, 40, False, BF16),     # halves of 20: 8-byte accesses
    (2, 3, 2, 33, 84, 84, True, FP16),
    (2, 3, 2, 33, 70, 36, False, BF16),      # halves of 18: 4-byte accesses
    (3, 2, 1, 50, 38, 22, True, FP16),
    (3, 2, 1, 50, 38, 22, False, FP16),      # halves of 11: value by value
])
def test_rotary_widths_of_access(B, H, Hk, S, D, R, inter, dtype):
    test_rotary_matches_64_bits(B, H, Hk, S, D, R, inter, dtype)


def test_rotary_alignment_of_views():
    """Rows at 2, 4 and 8 bytes, of head dims that are whole vectors: the same bits as aligned ones."""
    import tiledattention_b200 as ta

    freq, mag = ta.rotary_frequencies(64, device=DEV)
    pos = torch.arange(30, device=DEV)
    x = _randn(2, 3, 30, 64, seed=4)
    for inter in (False, True):
        want = ta.rotary(x, x, pos, freq, magnitude=mag, interleaved=inter)
        for pad in (1, 2, 4, 6):
            wide = torch.zeros(2, 3, 30, 64 + 2 * pad, dtype=BF16, device=DEV)
            view = wide[..., pad:pad + 64]
            view.copy_(x)
            for pair in ((view, x), (x, view), (view, view)):
                got = ta.rotary(*pair, pos, freq, magnitude=mag, interleaved=inter)
                assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("fast", [True, False])
def test_rotary_gradient_of_one_output(fast, monkeypatch):
    """Where only one of the outputs is used, the other input's gradient is none or zero, and only
    one rotation runs backward."""
    import tiledattention_b200 as ta

    if not fast:
        monkeypatch.setenv("TILEDATTN_SYNC_MODE", "post")  # the Python path
    freq, mag = ta.rotary_frequencies(64, device=DEV)
    pos = torch.arange(9, device=DEV)
    for used in (0, 1):
        q, k = (_randn(2, 3, 9, 64, seed=i).requires_grad_() for i in (1, 2))
        out = ta.rotary(q, k, pos, freq, magnitude=mag)
        g = _randn(2, 3, 9, 64, seed=5)
        out[used].backward(g)
        want = ta.rotary(g, None, pos, freq, magnitude=mag, inverse=True)[0]
        assert torch.equal((q, k)[used].grad, want)
        other = (q, k)[1 - used].grad
        assert other is None or not other.any()
        # a gradient that is the broadcast of one number
        q2 = q.detach().requires_grad_()
        ta.rotary(q2, None, pos, freq)[0].sum().backward()
        assert torch.equal(q2.grad, ta.rotary(torch.ones_like(q2), None, pos, freq, inverse=True)[0])
