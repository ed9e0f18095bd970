"""Attention of many query rows over the 8-bit cache (more than 32 per cache head, 48 above head
dim 128) on the GPU: blocks of rows, masks, values out of the ordinary, far offsets. Bounds as
in serving_plain.py."""

import math

import pytest
import torch

import serving_plain as plain
from test_gpu_serving import BF16, DEV, FP16, _attend_case, _ints, _randn, _table, _within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [48, 64, 80, 96, 128, 144, 192, 256])
@pytest.mark.parametrize("causal", [True, False])
def test_several_blocks_of_rows(D, causal):
    """Blocks of 256 rows (128 above head dim 128), the last of them short: of one row tile where
    the others have two, of two, and of one row."""
    for T, lengths in ((300, [300, 777, 1]), (200, [641, 200, 0]), (129, [130, 129, 1000])):
        _attend_case(3, 4, 2, T, D, 32, lengths, [min(T, n) for n in lengths], BF16, causal=causal, seed=T + D)
    _attend_case(2, 3, 1, 171, D, 16, [171, 500], None, FP16, causal=causal, seed=D)  # 513 rows


@pytest.mark.parametrize("D", [64, 128, 256])
def test_more_blocks_in_a_run_than_are_kept(D):
    """Hundreds of blocks of one or two key tiles: a CTA's run has more of them than its rings."""
    B, Hq, Hkv, T = 40, 64, 8, 128
    lengths = [(128, 130, 256, 90, 17)[b % 5] for b in range(B)]
    _attend_case(B, Hq, Hkv, T, D, 64, lengths, [min(T, n) for n in lengths], BF16, seed=D)


@pytest.mark.parametrize("D", [80, 128, 256])
def test_counts_that_leave_blocks_empty(D):
    B, T = 7, 400
    lengths = [900, 400, 5, 1000, 0, 333, 129]
    counts = [400, 1, 5, 0, 0, 128, 129]
    for causal in (True, False):
        _attend_case(B, 6, 2, T, D, 16, lengths, counts, FP16, causal=causal, seed=D)
    _attend_case(B, 6, 2, T, D, 16, [0, 0, 0, 0, 0, 0, 0], [400, 0, 0, 0, 3, 0, 0], FP16, seed=D)
    # more rows than keys: the first blocks come before the sequence's first token
    _attend_case(2, 6, 2, T, D, 16, [30, 1], None, FP16, seed=D)


@pytest.mark.parametrize("D", [64, 128, 192, 256])
def test_scales_queries_and_weights_of_many_sizes(D):
    case = dict(B=2, Hq=4, Hkv=2, T=40, D=D, page=32, lengths=[500, 80], counts=None)
    _attend_case(**case, dtype=BF16, v_spread=20)
    _attend_case(**case, dtype=FP16, v_spread=20, q_scale=6.0)
    _attend_case(**case, dtype=BF16, q_scale=30.0)
    _attend_case(**case, dtype=BF16, scale=1e-3, q_scale=1e4)
    _attend_case(**case, dtype=BF16, scale=1e9, q_scale=1e-9)
    _attend_case(**case, dtype=BF16, q=torch.zeros(2, 4, 40, D, dtype=BF16, device=DEV))
    q = _randn(2, 4, 40, D, seed=5)
    q[..., ::2] *= 1e-6  # values far below the row's largest
    _attend_case(**case, dtype=BF16, q=q)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_nan_and_infinite_queries_stay_in_their_rows(D):
    import tiledattention_b200 as ta

    cache = ta.KVCache8(*plain.make_cache(40, 2, 16, D, 1, DEV))
    table = _table(2, 20, 40, 2)
    for lengths in ([300, 133], [60, 320]):
        q = _randn(2, 8, 60, D, seed=3)
        clean = ta.sdpa_kv_cache(q, cache, table, _ints(lengths), causal=False)
        q[0, 1, 0, 3] = float("nan")
        q[1, 6, 59, 0] = float("inf")
        got = ta.sdpa_kv_cache(q, cache, table, _ints(lengths), causal=False)
        bad = torch.isnan(got).any(-1)
        assert bad[0, 1, 0] and bad[1, 6, 59] and int(bad.sum()) == 2
        assert torch.equal(got[~bad], clean[~bad])


@pytest.mark.parametrize("D", [64, 128, 256])
def test_nan_values_reach_the_rows_that_see_them(D):
    """A NaN in one dim of one token's value, at places before, at and behind the border of the rows
    that see it: those rows' dim is NaN, everything else keeps its bits."""
    import tiledattention_b200 as ta

    T, n, page = 150, 420, 32
    for at in (0, 100, n - T, n - T + 1, n - 77, n - 1):
        cache = ta.KVCache8(*plain.make_cache(20, 2, page, D, 1, DEV))
        table = _table(1, 14, 20, 2)
        q = _randn(1, 4, T, D, seed=3)
        clean, lse = ta.sdpa_kv_cache(q, cache, table, _ints([n]), return_lse=True)
        cache.v.view(torch.uint8)[table[0, at // page].long(), 1, at % page, 5] = 0xFF
        got, lse2 = ta.sdpa_kv_cache(q, cache, table, _ints([n]), return_lse=True)
        sees = n - T + torch.arange(T, device=DEV) >= at
        assert torch.isnan(got[0, 2:, sees, 5]).all()
        want = clean.clone()
        want[0, 2:, :, 5] = torch.where(sees, torch.full_like(want[0, 2:, :, 5], math.nan), want[0, 2:, :, 5])
        assert torch.equal(torch.nan_to_num(got, 77.0), torch.nan_to_num(want, 77.0))
        assert torch.equal(lse, lse2)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_bad_pages_and_lengths_are_reported(D):
    import tiledattention_b200 as ta

    T = 60
    cache = ta.KVCache8(*plain.make_cache(20, 1, 16, D, 1, DEV))
    q = _randn(2, 2, T, D, seed=1)
    table = _ints([list(range(10)), list(range(10, 20))])
    lengths = _ints([150, 160])
    ta.check_device_status(DEV)
    clean = ta.sdpa_kv_cache(q, cache, table, lengths)
    for slot, bad in ((9, 20), (0, -7), (4, 2 ** 31 - 1)):
        broken = table.clone()
        broken[1, slot] = bad
        got = ta.sdpa_kv_cache(q, cache, broken, lengths, causal=False)
        with pytest.raises(ta.KernelError, match="page id"):
            ta.check_device_status(DEV)
        kept = torch.cat((table[1, :slot], table[1, slot + 1:]))[None]
        want, _, tol, _ = plain.attend64(q[1:], *cache, kept, [144], causal=False)
        _within(got[1:], want, tol)
        assert torch.equal(got[:1], ta.sdpa_kv_cache(q[:1], cache, table[:1], lengths[:1], causal=False))
    nothing = ta.sdpa_kv_cache(q, cache, table - 20, lengths, return_lse=True)
    assert not nothing[0].any() and (nothing[1] == -math.inf).all()
    with pytest.raises(ta.KernelError, match="page id"):
        ta.check_device_status(DEV)
    for n, c in (([161, 160], None), ([-1, 160], None), ([150, 160], [T + 1, T]), ([150, 160], [-1, T])):
        got = ta.sdpa_kv_cache(q, cache, table, _ints(n), counts=None if c is None else _ints(c))
        assert torch.equal(got[1], clean[1])
        with pytest.raises(ta.KernelError, match="outside its range"):
            ta.check_device_status(DEV)


@pytest.mark.parametrize("Hq,T", [(8, 1), (32, 20)])
def test_offsets_beyond_32_bits(Hq, T):
    """Pages whose byte offsets pass 2^32, for few rows of a cache head and for many."""
    import tiledattention_b200 as ta

    H, page, D = 8, 128, 256
    pages = (1 << 32) // (H * page * D) + 8
    cache = ta.kv_cache_alloc(pages, H, page, D, device=DEV)
    table = _ints([[pages - 1, 3, pages - 2]])
    x = _randn(1, H, 300, D, seed=1)
    ta.kv_cache_append(x, -x, cache, table, _ints([0]))
    q = _randn(1, Hq, T, D, seed=2)
    got = ta.sdpa_kv_cache(q, cache, table, _ints([300]))
    ta.check_device_status(DEV)
    ids = table[0].long()
    small = ta.KVCache8(*(t[ids].contiguous() if t.ndim == 2 else
                          t.view(torch.uint8)[ids].view(torch.float8_e4m3fn) for t in cache))
    want, _, tol, _ = plain.attend64(q, *small, _ints([[0, 1, 2]]), [300])
    _within(got, want, tol)


def test_each_chunk_sees_what_the_calls_before_wrote():
    """A prompt in chunks through rotation, write and attention, eagerly and in a graph, against the
    same calls with the device idle between them."""
    import tiledattention_b200 as ta

    B, Hq, Hkv, D, page, T, steps = 2, 8, 2, 128, 16, 40, 6
    freq, mag = ta.rotary_frequencies(D, device=DEV)
    q, k, v = (_randn(B, h, T, D, seed=i) for i, h in enumerate((Hq, Hkv, Hkv)))
    table = _table(B, 16, B * 16, 1)

    def step(cache, at, x, idle):
        pos = at.view(B, 1) + torch.arange(T, device=DEV, dtype=torch.int32)
        qr, kr = ta.rotary(x, k, pos, freq, magnitude=mag)
        idle()
        ta.kv_cache_append(kr, v, cache, table, at)
        idle()
        at += T
        idle()
        out = ta.sdpa_kv_cache(qr, cache, table, at)
        idle()
        x.copy_(out)
        idle()

    def start():
        return ta.kv_cache_alloc(B * 16, Hkv, page, D, device=DEV), _ints([0, 13]), q.clone()

    def run(idle):
        cache, at, x = start()
        for _ in range(steps):
            step(cache, at, x, idle)
        return x, cache

    same = lambda a, b: all(torch.equal(s.view(torch.uint8), t.view(torch.uint8)) for s, t in zip(a, b))  # noqa: E731
    want, want_cache = run(torch.cuda.synchronize)
    got, cache = run(lambda: None)
    assert torch.equal(got, want) and same(cache, want_cache)
    cache, at, x = start()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for _ in range(2):
            step(cache, at, x, lambda: None)
    for _ in range(steps // 2):
        g.replay()
    assert torch.equal(x, want) and same(cache, want_cache)
    ta.check_device_status(DEV)


@pytest.mark.parametrize("T", [1, 40])
def test_captured_streams_that_part_and_join(T):
    """Calls on two streams of one captured graph, each behind work of the other stream."""
    import tiledattention_b200 as ta

    B, Hq, Hkv, D, page = 3, 8, 2, 128, 16
    freq, mag = ta.rotary_frequencies(D, device=DEV)
    q, k, v = (_randn(B, h, T, D, seed=i) for i, h in enumerate((Hq, Hkv, Hkv)))
    table = _table(B, 8, B * 8, 1)
    starts = _ints([0, 13, 40])
    caches = [ta.kv_cache_alloc(B * 8, Hkv, page, D, device=DEV) for _ in range(3)]

    def work(cache, side):
        main = torch.cuda.current_stream()
        side = side or main
        pos = starts.view(B, 1) + torch.arange(T, device=DEV, dtype=torch.int32)
        side.wait_stream(main)
        with torch.cuda.stream(side):
            _, kr = ta.rotary(k, k, pos, freq, magnitude=mag)
            ta.kv_cache_append(kr, v, cache, table, starts)
        qr, _ = ta.rotary(q, None, pos, freq, magnitude=mag)
        main.wait_stream(side)
        out = ta.sdpa_kv_cache(qr, cache, table, starts + T)
        side.wait_stream(main)
        with torch.cuda.stream(side):
            twice = ta.sdpa_kv_cache(out, cache, table, starts + T)
        main.wait_stream(side)
        return ta.sdpa_kv_cache(qr + twice, cache, table, starts + T)

    want = work(caches[0], None)
    side = torch.cuda.Stream()
    assert torch.equal(work(caches[1], side), want)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = work(caches[2], side)
    for _ in range(3):
        got.fill_(7)
        g.replay()
        assert torch.equal(got, want)
    ta.check_device_status(DEV)
