"""Attention over the 8-bit cache where scores are so large that a float32 near them is whole units
apart: the weights stay inside their type, and the heaviest key has the row."""

import math

import pytest
import torch

import serving_plain as plain
from test_gpu_serving import BF16, DEV, _attend_case, _ints, _randn, _table

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [4, 60])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_large_scores(D, T):
    import tiledattention_b200 as ta

    cache = ta.KVCache8(*plain.make_cache(20, 2, 16, D, 1, DEV))
    table, n = _table(2, 9, 20, 2), [140, 61]
    q = _randn(2, 4, T, D, seed=3)
    k, v = ((plain.values(c)[table.long().cpu()] * s.double().cpu()[table.long().cpu()][..., None, None])
            .transpose(1, 2).flatten(2, 3).repeat_interleave(2, 1).to(DEV) for c, s in
            ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))  # [B, Hq, tokens, D]
    s = torch.einsum("bhtd,bhnd->bhtn", q.double(), k)
    size = torch.einsum("bhtd,bhnd->bhtn", q.double().abs(), k.abs())
    pos = torch.arange(s.shape[-1], device=DEV)
    last = _ints(n).view(2, 1, 1, 1) - T + torch.arange(T, device=DEV).view(T, 1)
    s = s.masked_fill(pos > last, -math.inf)
    top, at = s.topk(2, -1)
    one = torch.gather(v, 2, at[..., :1].expand(2, 4, T, D))
    # the sums of D products and the rounding of t leave the order of the first two as it is
    clear = top[..., 0] - top[..., 1] > (2 * D * 2.0 ** -23) * size.amax(-1)
    assert clear.float().mean() > 0.9
    for scale in (1e6, 1e7, 1e8, 1e9, 1e12, 1e20):
        got, lse = ta.sdpa_kv_cache(q, cache, table, _ints(n), scale=scale, return_lse=True)
        ta.check_device_status(DEV)
        assert torch.isfinite(got).all() and torch.isfinite(lse).all(), scale
        off = (lse.double() - top[..., 0] * scale).abs()
        assert (off <= (D * 2.0 ** -23 * size.amax(-1) + 2.0 ** -22 * top[..., 0].abs()) * scale + math.log(140)).all()
        # behind a gap of 100 in the exponent the second key's weight, below 2^-100, is nothing
        sure = clear & ((top[..., 0] - top[..., 1]) * scale > 200)
        err = (got.double() - one).abs()
        assert (err[sure] <= plain.half_step(BF16) * one.abs()[sure]).all()
        if scale >= 1e8:
            assert sure.float().mean() > 0.9


@pytest.mark.parametrize("T", [1, 40])
def test_a_weight_at_the_border(T):
    """Two keys whose t are 2^24 + 16 and 2^24 + 24, in different steps of one warp: the first one's
    reference is 2^24 + 8 as float32 rounds it, and the second one's weight against it 2^16, which
    fp16 does not hold; 2^24 + 8 + 15 rounds to 2^24 + 24, which is not below the second's t."""
    import tiledattention_b200 as ta

    B, D, page = 2000, 16, 16  # so many sequences that a block has both steps of most of them
    cache = ta.kv_cache_alloc(20, 1, page, D, device=DEV)
    code = lambda x: torch.tensor(x).to(torch.float8_e4m3fn).view(torch.uint8).item()  # noqa: E731
    k, v = cache.k.view(torch.uint8), cache.v.view(torch.uint8)
    for key, second in ((0, 2.0), (128, 3.0)):
        k[key // page, 0, key % page, 0] = code(128.0)
        k[key // page, 0, key % page, 1] = code(second)
        v[key // page, 0, key % page] = code(second)
    q = torch.zeros(B, 1, T, D, dtype=BF16, device=DEV)
    q[..., 0], q[..., 1] = 2.0 ** 17, 8.0
    table = torch.arange(20, dtype=torch.int32, device=DEV).repeat(B, 1)
    # the scale's log2(e) times is 1 in float32
    got, lse = ta.sdpa_kv_cache(q, cache, table, _ints([250] * B), scale=math.log(2.0), causal=False, return_lse=True)
    want = (3 + 2 * 2.0 ** -8) / (1 + 2.0 ** -8)
    assert ((got.double() - want).abs() <= 2.0 ** -7).all(), got[0, 0, :, 0]  # a step of bf16 at 3
    assert ((lse.double() - (2.0 ** 24 + 24) * math.log(2.0)).abs() <= 4).all()  # float32 there: steps of 1


@pytest.mark.parametrize("scale", [1e4, 3e5, 1e6])
@pytest.mark.parametrize("T", [3, 50])
def test_scores_on_both_sides_of_the_border(scale, T):
    """Rows whose references lie on either side of where differences are taken another way."""
    _attend_case(2, 4, 2, T, 128, 32, [300, 77], None, BF16, scale=scale, seed=T)
    q = _randn(2, 4, T, 128, seed=9) * torch.exp2(torch.arange(4, device=DEV).float() * 3 - 9).view(1, 4, 1, 1).to(BF16)
    _attend_case(2, 4, 2, T, 128, 32, [300, 77], None, BF16, scale=scale, q=q)
