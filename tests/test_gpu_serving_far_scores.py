"""Attention over the 8-bit cache where scores are so large that a float32 near them is whole units
apart: the weights stay inside their type, and the heaviest key has the row."""

import math

import pytest
import torch

from test_gpu_serving import BF16, DEV, _ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [1])
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
