"""Queries with infinities against the 8-bit cache: softmax of infinite scores is NaN, also where all
of them are -inf, and nobody else's row is."""

import math

import pytest
import torch

import serving_plain as plain
from test_gpu_serving import BF16, DEV, FP16, _ints, _randn, _table

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D,T", [(64, 1), (128, 4), (256, 5), (64, 60), (128, 150), (256, 70)])
def test_scores_of_minus_infinity(D, T, dtype):
    import tiledattention_b200 as ta

    cache = ta.KVCache8(*plain.make_cache(60, 2, 16, D, 1, DEV))
    cache.k.view(torch.uint8)[..., 0] = 0x38  # 1.0: every key's first dim is positive
    table = _table(3, 18, 60, 2)
    lengths = _ints([280, T, max(1, T - 1)])  # the last one's first row sees no key where T > 1
    q = _randn(3, 4, T, D, dtype=dtype, seed=3)
    clean, lse = ta.sdpa_kv_cache(q, cache, table, lengths, return_lse=True)
    at = [(0, 0, 0), (1, 3, T - 1), (2, 1, 0), (2, 2, T - 1)]
    for (b, h, t), x in zip(at, (-math.inf, -math.inf, -math.inf, math.inf)):
        q[b, h, t, 0] = x
    got, lse2 = ta.sdpa_kv_cache(q, cache, table, lengths, return_lse=True)
    ta.check_device_status(DEV)
    bad = torch.zeros(3, 4, T, dtype=torch.bool, device=DEV)
    for b, h, t in at:
        if not torch.isinf(lse[b, h, t]):
            bad[b, h, t] = True
    assert int(bad.sum()) == (4 if T == 1 else 3)
    assert torch.isnan(got[bad]).all() and torch.isnan(lse2[bad]).all()
    assert torch.equal(got[~bad], clean[~bad]) and torch.equal(lse2[~bad], lse[~bad])
