"""Tensors of more than 2^31 values through rotation, cache writes and cache attention: the far ends
are what the same calls give on slices of them."""

import pytest
import torch

import serving_plain as plain
from test_gpu_serving import BF16, DEV, _ints, _randn, _within

pytestmark = pytest.mark.gpu


def _large(*shape):
    t = torch.empty(shape, dtype=BF16, device=DEV)
    assert t.numel() > 2 ** 31
    return t


def test_rotary_of_more_than_2_31_values():
    import tiledattention_b200 as ta

    S, D = (1 << 23) + 5, 128
    q = _large(1, 3, S, D)
    for h in range(3):
        q[0, h].normal_()
    freq, _ = ta.rotary_frequencies(D, device=DEV)
    pos = torch.arange(S, device=DEV)
    got = ta.rotary(q, q[:, 1:2], pos, freq)
    for at in (slice(0, 70), slice(S // 2, S // 2 + 70), slice(S - 70, S)):
        want = ta.rotary(q[:, :, at].contiguous(), q[:, 1:2, at].contiguous(), pos[at], freq)
        assert torch.equal(got[0][:, :, at], want[0]) and torch.equal(got[1][:, :, at], want[1])
    flat = ta.rotary(q.view(3, 1, S, D).transpose(1, 2).reshape(1, 1, 3 * S, D)[..., :10], None,
                     pos.repeat(3), freq[:3])[0]  # value by value
    at = 3 * S - 50
    want = ta.rotary(q[:, 2:, S - 50:, :10].contiguous(), None, pos[-50:], freq[:3])[0]
    assert torch.equal(flat[:, :, at:], want)


def test_append_of_more_than_2_31_values():
    import tiledattention_b200 as ta

    T, D, page = (1 << 23) + 77, 256, 128
    x = _large(1, 1, T, D)
    x.normal_()
    pages = -(-(T + 3) // page)
    cache = ta.kv_cache_alloc(pages, 1, page, D, device=DEV)
    table = torch.arange(pages, dtype=torch.int32, device=DEV).flip(0).view(1, pages).contiguous()
    ta.kv_cache_append(x, x, cache, table, _ints([3]))
    ta.check_device_status(DEV)
    small = ta.kv_cache_alloc(3, 1, page, D, device=DEV)
    first = (pages - 3) * page - 3  # the token in row 0 of the last three pages
    ta.kv_cache_append(x[:, :, first:].contiguous(), x[:, :, first:].contiguous(), small, _ints([[2, 1, 0]]), _ints([0]))
    for a, b in zip(cache, small):
        assert torch.equal(a[:3].view(torch.uint8), b.view(torch.uint8))


def test_attention_of_more_than_2_31_values():
    """A padded batch of one: 2^22 rows a head, of which the last 40 see keys."""
    import tiledattention_b200 as ta

    T, D, n = (1 << 22) + 3, 256, 40
    cache = ta.KVCache8(*plain.make_cache(4, 1, 32, D, 1, DEV))
    table = _ints([[2, 0]])
    q = _large(1, 2, T, D)
    q.zero_()
    q[:, :, -50:] = _randn(1, 2, 50, D, seed=1)
    q[:, :, :3] = float("nan")
    got, lse = ta.sdpa_kv_cache(q, cache, table, _ints([n]), return_lse=True)
    ta.check_device_status(DEV)
    assert not got[:, :, :-n].any() and torch.isneginf(lse[:, :, :-n]).all()
    want, want_lse, tol, lse_tol = plain.attend64(q[:, :, -n:], *cache, table, [n])
    _within(got[:, :, -n:], want, tol)
    _within(lse[:, :, -n:], want_lse, lse_tol)
