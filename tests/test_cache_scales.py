"""Caches made elsewhere, whose scales need not be powers of two: the values of a page are its codes
times its scale, for keys and values alike."""

import math
import os
import shutil
import subprocess

import pytest
import torch

import serving_plain as plain

HERE = os.path.dirname(os.path.abspath(__file__))


def test_how_scales_are_held(tmp_path):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("nvcc not available")
    exe = str(tmp_path / "kv8_scales_check")
    subprocess.run([nvcc, "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a",
                    os.path.join(HERE, "native", "kv8_scales_check.cu"), "-o", exe],
                   check=True, capture_output=True, timeout=600)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.startswith("ok "), r.stdout + r.stderr


def _cache(pages, heads, page, dim, seed, spread):
    """A cache whose scales lie between powers of two: 2^(-7 +- 1), those of the values 2^(-7 +- spread)."""
    import tiledattention_b200 as ta
    from test_gpu_serving import DEV

    c = ta.KVCache8(*plain.make_cache(pages, heads, page, dim, seed, DEV))
    g = torch.Generator().manual_seed(seed)
    for t, width in ((c.k_scale, 1.0), (c.v_scale, float(spread))):
        t.copy_(torch.exp2((torch.rand(pages, heads, generator=g) * 2 - 1) * width - 7).to(DEV))
    return c


@pytest.mark.gpu
@pytest.mark.parametrize("D,page,T", [(64, 16, 1), (128, 64, 3), (192, 32, 6), (256, 32, 13), (128, 16, 30),
                                      (64, 16, 70), (128, 32, 40), (256, 128, 60)])
@pytest.mark.parametrize("spread", [1, 20, 40])
def test_scales_between_powers_of_two(D, page, T, spread):
    import tiledattention_b200 as ta
    from test_gpu_serving import BF16, DEV, _ints, _randn, _table, _within

    cache = _cache(40, 2, page, D, D + T, spread)
    table, n = _table(2, 18, 40, 2), [min(17 * page, 500), T + 3]
    q = _randn(2, 4, T, D, dtype=BF16, seed=3)
    got, lse = ta.sdpa_kv_cache(q, cache, table, _ints(n), return_lse=True)
    ta.check_device_status(DEV)
    # the bounds' 110 * 2^-22 of an exponent hold the rounding of log2 of a value scale (half a unit
    # of 2^-18 below 64, and 2^-22 of lg2.approx) and two units of its reciprocal
    want, want_lse, tol, lse_tol = plain.attend64(q, *cache, table, n)
    _within(got, want, tol)
    _within(lse, want_lse, lse_tol)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [2, 50])
def test_scales_of_zero(T):
    """Pages of zeros that say so by their scale."""
    import tiledattention_b200 as ta
    from test_gpu_serving import BF16, _ints, _randn, _table, _within

    cache = _cache(20, 2, 16, 64, 1, 2)
    table, n = _table(2, 9, 20, 2), [140, 60]
    cache.k_scale[table[0, 2].long()] = 0.0
    cache.v_scale[table[0, 3].long()] = 0.0
    cache.v_scale[table[1, 0].long(), 1] = 0.0
    q = _randn(2, 4, T, 64, dtype=BF16, seed=3)
    got, lse = ta.sdpa_kv_cache(q, cache, table, _ints(n), return_lse=True)
    want, want_lse, tol, lse_tol = plain.attend64(q, *cache, table, n)
    _within(got, want, tol)
    _within(lse, want_lse, lse_tol)


@pytest.mark.gpu
@pytest.mark.parametrize("size", [0.01, 3.0, 900.0])
def test_append_into_started_pages(size):
    """The larger of the page's scale and the needed power of two; codes within half a step of
    e4m3 of what they stand for, give or take float32's reciprocal."""
    import tiledattention_b200 as ta
    from test_gpu_serving import DEV, FP16, _ints, _randn

    page, D, start, T = 16, 64, 5, 20
    cache = _cache(4, 2, page, D, 1, 3)
    before = [(plain.values(c), s.double().cpu().clone()) for c, s in
              ((cache.k, cache.k_scale), (cache.v, cache.v_scale))]
    x = _randn(1, 2, T, D, dtype=FP16, seed=2, scale=size)
    table = [2, 0]
    ta.kv_cache_append(x, x, cache, _ints([table]), _ints([start]))
    ta.check_device_status(DEV)
    new = x[0].double().cpu()
    for (old, olds), codes, scale in zip(before, (cache.k, cache.v), (cache.k_scale, cache.v_scale)):
        got, s = plain.values(codes), scale.double().cpu()
        for h in range(2):
            part = new[h, :page - start]
            want = max(float(olds[2, h]), plain.scale_of(float(part.abs().max())))
            assert float(s[2, h]) == want and float(s[0, h]) == plain.scale_of(float(new[h, page - start:].abs().max()))
            exact = torch.cat((old[2, h, :start] * (float(olds[2, h]) / want), part / want))
            half = torch.clamp(exact.abs() * 2.0 ** -4, min=2.0 ** -10) * (1 + 2.0 ** -20)
            assert ((got[2, h] - exact).abs() <= half).all()
            if want == float(olds[2, h]):
                assert torch.equal(got[2, h, :start], old[2, h, :start])
        keep = torch.tensor([1, 3])
        assert torch.equal(got[keep], old[keep]) and torch.equal(s[keep], olds[keep])
    assert math.isfinite(float(s.sum()))
