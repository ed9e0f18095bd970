"""Sequences of nearly 2^31 tokens: the most that a page table may hold."""

import os
import shutil
import subprocess

import pytest
import torch

import serving_plain as plain

HERE = os.path.dirname(os.path.abspath(__file__))


def test_counts_of_tiles_and_slots(tmp_path):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("nvcc not available")
    exe = str(tmp_path / "kv8_far_check")
    subprocess.run([nvcc, "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a",
                    os.path.join(HERE, "native", "kv8_far_check.cu"), "-o", exe],
                   check=True, capture_output=True, timeout=600)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.startswith("ok"), r.stdout + r.stderr


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 40])
def test_the_longest_table(T):
    """2^31 - 16 tokens, the pages of a small cache over and over: attention over these is attention
    over the small cache with every key as often as its page is in the table."""
    import tiledattention_b200 as ta
    from test_gpu_serving import DEV, _ints, _randn

    D, page, pages = 16, 16, 1024
    width = (1 << 27) - 1
    cache = ta.KVCache8(*plain.make_cache(pages, 1, page, D, 1, DEV))
    table = (torch.arange(width, dtype=torch.int32, device=DEV) % pages).view(1, width)
    q = _randn(1, 1, T, D, seed=2)
    got, lse = ta.sdpa_kv_cache(q, cache, table, _ints([width * page]), return_lse=True, causal=False)
    ta.check_device_status(DEV)
    order = torch.arange(pages, dtype=torch.int32, device=DEV).view(1, pages)
    want, want_lse, tol, lse_tol = plain.attend64(q, *cache, order, [pages * page], causal=False)
    times = width / pages
    # One page is there once less than the others: 2^-17 of the weight at most, in a row whose keys
    # weigh alike. A lane's sums take 2^31 / (2 * 148 * 4 * 32) terms of two keys or more, an
    # accumulator of the matrix unit 2^31 / (148 * 64) or fewer: 2^18 roundings of 2^-24.
    more = 2.0 ** -6
    assert ((lse.double() - want_lse - torch.tensor(times).double().log().item()).abs() <= lse_tol + more).all()
    size = max(float(want.abs().max()), float((plain.values(cache.v) * cache.v_scale.double().cpu()[..., None, None]).abs().mean()))
    assert ((got.double() - want).abs() <= tol + more * size).all()
    if T > 1:  # causal: the last rows see all but a few keys
        less = ta.sdpa_kv_cache(q, cache, table, _ints([width * page]))
        ta.check_device_status(DEV)
        assert ((less.double() - want).abs() <= tol + more * size).all()
