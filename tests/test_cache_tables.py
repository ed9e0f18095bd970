"""Page tables in layouts of their own: one row for the whole batch, windows into a wider row."""

import pytest
import torch

import serving_plain as plain


@pytest.fixture(params=["fast", "python"])
def path(request, monkeypatch):
    from tiledattention_b200 import _native

    if request.param == "python":
        monkeypatch.setattr(_native, "_fast", None)


def test_rows_that_overlap_are_copied():
    from tiledattention_b200.kv_cache import _table_rows

    t = torch.arange(12, dtype=torch.int32)
    for view, same in ((t.view(3, 4), True), (t.view(3, 4)[:, :2], True), (t.view(3, 4)[:1], True),
                       (t[:4].expand(1, 4), True), (t[:4].expand(3, 4), False), (t.view(4, 3).t(), False),
                       (t.as_strided((4, 5), (2, 1)), False)):
        got = _table_rows(view)
        assert torch.equal(got, view) and (got is view) == same
        assert got.stride(1) == 1 and (got.shape[0] == 1 or got.stride(0) >= got.shape[1])


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 40])
def test_one_row_for_the_batch(T, path):
    """Several sequences over one table: samples of one prompt that have not gone apart yet."""
    import tiledattention_b200 as ta
    from test_gpu_serving import DEV, _ints, _randn, _table

    cache = ta.KVCache8(*plain.make_cache(20, 2, 16, 64, 1, DEV))
    row, n, q = _table(1, 9, 20, 2), _ints([140, 60, 141]), _randn(3, 4, T, 64, seed=3)
    want = ta.sdpa_kv_cache(q, cache, row.repeat(3, 1), n)
    assert torch.equal(ta.sdpa_kv_cache(q, cache, row.expand(3, 9), n), want)
    windows = torch.arange(13, dtype=torch.int32, device=DEV).as_strided((3, 9), (2, 1))
    assert torch.equal(ta.sdpa_kv_cache(q, cache, windows, n), ta.sdpa_kv_cache(q, cache, windows.contiguous(), n))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = ta.sdpa_kv_cache(q, cache, row.expand(3, 9), n)
    row.copy_(row.flip(1))
    g.replay()
    assert torch.equal(got, ta.sdpa_kv_cache(q, cache, row.repeat(3, 1), n))
    ta.check_device_status(DEV)


@pytest.mark.gpu
def test_append_through_one_row(path):
    """Sequences that write different pages of one table."""
    import tiledattention_b200 as ta
    from test_gpu_serving import DEV, _ints, _randn, _table

    row, starts = _table(1, 9, 20, 2), _ints([0, 32, 80])
    k, v = (_randn(3, 2, 20, 64, seed=i) for i in (1, 2))
    caches = [ta.kv_cache_alloc(20, 2, 16, 64, device=DEV) for _ in range(2)]
    ta.kv_cache_append(k, v, caches[0], row.repeat(3, 1), starts)
    ta.kv_cache_append(k, v, caches[1], row.expand(3, 9), starts)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(*caches))
    assert caches[0].k.view(torch.uint8).any()
    ta.check_device_status(DEV)
