"""The operators around a decoder's attention without a GPU: their index and scale arithmetic
compiled for the host, the C ABI's refusals, the Python checks, and the frequencies."""

import math
import os
import shutil
import subprocess
import sys

import pytest
import torch

import tiledattention_b200 as ta
from tiledattention_b200 import _native, _runtime, build, kv_cache
from tiledattention_b200 import DTypeNotSupportedError, InvalidShapeError, UnsupportedPlatformError

rotary_mod = sys.modules["tiledattention_b200.rotary"]
HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)


def test_index_and_scale_arithmetic(tmp_path):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("nvcc not available")
    exe = str(tmp_path / "kv8_check")
    subprocess.run([nvcc, "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a",
                    os.path.join(HERE, "native", "kv8_check.cu"), "-o", exe],
                   check=True, capture_output=True, timeout=600)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    assert r.stdout.startswith("ok "), r.stdout


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_native.LIB_PATH):
        build.build()
    return _native.load_library(_native.LIB_PATH)


def _strides(heads, tokens, dim):
    return _native.strides4([heads * tokens * dim, tokens * dim, dim, 1])


def _append(lib, **change):
    a = dict(k=0x1000, v=0x1000, kst=_strides(2, 4, 64), vst=_strides(2, 4, 64), kp=0x1000,
             vp=0x1000, ks=0x1000, vs=0x1000, pages=8, page=16, table=0x1000, stride=4, width=4,
             starts=0x1000, counts=None, B=1, H=2, T=4, D=64, dtype=1, status=None, stream=None)
    assert set(change) <= set(a)
    return lib.ta_kv8_append(*{**a, **change}.values())


def test_append_refusals(lib):
    bad = _native.TA_ERR_INVALID_ARGUMENT
    for change in ({"k": None}, {"starts": None}, {"ks": None}, {"table": None}, {"page": 8},
                   {"page": 48}, {"page": 256}, {"pages": 0}, {"width": 0}, {"B": 0}, {"T": 0},
                   {"width": 1 << 28, "stride": 1 << 28}, {"H": 70000}):
        assert _append(lib, **change) == bad, change
    for D in (8, 24, 72, 272):
        assert _append(lib, D=D) == _native.TA_ERR_UNSUPPORTED_DIM
    assert _append(lib, dtype=2) == _native.TA_ERR_UNSUPPORTED_DTYPE
    layout = _native.TA_ERR_LAYOUT
    assert _append(lib, k=0x1008) == layout
    assert _append(lib, vp=0x1004) == layout
    assert _append(lib, kst=_native.strides4([512, 260, 64, 1])) == layout
    assert _append(lib, vst=_native.strides4([512, 256, 64, 2])) == layout
    assert _append(lib, B=2, stride=3) == layout


def _attend(lib, **change):
    a = dict(q=0x1000, qst=_strides(4, 1, 64), o=0x1000, ost=_strides(4, 1, 64), lse=None,
             kp=0x1000, vp=0x1000, ks=0x1000, vs=0x1000, pages=8, page=16, table=0x1000, stride=4,
             width=4, lengths=0x1000, counts=None, B=1, Hq=4, H=2, T=1, D=64, dtype=0, causal=1,
             scale=0.1, work=0x1000, nbytes=1 << 40, status=None, stream=None)
    assert set(change) <= set(a)
    return lib.ta_sdpa_kv8(*{**a, **change}.values())


def test_attend_refusals(lib):
    bad = _native.TA_ERR_INVALID_ARGUMENT
    for change in ({"q": None}, {"o": None}, {"lengths": None}, {"work": None}, {"Hq": 3},
                   {"Hq": 0}, {"scale": 0.0}, {"scale": -1.0}, {"scale": float("nan")},
                   {"scale": float("inf")}, {"page": 0}, {"T": 1 << 25}, {"width": -1}):
        assert _attend(lib, **change) == bad, change
    assert _attend(lib, D=100) == _native.TA_ERR_UNSUPPORTED_DIM
    assert _attend(lib, dtype=3) == _native.TA_ERR_UNSUPPORTED_DTYPE
    assert _attend(lib, qst=_native.strides4([256, 64, 64, 2])) == _native.TA_ERR_LAYOUT
    assert _attend(lib, o=0x1002) == _native.TA_ERR_LAYOUT


def _rotary(lib, **change):
    st = _strides(2, 4, 64)
    a = dict(q=0x1000, qo=0x1000, qst=st, qost=st, Hq=2, k=None, ko=None, kst=None, kost=None, Hk=0,
             B=1, S=4, D=64, R=64, pos=0x1000, p64=0, pst=_native.strides4([4, 1, 0, 0]),
             freq=0x1000, inter=0, inv=0, mag=1.0, dtype=0, stream=None)
    assert set(change) <= set(a)
    return lib.ta_rotary(*{**a, **change}.values())


def test_rotary_refusals(lib):
    bad = _native.TA_ERR_INVALID_ARGUMENT
    for change in ({"q": None}, {"pos": None}, {"freq": None}, {"k": 0x1000}, {"Hk": 1}, {"B": 0},
                   {"mag": float("inf")}, {"mag": float("nan")}, {"S": -1}):
        assert _rotary(lib, **change) == bad, change
    for R in (0, 3, 66, -2):
        assert _rotary(lib, R=R) == _native.TA_ERR_UNSUPPORTED_DIM
    assert _rotary(lib, dtype=2) == _native.TA_ERR_UNSUPPORTED_DTYPE
    assert _rotary(lib, qst=_native.strides4([512, 256, 64, 2])) == _native.TA_ERR_LAYOUT


def test_workspace_size_without_a_gpu(lib):
    assert lib.ta_sdpa_kv8_workspace(1, 3, 2, 1, 64) == 0  # heads do not divide
    assert lib.ta_sdpa_kv8_workspace(0, 4, 2, 1, 64) == 0


# ------------------------------------------------------------------------- Python checks



@pytest.fixture
def as_cuda(monkeypatch):
    """The checks with host tensors passing as CUDA ones, up to the launch."""
    launched = []
    monkeypatch.setattr(_runtime, "require_supported_runtime", lambda: None)
    monkeypatch.setattr(_native, "_fast", None)
    for mod, name in ((kv_cache, "run_kv_cache_append"), (kv_cache, "run_sdpa_kv_cache"),
                      (rotary_mod, "run_rotary")):
        monkeypatch.setattr(mod, name, lambda *a, _n=name: launched.append(_n) or [None, None])
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda self: True))
    return launched


def _cache(pages=4, heads=2, page=16, dim=64):
    return ta.kv_cache_alloc(pages, heads, page, dim, device="cpu")


def _ints(*v):
    return torch.tensor(v, dtype=torch.int32)


def test_cache_alloc():
    c = _cache()
    assert c.k.shape == (4, 2, 16, 64) and c.k.dtype == torch.float8_e4m3fn
    assert c.v_scale.shape == (4, 2) and float(c.k_scale.min()) == 1.0
    assert not c.k.view(torch.uint8).any()
    for bad in ((0, 2, 16, 64), (4, 0, 16, 64), (4, 2, 8, 64), (4, 2, 48, 64), (4, 2, 16, 60),
                (4, 2, 16, 272), (4, 2, 16, 0), (4.0, 2, 16, 64)):
        with pytest.raises(InvalidShapeError):
            ta.kv_cache_alloc(*bad, device="cpu")


def test_append_checks(as_cuda):
    k = torch.zeros(2, 2, 3, 64, dtype=torch.bfloat16)
    table, starts = torch.zeros(2, 4, dtype=torch.int32), _ints(0, 5)
    ta.kv_cache_append(k, k, _cache(), table, starts)
    ta.kv_cache_append(k, k, _cache(), table, starts, counts=_ints(1, 3))
    assert as_cuda == ["run_kv_cache_append"] * 2
    shape = [
        (k[0], k, _cache(), table, starts), (k, k[:, :1], _cache(), table, starts),
        ("k", k, _cache(), table, starts), (k, k, _cache(heads=1), table, starts),
        (k, k, _cache(dim=80), table, starts), (k, k, tuple(_cache())[:3], table, starts),
        (k, k, list(_cache()), table, starts), (k, k, _cache(), table[:1], starts),
        (k, k, _cache(), table[0], starts), (k, k, _cache(), table, _ints(0)),
        (k, k, _cache(), table[:, :0], starts), (k, k, _cache()._replace(k=None), table, starts),
        (k, k, _cache()._replace(k=_cache().k.transpose(2, 3)), table, starts),
        (k, k, _cache()._replace(v=_cache(pages=5).v), table, starts),
        (k, k, _cache()._replace(v_scale=torch.ones(4, 3)), table, starts),
    ]
    for args in shape:
        with pytest.raises(InvalidShapeError):
            ta.kv_cache_append(*args)
    dtype = [
        (k.float(), k.float(), _cache(), table, starts), (k, k.half(), _cache(), table, starts),
        (k, k, _cache(), table.long(), starts), (k, k, _cache(), table, starts.long()),
        (k, k, _cache()._replace(k=_cache().k.view(torch.uint8)), table, starts),
        (k, k, _cache()._replace(k_scale=torch.ones(4, 2, dtype=torch.float64)), table, starts),
    ]
    for args in dtype:
        with pytest.raises(DTypeNotSupportedError):
            ta.kv_cache_append(*args)
    with pytest.raises(InvalidShapeError):
        ta.kv_cache_append(k, k, _cache(), table, starts, counts=_ints(1))
    assert len(as_cuda) == 2


def test_attention_checks(as_cuda):
    q = torch.zeros(2, 6, 3, 64, dtype=torch.float16)
    table, lengths = torch.zeros(2, 4, dtype=torch.int32), _ints(9, 3)
    ta.sdpa_kv_cache(q, _cache(), table, lengths)
    ta.sdpa_kv_cache(q, _cache(), table, lengths, counts=_ints(1, 0), causal=False, scale=2,
                     return_lse=True)
    assert as_cuda == ["run_sdpa_kv_cache"] * 2
    for scale in (0, -1.0, -1, "x", float("inf"), float("nan"), True - 1):
        with pytest.raises(InvalidShapeError):
            ta.sdpa_kv_cache(q, _cache(), table, lengths, scale=scale)
    for kw in ({"causal": 1}, {"return_lse": None}, {"counts": _ints(1, 2, 3)}):
        with pytest.raises(InvalidShapeError):
            ta.sdpa_kv_cache(q, _cache(), table, lengths, **kw)
    for args in ((q[:, :5], _cache(), table, lengths), (q[..., :32], _cache(), table, lengths),
                 (q[0], _cache(), table, lengths), (q, _cache(), table[:1], lengths),
                 (q, _cache(), table, lengths[:1]), (None, _cache(), table, lengths)):
        with pytest.raises(InvalidShapeError):
            ta.sdpa_kv_cache(*args)
    for args in ((q.float(), _cache(), table, lengths), (q, _cache(), table, lengths.long())):
        with pytest.raises(DTypeNotSupportedError):
            ta.sdpa_kv_cache(*args)
    assert len(as_cuda) == 2


def test_rotary_checks(as_cuda):
    q = torch.zeros(2, 4, 5, 64, dtype=torch.bfloat16)
    k, pos = q[:, :1], torch.arange(5)
    freq, _ = ta.rotary_frequencies(32)
    for p in (pos, pos.int(), pos[None], pos.expand(2, 5)):
        ta.rotary(q, k, p, freq)
    ta.rotary(q, None, pos, freq, interleaved=True, magnitude=2, inverse=True)
    assert as_cuda == ["run_rotary"] * 5
    for args in ((q[0], k, pos, freq), (q, k[:1], pos, freq), (q, k[..., :32], pos, freq),
                 (q, k[:, :, :4], pos, freq), (q, k, pos[:4], freq), (q, k, pos.expand(3, 5), freq),
                 (q, k, pos, freq[None]), (q, k, pos, freq[:0]), (q, k, None, freq),
                 (q, k, pos, ta.rotary_frequencies(66)[0]), (None, k, pos, freq)):
        with pytest.raises(InvalidShapeError):
            ta.rotary(*args)
    for args in ((q.float(), None, pos, freq), (q, k.half(), pos, freq), (q, k, pos.double(), freq),
                 (q, k, pos, freq.float())):
        with pytest.raises(DTypeNotSupportedError):
            ta.rotary(*args)
    for kw in ({"interleaved": 1}, {"inverse": None}, {"magnitude": "1"},
               {"magnitude": float("nan")}):
        with pytest.raises(InvalidShapeError):
            ta.rotary(q, k, pos, freq, **kw)
    assert len(as_cuda) == 5


def test_frequencies():
    f, m = ta.rotary_frequencies(64)
    i = torch.arange(32, dtype=torch.float64)
    assert f.dtype == torch.float64 and m == 1.0
    assert torch.allclose(f, 10000.0 ** (-i / 32), rtol=1e-14)
    assert torch.allclose(ta.rotary_frequencies(64, scaling="linear", factor=4)[0], f / 4, rtol=1e-14)
    n = ta.rotary_frequencies(64, scaling="ntk", factor=4)[0]
    assert n[0] == 1.0 and math.isclose(n[-1], f[-1] / 4, rel_tol=1e-12)
    assert (n[1:] < f[1:]).all() and (n > f / 4.0001).all()
    y, m = ta.rotary_frequencies(64, scaling="yarn", factor=4, original_length=4096)
    assert math.isclose(m, 0.1 * math.log(4) + 1)
    turns = 4096 * f / (2 * math.pi)
    assert torch.equal(y[turns >= 32], f[turns >= 32])
    assert torch.allclose(y[turns <= 1], f[turns <= 1] / 4, rtol=1e-14)
    mid = (turns > 1) & (turns < 32)
    assert mid.any() and (y[mid] < f[mid]).all() and (y[mid] > f[mid] / 4).all()
    b, m = ta.rotary_frequencies(64, scaling="bands", factor=4, original_length=4096)
    assert m == 1.0 and torch.equal(b, y)
    assert ta.rotary_frequencies(2, scaling="ntk", factor=4)[0].tolist() == [1.0]
    for kw in ({"rotary_dim": 3}, {"rotary_dim": 0}, {"rotary_dim": 64, "scaling": "x"},
               {"rotary_dim": 64, "base": 0}, {"rotary_dim": 64, "factor": -1},
               {"rotary_dim": 64, "fast": 1, "slow": 2}, {"rotary_dim": 64, "base": float("inf")}):
        with pytest.raises(InvalidShapeError):
            ta.rotary_frequencies(**kw)


@pytest.mark.skipif(torch.cuda.is_available(), reason="the gate without a GPU")
def test_platform_gate():
    _runtime._reset_runtime_cache_for_tests()
    q = torch.zeros(1, 2, 1, 64, dtype=torch.float16)
    with pytest.raises(UnsupportedPlatformError):
        ta.rotary(q, None, _ints(0), ta.rotary_frequencies(64)[0])
    with pytest.raises(UnsupportedPlatformError):
        ta.kv_cache_append(q, q, _cache(), _ints(0)[None], _ints(0))
    with pytest.raises(UnsupportedPlatformError):
        ta.sdpa_kv_cache(q, _cache(), _ints(0)[None], _ints(0))


def test_launcher_declines_host_tensors(lib):
    fast = _native.load_fast_launch(_native.load_library())
    if fast is None:
        pytest.skip("launcher not built for this interpreter")
    q = torch.zeros(1, 2, 1, 64, dtype=torch.float16)
    before = fast.launches()
    freq = ta.rotary_frequencies(64)[0]
    assert fast.rotary(q, None, _ints(0), freq, False, 1.0, False) is None
    assert fast.rotary(1, 2, 3, 4, False, 1.0, False) is None and fast.rotary(q) is None
    assert fast.kv8_append(q, q, *_cache(), _ints(0)[None], _ints(0), None) is None
    assert fast.kv8_append(*[None] * 9) is None
    assert fast.sdpa_kv8(q, *_cache(), _ints(0)[None], _ints(0), None, True, -1.0, False) is None
    assert fast.sdpa_kv8(*[None] * 11) is None
    assert fast.launches() == before


def test_attend_groups_and_workspace(lib):
    assert _attend(lib, Hq=257 * 2) == _native.TA_ERR_INVALID_ARGUMENT
    assert b"256 query heads" in lib.ta_last_error()
    assert _attend(lib, Hq=64, T=1 << 19) == _native.TA_ERR_INVALID_ARGUMENT  # 2^24 rows
