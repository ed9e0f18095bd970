"""What the gradient of rotary launches: one kernel for what is used and wanted, none for the rest."""

import sys

import pytest
import torch

from test_gpu_serving import DEV, _randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fast", [True, False])
def test_one_rotation_runs_backward(fast, monkeypatch):
    import tiledattention_b200 as ta
    from tiledattention_b200 import _native

    rotary_mod = sys.modules["tiledattention_b200.rotary"]
    freq, _ = ta.rotary_frequencies(64, device=DEV)
    pos = torch.arange(9, device=DEV)
    ta.rotary(_randn(1, 1, 9, 64), None, pos, freq)
    if fast:
        if _native._fast is None:
            pytest.skip("launcher not built for this interpreter")
        count = _native._fast.launches
    else:
        monkeypatch.setattr(_native, "_fast", None)
        calls, run = [], rotary_mod.run_rotary
        monkeypatch.setattr(rotary_mod, "run_rotary", lambda *a: calls.append(a[1] is not None) or run(*a))
        count = lambda: len(calls)  # noqa: E731
    g = _randn(2, 3, 9, 64, seed=5)
    for wants in ((True, True), (True, False), (False, True)):
        for used in ((0,), (1,), (0, 1)):
            if not any(wants[i] for i in used):
                continue
            q, k = (_randn(2, 3, 9, 64, seed=i).requires_grad_(w) for i, w in enumerate(wants))
            before = count()
            out = ta.rotary(q, k, pos, freq)
            torch.cuda.synchronize()
            assert count() == before + 1
            torch.autograd.backward([out[i] for i in used], [g] * len(used))
            torch.cuda.synchronize()
            assert count() == before + 2
            if not fast:  # with one gradient only, one tensor is turned
                assert calls[-1] == (len(used) == 2 and all(wants))
            want = ta.rotary(g, None, pos, freq, inverse=True)[0]
            for i, t in enumerate((q, k)):
                if i in used and wants[i]:
                    assert torch.equal(t.grad, want)
                else:
                    assert t.grad is None
