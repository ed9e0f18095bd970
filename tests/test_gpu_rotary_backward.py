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


@pytest.mark.parametrize("fast", [True, False])
@pytest.mark.parametrize("reentrant", [True, False])
def test_under_activation_checkpointing(fast, reentrant, monkeypatch):
    """The forward pass runs again in the backward pass, which torch ends early by an exception from
    a saved tensor's hook: it has to come through."""
    import tiledattention_b200 as ta
    from tiledattention_b200 import _native
    from torch.utils.checkpoint import checkpoint

    freq, _ = ta.rotary_frequencies(64, device=DEV)
    pos = torch.arange(9, device=DEV)
    g = _randn(2, 3, 9, 64, seed=5)
    ta.rotary(g, None, pos, freq)
    if not fast:
        monkeypatch.setattr(_native, "_fast", None)
    for second in (False, True):
        q, k = (_randn(2, 3, 9, 64, seed=i).requires_grad_() for i in (1, 2))

        def block(a, b):
            a, b = ta.rotary(a * 2, b if second else None, pos, freq)
            return ta.rotary(a + b if second else a, None, pos, freq)[0]

        want = torch.autograd.grad(block(q, k), (q, k), g, allow_unused=True)
        checkpoint(block, q, k, use_reentrant=reentrant).backward(g)
        assert torch.equal(q.grad, want[0])
        assert torch.equal(k.grad, want[1]) if second else k.grad is None


@pytest.mark.parametrize("fast", [True, False])
def test_errors_of_saved_tensor_hooks(fast, monkeypatch):
    import tiledattention_b200 as ta
    from tiledattention_b200 import _native

    freq, _ = ta.rotary_frequencies(64, device=DEV)
    pos = torch.arange(9, device=DEV)
    q = _randn(2, 3, 9, 64, seed=1).requires_grad_()
    ta.rotary(q, None, pos, freq)
    if not fast:
        monkeypatch.setattr(_native, "_fast", None)
    packs = []

    def refuse(t):
        packs.append(t)
        raise KeyError("not saved")

    with torch.autograd.graph.saved_tensors_hooks(refuse, lambda t: t):
        with pytest.raises(KeyError, match="not saved"):
            ta.rotary(q, None, pos, freq)
    assert len(packs) == 1  # the call was not made a second time
    with torch.autograd.graph.save_on_cpu():
        out = ta.rotary(q, None, pos, freq)[0]
    g = _randn(2, 3, 9, 64, seed=5)
    out.backward(g)
    assert torch.equal(q.grad, ta.rotary(g, None, pos, freq, inverse=True)[0])
