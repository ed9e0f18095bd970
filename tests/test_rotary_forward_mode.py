"""Forward-mode derivatives of rotary: the rotation is linear, so a tangent turns as its tensor does."""

import sys

import pytest
import torch
import torch.autograd.forward_ad as fwad

import tiledattention_b200 as ta
from tiledattention_b200 import _native, _runtime

BF16, FP16 = torch.bfloat16, torch.float16


def _tangent(t):
    return fwad.unpack_dual(t).tangent


@pytest.fixture
def plain_kernel(monkeypatch):
    """Host tensors pass as CUDA ones, and the kernel is the formula in torch."""
    def run(q, k, positions, inv_freq, interleaved, magnitude, inverse):
        half = inv_freq.shape[0]
        angle = positions.double()[:, None] * inv_freq
        c, s = angle.cos() * magnitude, angle.sin() * magnitude * (-1 if inverse else 1)

        def turn(t):
            if t is None:
                return None
            assert _tangent(t) is None  # a kernel sees values only
            v = t.detach().double()
            a, b = v[..., :half], v[..., half:]
            return torch.cat((a * c - b * s, b * c + a * s), -1).to(t.dtype)
        return [turn(q), turn(k)]

    monkeypatch.setattr(_runtime, "require_supported_runtime", lambda: None)
    monkeypatch.setattr(_native, "_fast", None)
    monkeypatch.setattr(sys.modules["tiledattention_b200.rotary"], "run_rotary", run)
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda self: True))


def _check(dev):
    g = torch.Generator().manual_seed(1)
    q, dq, k, dk = (torch.randn(2, h, 5, 64, generator=g).to(FP16).to(dev) for h in (4, 4, 2, 2))
    pos = torch.arange(5, device=dev)
    freq, mag = ta.rotary_frequencies(64, scaling="yarn", factor=4.0, device=dev)
    how = dict(magnitude=mag, inverse=True)
    want_q, want_k = ta.rotary(q, k, pos, freq, **how)
    turned_q, turned_k = ta.rotary(dq, dk, pos, freq, **how)
    with fwad.dual_level():
        for with_q, with_k in ((True, True), (True, False), (False, True)):
            for leaf in (False, True):
                a = fwad.make_dual(q.clone().requires_grad_(leaf), dq) if with_q else q
                b = fwad.make_dual(k.clone().requires_grad_(leaf), dk) if with_k else k
                oq, ok = ta.rotary(a, b, pos, freq, **how)
                assert torch.equal(fwad.unpack_dual(oq).primal, want_q)
                assert torch.equal(fwad.unpack_dual(ok).primal, want_k)
                for out, has, want in ((oq, with_q, turned_q), (ok, with_k, turned_k)):
                    assert (_tangent(out) is not None) == has
                    assert not has or torch.equal(_tangent(out), want)
                assert (oq if with_q else ok).requires_grad == leaf
        out, none = ta.rotary(fwad.make_dual(q, dq), None, pos, freq, **how)
        assert none is None and torch.equal(_tangent(out), turned_q)
        with torch.no_grad():  # says nothing about forward mode
            out = ta.rotary(fwad.make_dual(q, dq), None, pos, freq, **how)[0]
        assert torch.equal(_tangent(out), turned_q)
        zero = fwad.make_dual(q, torch._efficientzerotensor(q.shape, dtype=q.dtype, device=dev))
        for other in (k, fwad.make_dual(k, dk)):
            oq, ok = ta.rotary(zero, other, pos, freq, **how)
            assert _tangent(oq) is None or not _tangent(oq).any()
            assert torch.equal(fwad.unpack_dual(oq).primal, want_q)
            assert other is k or torch.equal(_tangent(ok), turned_k)
        out = ta.rotary(q, k, pos, freq, **how)  # a level, but no tangent
        assert _tangent(out[0]) is None and torch.equal(out[0], want_q)
        # both modes: the gradient of the turned tangent, and of the value
        leaf, seed = q.clone().requires_grad_(), dq.clone().requires_grad_()
        out = ta.rotary(fwad.make_dual(leaf, seed), None, pos, freq, **how)[0]
        back = ta.rotary(dq, None, pos, freq, magnitude=mag)[0]
        assert torch.equal(torch.autograd.grad(_tangent(out), seed, dq, retain_graph=True)[0], back)
        assert torch.equal(torch.autograd.grad(fwad.unpack_dual(out).primal, leaf, dq)[0], back)


def test_tangents_on_the_host(plain_kernel):
    _check("cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("fast", [True, False])
def test_tangents(fast, monkeypatch):
    q = torch.zeros(1, 1, 1, 64, dtype=FP16, device="cuda:0")
    ta.rotary(q, None, torch.zeros(1, dtype=torch.int32, device="cuda:0"), ta.rotary_frequencies(64, device="cuda:0")[0])
    if not fast:
        monkeypatch.setattr(_native, "_fast", None)
    _check("cuda:0")
