"""Rotary positions for q and k, the step before sdpa in a decoder.

rotary(q, k, positions, inv_freq) turns every pair of dims of [B, H, S, D] tensors by the
angle position * inv_freq[i] in one kernel launch (csrc/rotary.cu), with a gradient;
rotary_frequencies() gives inv_freq and the magnitude for a base and a long-context scaling.
The reference has no positions; argument checks, errors and launches follow sdpa's.
"""

from __future__ import annotations

import math
from numbers import Real

from . import _native, _runtime
from ._errors import DTypeNotSupportedError, InvalidShapeError
from .launch import _NULL_CTX, _dtype_code, _raise_for, _raw_stream, _sync_mode, check_device_status
from .sdpa import _async_mode

SCALINGS = ("none", "linear", "ntk", "yarn", "bands")


def rotary_frequencies(rotary_dim: int, *, base: float = 10000.0, scaling: str = "none",
                       factor: float = 1.0, original_length: int = 8192, fast: float = 32.0,
                       slow: float = 1.0, device=None):
    """(inv_freq, magnitude) for rotary(): radians per position of each of the rotary_dim / 2
    pairs, float64 on `device`, and the factor on cos and sin.

    inv_freq[i] = base^(-2i / rotary_dim), changed for contexts `factor` times as long as the
    `original_length` that a model was trained on:

    "none"    as it is (factor is not used).
    "linear"  divided by factor: positions interpolated.
    "ntk"     the base times factor^(R / (R - 2)), which divides the slowest pair by factor and
              leaves the fastest.
    "yarn"    pairs that turn at least `fast` times over the original context keep their speed,
              those that turn at most `slow` times are divided by factor, a linear ramp in
              turns between, as the method's paper has it; magnitude 0.1 ln(factor) + 1. Many
              published checkpoints were made with a ramp linear in the pair's index, whose
              frequencies between differ (up to some 2 times): pass rotary() such a model's own
              inv_freq.
    "bands"   as "yarn" with magnitude 1.
    """
    torch_mod = _runtime.get_torch_module()
    if not isinstance(rotary_dim, int) or rotary_dim < 2 or rotary_dim % 2:
        raise InvalidShapeError("rotary_dim must be a positive even int.")
    if scaling not in SCALINGS:
        raise InvalidShapeError(f"scaling must be one of {', '.join(SCALINGS)}.")
    for name, value in (("base", base), ("factor", factor), ("original_length", original_length)):
        if not isinstance(value, Real) or not 0 < float(value) < math.inf:
            raise InvalidShapeError(f"{name} must be a positive number.")
    if not 0 < slow < fast:
        raise InvalidShapeError("slow and fast must be positive, slow the smaller.")
    base = float(base)
    if scaling == "ntk" and rotary_dim > 2:
        base *= float(factor) ** (rotary_dim / (rotary_dim - 2))
    i = torch_mod.arange(rotary_dim // 2, dtype=torch_mod.float64)
    freq = base ** (-2.0 * i / rotary_dim)
    magnitude = 1.0
    if scaling == "linear":
        freq = freq / factor
    elif scaling in ("yarn", "bands"):
        turns = original_length * freq / (2 * math.pi)
        keep = ((turns - slow) / (fast - slow)).clamp(0, 1)
        freq = freq * keep + freq / factor * (1 - keep)
        if scaling == "yarn":
            magnitude = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    return freq.to(device) if device is not None else freq, magnitude


def _check(torch_mod, q, k, positions, inv_freq):
    tensors = [("q", q)] + ([("k", k)] if k is not None else [])
    for name, t in tensors:
        if not isinstance(t, torch_mod.Tensor):
            raise InvalidShapeError(f"{name} must be a torch.Tensor.")
        if t.ndim != 4:
            raise InvalidShapeError(f"{name} must have shape [B, H, S, D].")
        if not t.is_cuda:
            raise InvalidShapeError(f"{name} must be a CUDA tensor.")
    for name, t in (("positions", positions), ("inv_freq", inv_freq)):
        if not isinstance(t, torch_mod.Tensor):
            raise InvalidShapeError(f"{name} must be a torch.Tensor.")
        if t.device != q.device:
            raise InvalidShapeError(f"{name} must be on q's device.")
    batch, _, seq, dim = q.shape
    if k is not None:
        if k.device != q.device:
            raise InvalidShapeError("q and k must be on the same CUDA device.")
        if k.shape[0] != batch or k.shape[2] != seq or k.shape[3] != dim:
            raise InvalidShapeError("q and k must agree in batch, sequence and head dim.")
    if q.dtype not in (torch_mod.float16, torch_mod.bfloat16):
        raise DTypeNotSupportedError("q dtype must be torch.float16 or torch.bfloat16.")
    if k is not None and k.dtype != q.dtype:
        raise DTypeNotSupportedError("q and k must have identical dtype.")
    if positions.dtype not in (torch_mod.int32, torch_mod.int64):
        raise DTypeNotSupportedError("positions dtype must be torch.int32 or torch.int64.")
    if inv_freq.dtype != torch_mod.float64:
        raise DTypeNotSupportedError("inv_freq dtype must be torch.float64.")
    shape = tuple(positions.shape)
    if shape != (seq,) and shape != (batch, seq) and shape != (1, seq):
        raise InvalidShapeError("positions must have shape [S], [1, S] or [B, S].")
    if inv_freq.ndim != 1 or not 2 <= 2 * inv_freq.shape[0] <= dim:
        raise InvalidShapeError("inv_freq must have shape [R / 2] with R at most the head dim.")


def run_rotary(q, k, positions, inv_freq, interleaved, magnitude, inverse):
    """Launches the kernel on checked inputs; returns new contiguous (q, k)."""
    torch_mod = _runtime.get_torch_module()
    lib = _runtime.get_native_library()
    outs = [None if t is None else torch_mod.empty(t.shape, dtype=t.dtype, device=t.device)
            for t in (q, k)]
    if q.numel() == 0 and (k is None or k.numel() == 0):
        return outs
    mode = _sync_mode()
    if q.numel() == 0:  # no query heads: k takes the first place
        outs[1] = run_rotary(k, None, positions, inv_freq, interleaved, magnitude, inverse)[0]
        return outs
    has_k = k is not None and k.numel() > 0
    q, k = (t if t is None or t.stride(3) == 1 or t.shape[3] == 1 else t.contiguous()
            for t in (q, k))
    inv_freq = inv_freq.contiguous()
    batch, heads, seq, dim = q.shape
    pos_strides = (0 if positions.ndim == 1 or positions.shape[0] == 1 else positions.stride(0),
                   positions.stride(-1))
    with torch_mod.cuda.device(q.device) if q.device.index != torch_mod.cuda.current_device() else _NULL_CTX:
        stream = _raw_stream(torch_mod, q.device.index)
        if mode == "strict":
            torch_mod.cuda.synchronize(q.device)

        def strides(t):
            return _native.strides4((*t.stride()[:3], 1))

        rc = lib.ta_rotary(
            q.data_ptr(), outs[0].data_ptr(), strides(q), strides(outs[0]), heads,
            k.data_ptr() if has_k else None, outs[1].data_ptr() if has_k else None,
            strides(k) if has_k else None, strides(outs[1]) if has_k else None,
            k.shape[1] if has_k else 0, batch, seq, dim, 2 * inv_freq.shape[0],
            positions.data_ptr(), int(positions.dtype == torch_mod.int64),
            _native.strides4((*pos_strides, 0, 0)), inv_freq.data_ptr(), int(interleaved),
            int(inverse), magnitude, _dtype_code(torch_mod, q.dtype), stream)
        if rc != _native.TA_OK:
            _raise_for(lib, rc)
        if mode in ("post", "strict"):
            check_device_status(q.device)
    return outs


def _fast_launch(q, k, positions, inv_freq, interleaved, magnitude, inverse):
    """The one-call native launcher, which differentiates too, or None (an argument is not as it
    should be, or the launcher is not there): see sdpa._fast_launch."""
    fast = _native._fast
    if fast is None or not _runtime._runtime_ready or not _async_mode():
        return None
    return fast.rotary(q, k, positions, inv_freq, interleaved, magnitude, inverse)


_function = None


def _autograd_function():
    """The autograd function of the Python path (made once torch is there): the gradient turns
    the other way."""
    global _function
    if _function is not None:
        return _function
    torch_mod = _runtime.get_torch_module()

    class Rotary(torch_mod.autograd.Function):
        @staticmethod
        def forward(ctx, q, k, positions, inv_freq, interleaved, magnitude, inverse):
            ctx.save_for_backward(positions, inv_freq)
            ctx.set_materialize_grads(False)
            ctx.how = (interleaved, magnitude, inverse)
            out_q, out_k = run_rotary(q, k, positions, inv_freq, interleaved, magnitude, inverse)
            return out_q if k is None else (out_q, out_k)

        @staticmethod
        def backward(ctx, grad_q, grad_k=None):
            positions, inv_freq = ctx.saved_tensors
            interleaved, magnitude, inverse = ctx.how
            rest = (positions, inv_freq, interleaved, magnitude, not inverse)
            # A gradient that nobody needs, or that never came, costs nothing.
            need_q = ctx.needs_input_grad[0] and grad_q is not None
            need_k = ctx.needs_input_grad[1] and grad_k is not None
            if need_q and need_k:
                grad_q, grad_k = Rotary.apply(grad_q, grad_k, *rest)
            elif need_q:
                grad_q = Rotary.apply(grad_q, None, *rest)
            elif need_k:
                grad_k = Rotary.apply(grad_k, None, *rest)
            return (grad_q if need_q else None, grad_k if need_k else None, *[None] * 5)

    _function = Rotary
    return Rotary


def _forward_mode(torch_mod, q, k, positions, inv_freq, **how):
    """(q, k) turned with their tangents, which a linear map takes to the tangents' own rotation;
    None where neither carries one."""
    fwad = torch_mod.autograd.forward_ad
    if not torch_mod._C._is_fwd_grad_enabled():
        return None
    (q, dq), (k, dk) = (fwad.unpack_dual(t) if t is not None else (None, None) for t in (q, k))
    dual = dq is not None or dk is not None
    # torch's tangents of zero may have no memory to read; a zero turns into a zero, which is none
    dq, dk = (None if d is None or d._is_zerotensor() else d for d in (dq, dk))
    if dq is None and dk is None:
        return rotary(q, k, positions, inv_freq, **how) if dual else None
    q, k = rotary(q, k, positions, inv_freq, **how)
    if dq is not None:
        dq, dk = rotary(dq, dk, positions, inv_freq, **how)
    else:
        dk = rotary(dk, None, positions, inv_freq, **how)[0]
    return tuple(t if d is None else fwad.make_dual(t, d) for t, d in ((q, dq), (k, dk)))


def rotary(q, k, positions, inv_freq, *, interleaved: bool = False, magnitude: float = 1.0,
           inverse: bool = False):
    """Rotary positions: (q, k) with every pair of dims turned by position * inv_freq.

    q, k:        [B, H, S, D] and [B, Hk, S, D] CUDA tensors, float16 or bfloat16, any strides;
                 k may be None (the result is then (q, None)).
    positions:   int32 or int64 [S], [1, S] or [B, S] on q's device.
    inv_freq:    float64 [R / 2], radians per position (rotary_frequencies()); dims from R on
                 are copied.
    interleaved: pairs are dims (2i, 2i + 1) instead of (i, R / 2 + i).
    magnitude:   factor on the turned dims.
    inverse:     turn the other way (what the gradient does).

    Returns new contiguous tensors, computed asynchronously on the current torch stream;
    differentiable in q and k, in reverse mode (twice too) and in forward mode. positions and
    inv_freq are constants to it.
    """
    out = _fast_launch(q, k, positions, inv_freq, interleaved, magnitude, inverse)
    if out is not None:
        return out
    for name, value in (("interleaved", interleaved), ("inverse", inverse)):
        if not isinstance(value, bool):
            raise InvalidShapeError(f"{name} must be a bool.")
    if not isinstance(magnitude, Real) or not math.isfinite(magnitude):
        raise InvalidShapeError("magnitude must be a finite number.")
    _runtime.require_supported_runtime()
    torch_mod = _runtime.get_torch_module()
    _check(torch_mod, q, k, positions, inv_freq)
    magnitude = float(magnitude)
    if torch_mod.autograd.forward_ad._current_level >= 0:
        out = _forward_mode(torch_mod, q, k, positions, inv_freq, interleaved=interleaved,
                            magnitude=magnitude, inverse=inverse)
        if out is not None:
            return out
    if torch_mod.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        out = _autograd_function().apply(q, k, positions, inv_freq, interleaved, magnitude, inverse)
        return (out, None) if k is None else out
    q_out, k_out = run_rotary(q, k, positions, inv_freq, interleaved, magnitude, inverse)
    return q_out, k_out
