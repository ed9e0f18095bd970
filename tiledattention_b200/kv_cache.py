"""The paged 8-bit key/value cache and attention over it: what takes sdpa's place once a
decoder generates tokens.

A cache holds e4m3 codes in pages [P, Hkv, page, D] with one float32 scale (a power of two where
it is written here) for each (page, head); a page table [B, width] says which page holds which tokens of a sequence.
kv_cache_append() writes new tokens (csrc/kv8_append.cu), sdpa_kv_cache() attends to the cached
ones (csrc/sdpa_kv8.cu). The reference has no cache; argument checks, errors and launches
follow sdpa's.
"""

from __future__ import annotations

import math
from numbers import Real
from typing import Any, NamedTuple

from . import _native, _runtime
from ._errors import DTypeNotSupportedError, InvalidShapeError
from .launch import (
    _NULL_CTX,
    _dtype_code,
    _raise_for,
    _raw_stream,
    _status_word,
    _sync_mode,
    _tma_compatible,
    check_device_status,
)
from .sdpa import _async_mode

PAGE_SIZES = (16, 32, 64, 128)


class KVCache8(NamedTuple):
    """Storage of an 8-bit cache (one layer's): torch tensors that the caller owns.

    k, v:             float8_e4m3fn [P, Hkv, page, D], contiguous.
    k_scale, v_scale: float32 [P, Hkv], contiguous, zero or from 2^-50 to 2^50; the values of a
                      page are its codes times its scale. kv_cache_append writes powers of two,
                      pages filled elsewhere may have others.
    """

    k: Any
    v: Any
    k_scale: Any
    v_scale: Any


def kv_cache_alloc(num_pages: int, num_heads: int, page_size: int, head_dim: int, *,
                   device=None) -> KVCache8:
    """An empty cache: codes of zero, scales of one."""
    torch_mod = _runtime.get_torch_module()
    for name, value in (("num_pages", num_pages), ("num_heads", num_heads)):
        if not isinstance(value, int) or value < 1:
            raise InvalidShapeError(f"{name} must be a positive int.")
    _check_page(page_size, head_dim)
    device = torch_mod.device("cuda" if device is None else device)
    shape = (num_pages, num_heads, page_size, head_dim)
    codes = [torch_mod.zeros(shape, dtype=torch_mod.uint8, device=device).view(
        torch_mod.float8_e4m3fn) for _ in range(2)]
    scales = [torch_mod.ones(shape[:2], dtype=torch_mod.float32, device=device) for _ in range(2)]
    return KVCache8(*codes, *scales)


def _check_page(page_size, head_dim):
    if page_size not in PAGE_SIZES:
        raise InvalidShapeError("the cache's page size must be 16, 32, 64 or 128.")
    if not isinstance(head_dim, int) or not 16 <= head_dim <= 256 or head_dim % 16:
        raise InvalidShapeError("the cache's head dim must be a multiple of 16 up to 256.")


def _check_cache(torch_mod, cache, device):
    if not isinstance(cache, tuple) or len(cache) != 4:
        raise InvalidShapeError("cache must be a KVCache8.")
    k, v, k_scale, v_scale = cache
    for name, t in (("k", k), ("v", v), ("k_scale", k_scale), ("v_scale", v_scale)):
        if not isinstance(t, torch_mod.Tensor):
            raise InvalidShapeError(f"cache.{name} must be a torch.Tensor.")
        if t.device != device:
            raise InvalidShapeError(f"cache.{name} must be on the other tensors' CUDA device.")
        if not t.is_contiguous():
            raise InvalidShapeError(f"cache.{name} must be contiguous.")
        if t.requires_grad:
            raise InvalidShapeError(f"cache.{name} must not require a gradient.")
    if k.dtype != torch_mod.float8_e4m3fn or v.dtype != torch_mod.float8_e4m3fn:
        raise DTypeNotSupportedError("cache.k and cache.v dtype must be torch.float8_e4m3fn.")
    if k_scale.dtype != torch_mod.float32 or v_scale.dtype != torch_mod.float32:
        raise DTypeNotSupportedError("cache scales' dtype must be torch.float32.")
    if k.ndim != 4 or v.shape != k.shape or k.numel() == 0:
        raise InvalidShapeError("cache.k and cache.v must have one shape [P, Hkv, page, D].")
    if k_scale.shape != k.shape[:2] or v_scale.shape != k.shape[:2]:
        raise InvalidShapeError("cache scales must have shape [P, Hkv].")
    if k.data_ptr() % 16 or v.data_ptr() % 16:
        raise InvalidShapeError("cache.k and cache.v must be 16-byte aligned.")
    _check_page(int(k.shape[2]), int(k.shape[3]))


def _check_ints(torch_mod, name, t, shape, device):
    if not isinstance(t, torch_mod.Tensor):
        raise InvalidShapeError(f"{name} must be a torch.Tensor.")
    if t.dtype != torch_mod.int32:
        raise DTypeNotSupportedError(f"{name} dtype must be torch.int32.")
    if t.device != device:
        raise InvalidShapeError(f"{name} must be on the other tensors' CUDA device.")
    if t.ndim != len(shape) or any(n is not None and t.shape[i] != n for i, n in enumerate(shape)):
        raise InvalidShapeError(f"{name} must have shape "
                                f"{'[B, width]' if len(shape) == 2 else '[B]'}.")


def _check_table(torch_mod, table, batch, device):
    _check_ints(torch_mod, "page_table", table, (batch, None), device)
    if table.shape[1] < 1 and batch > 0:
        raise InvalidShapeError("page_table must have at least one column.")


def _rows(t):
    """The tensor itself where a row of it is 16-byte vectors, else a contiguous copy."""
    return t if _tma_compatible(t) and all(s >= 0 for s in t.stride()) else t.clone(
        memory_format=_runtime.get_torch_module().contiguous_format)


def _table_rows(t):
    """The table itself where its rows are runs of ints side by side or apart, else a copy (of a
    row expanded over the batch, too)."""
    apart = t.shape[0] == 1 or t.stride(0) >= t.shape[1]
    return t if t.stride(1) == 1 and apart else t.contiguous()


def _device_of(torch_mod, t):
    same = t.device.index == torch_mod.cuda.current_device()
    return _NULL_CTX if same else torch_mod.cuda.device(t.device)


def kv_cache_append(k, v, cache: KVCache8, page_table, starts, *, counts=None) -> None:
    """Writes new tokens into an 8-bit cache, in place.

    k, v:       [B, Hkv, T, D] CUDA tensors, float16 or bfloat16.
    cache:      KVCache8 with Hkv heads and head dim D.
    page_table: int32 [B, width]: token i of sequence b is row i % page of page
                page_table[b, i // page].
    starts:     int32 [B]: tokens each sequence holds already; its new ones follow.
    counts:     int32 [B], how many of the T tokens are real (None: all); the others are not read.

    A page whose first row is written begins anew, with the least power-of-two scale that holds
    its tokens; one that holds tokens keeps the larger of its scale and the needed one, and where
    that grows its old codes are rounded again. Values round to nearest even; infinities
    saturate, NaN stays NaN, and neither raises a scale. Rows behind the last new token stay as
    they are.

    Runs asynchronously on the current torch stream. Page ids outside the cache are skipped, and
    starts and counts outside their range held in range: both are reported by
    check_device_status(). Pages that two sequences, or two slots of one, write in one call have no
    defined content.
    """
    fast = _native._fast
    if fast is not None and _runtime._runtime_ready and _async_mode() and type(cache) is KVCache8:
        if fast.kv8_append(k, v, *cache, page_table, starts, counts):
            return
    _runtime.require_supported_runtime()
    torch_mod = _runtime.get_torch_module()
    for name, t in (("k", k), ("v", v)):
        if not isinstance(t, torch_mod.Tensor):
            raise InvalidShapeError(f"{name} must be a torch.Tensor.")
        if t.ndim != 4:
            raise InvalidShapeError(f"{name} must have shape [B, H, S, D].")
        if not t.is_cuda:
            raise InvalidShapeError(f"{name} must be a CUDA tensor.")
    if k.shape != v.shape:
        raise InvalidShapeError("k and v must have matching shape [B, H, S, D].")
    if k.device != v.device:
        raise InvalidShapeError("k and v must be on the same CUDA device.")
    if k.dtype not in (torch_mod.float16, torch_mod.bfloat16):
        raise DTypeNotSupportedError("k dtype must be torch.float16 or torch.bfloat16.")
    if k.dtype != v.dtype:
        raise DTypeNotSupportedError("k and v must have identical dtype.")
    _check_cache(torch_mod, cache, k.device)
    batch, heads, tokens, dim = (int(x) for x in k.shape)
    if heads != cache[0].shape[1] or dim != cache[0].shape[3]:
        raise InvalidShapeError("k and v must have the cache's heads and head dim.")
    _check_table(torch_mod, page_table, batch, k.device)
    _check_ints(torch_mod, "starts", starts, (batch,), k.device)
    if counts is not None:
        _check_ints(torch_mod, "counts", counts, (batch,), k.device)
    run_kv_cache_append(k, v, cache, page_table, starts, counts)


def run_kv_cache_append(k, v, cache, page_table, starts, counts):
    """Launches the append kernel on checked inputs."""
    torch_mod = _runtime.get_torch_module()
    lib = _runtime.get_native_library()
    mode = _sync_mode()
    if k.numel() == 0:
        return
    k, v = _rows(k.detach()), _rows(v.detach())
    page_table = _table_rows(page_table)
    starts = starts.contiguous()
    counts = counts.contiguous() if counts is not None else None
    batch, heads, tokens, dim = (int(x) for x in k.shape)
    with _device_of(torch_mod, k):
        status = _status_word(torch_mod, k.device)
        stream = _raw_stream(torch_mod, k.device.index)
        if mode == "strict":
            torch_mod.cuda.synchronize(k.device)
        rc = lib.ta_kv8_append(
            k.data_ptr(), v.data_ptr(), _native.strides4(k.stride()), _native.strides4(v.stride()),
            *(t.data_ptr() for t in cache), int(cache[0].shape[0]), int(cache[0].shape[2]),
            page_table.data_ptr(), page_table.stride(0), int(page_table.shape[1]),
            starts.data_ptr(), counts.data_ptr() if counts is not None else None,
            batch, heads, tokens, dim, _dtype_code(torch_mod, k.dtype), status.data_ptr(), stream)
        if rc != _native.TA_OK:
            _raise_for(lib, rc)
        if mode in ("post", "strict"):
            check_device_status(k.device)


def sdpa_kv_cache(q, cache: KVCache8, page_table, lengths, *, counts=None, causal: bool = True,
                  scale: float | None = None, return_lse: bool = False):
    """Attention of new tokens over an 8-bit cache: softmax(scale q K^T + mask) V.

    q:          [B, Hq, T, D] CUDA tensor, float16 or bfloat16; Hq a multiple of the cache's
                heads, at most 256 times them (query head h reads cache head
                h // (Hq / Hkv)).
    cache:      KVCache8 whose pages hold the tokens, the new ones among them.
    page_table: int32 [B, width], as in kv_cache_append.
    lengths:    int32 [B]: tokens of each sequence in the cache; 0 for an unused row.
    counts:     int32 [B], how many of the T query rows are real (None: all). They are the
                sequence's last tokens.
    causal:     row t sees the keys up to its own position, lengths[b] - counts[b] + t
                (bottom-right); else all lengths[b].
    scale:      positive float; defaults to 1/sqrt(D).

    Returns a new [B, Hq, T, D] tensor of q's dtype (with return_lse also the float32
    [B, Hq, T] natural-log log-sum-exp), computed asynchronously on the current torch stream.
    Rows that see no key, and rows from counts[b] on, are 0 with lse -inf. Not differentiable.
    Tokens of page ids outside the cache are left out, and lengths and counts outside their range
    held in range: both are reported by check_device_status().
    """
    fast = _native._fast
    # -1.0 is the launcher's code for the default scale: a caller's own must be positive.
    if (fast is not None and _runtime._runtime_ready and _async_mode() and type(cache) is KVCache8
            and (scale is None or (scale.__class__ is float and scale > 0))):
        out = fast.sdpa_kv8(q, *cache, page_table, lengths, counts, causal,
                            -1.0 if scale is None else scale, return_lse)
        if out is not None:
            return out
    for name, value in (("causal", causal), ("return_lse", return_lse)):
        if not isinstance(value, bool):
            raise InvalidShapeError(f"{name} must be a bool.")
    if scale is not None and (not isinstance(scale, Real) or not 0 < float(scale) < math.inf):
        raise InvalidShapeError("scale must be a positive number when provided.")
    _runtime.require_supported_runtime()
    torch_mod = _runtime.get_torch_module()
    if not isinstance(q, torch_mod.Tensor):
        raise InvalidShapeError("q must be a torch.Tensor.")
    if q.ndim != 4:
        raise InvalidShapeError("q must have shape [B, H, S, D].")
    if not q.is_cuda:
        raise InvalidShapeError("q must be a CUDA tensor.")
    if q.dtype not in (torch_mod.float16, torch_mod.bfloat16):
        raise DTypeNotSupportedError("q dtype must be torch.float16 or torch.bfloat16.")
    _check_cache(torch_mod, cache, q.device)
    batch, heads, _, dim = (int(x) for x in q.shape)
    if dim != cache[0].shape[3]:
        raise InvalidShapeError("q must have the cache's head dim.")
    if heads % int(cache[0].shape[1]):
        raise InvalidShapeError("q's heads must be a multiple of the cache's heads.")
    _check_table(torch_mod, page_table, batch, q.device)
    _check_ints(torch_mod, "lengths", lengths, (batch,), q.device)
    if counts is not None:
        _check_ints(torch_mod, "counts", counts, (batch,), q.device)
    return run_sdpa_kv_cache(q, cache, page_table, lengths, counts, causal,
                             float(scale) if scale is not None else 1.0 / math.sqrt(dim), return_lse)


def run_sdpa_kv_cache(q, cache, page_table, lengths, counts, causal, scale, return_lse):
    """Launches the attention kernel on checked inputs."""
    torch_mod = _runtime.get_torch_module()
    lib = _runtime.get_native_library()
    mode = _sync_mode()
    batch, heads, tokens, dim = (int(x) for x in q.shape)
    out = torch_mod.empty((batch, heads, tokens, dim), dtype=q.dtype, device=q.device)
    lse = torch_mod.empty((batch, heads, tokens), dtype=torch_mod.float32,
                          device=q.device) if return_lse else None
    if out.numel() == 0:
        return (out, lse) if return_lse else out
    q = _rows(q.detach())
    page_table = _table_rows(page_table)
    lengths = lengths.contiguous()
    counts = counts.contiguous() if counts is not None else None
    kv_heads = int(cache[0].shape[1])
    with _device_of(torch_mod, q):
        status = _status_word(torch_mod, q.device)
        stream = _raw_stream(torch_mod, q.device.index)
        if mode == "strict":
            torch_mod.cuda.synchronize(q.device)
        nbytes = lib.ta_sdpa_kv8_workspace(batch, heads, kv_heads, tokens, dim)
        work = torch_mod.empty(nbytes, dtype=torch_mod.uint8, device=q.device)
        rc = lib.ta_sdpa_kv8(
            q.data_ptr(), _native.strides4(q.stride()), out.data_ptr(),
            _native.strides4(out.stride()), lse.data_ptr() if return_lse else None,
            *(t.data_ptr() for t in cache), int(cache[0].shape[0]), int(cache[0].shape[2]),
            page_table.data_ptr(), page_table.stride(0), int(page_table.shape[1]),
            lengths.data_ptr(), counts.data_ptr() if counts is not None else None,
            batch, heads, kv_heads, tokens, dim, _dtype_code(torch_mod, q.dtype),
            1 if causal else 0, scale, work.data_ptr(), nbytes, status.data_ptr(), stream)
        if rc != _native.TA_OK:
            _raise_for(lib, rc)
        if mode in ("post", "strict"):
            check_device_status(q.device)
    return (out, lse) if return_lse else out
