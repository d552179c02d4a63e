"""A KV cache of bounded size: how much attention every key has received, and eviction of the keys with the least.

:func:`decode_weights` is a decode step that adds every key's share of attention to a running sum, :func:`key_weights` takes
the same sum for queries whose attention has already been computed (the last tokens of a prompt), and :func:`evict` cuts a cache to
a budget: the most recent keys stay, and of the others those with the largest sums.

The reference's cache only grows (probjax/nn/layers/attention.py:631-643, 727-757).
"""

from __future__ import annotations

import functools
import math

import torch

from . import _lib
from .attention import (_DTYPES, _IMPL, _as_tensor, _band_args, _check_call, _launch, _ptr, _refuse_grad, _require_gpu, _status_word,
                        _stream, _workspace, _written)
from .drafts import _int32
from .masks import AttentionMask, split_mask


def _weights_args(what, weights, out, shape, dev):
    """``(weights, out)`` as float32 tensors of ``shape``; ``out`` is made where it is not given."""
    for name, t in (("weights", weights), ("out", out)):
        if t is not None and (t.shape != shape or t.dtype is not torch.float32 or t.device != dev):
            raise ValueError(f"{what}: {name} must be float32 {list(shape)} on {dev}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    if out is None:
        out = torch.empty(shape, dtype=torch.float32, device=dev)
    elif not out.is_contiguous():
        raise ValueError(f"{what}: out must be contiguous")
    if weights is not None and weights.data_ptr() != out.data_ptr():
        a, b, n = weights.data_ptr(), out.data_ptr(), out.numel() * 4
        if weights.is_contiguous() and a < b + n and b < a + n:
            raise ValueError(f"{what}: weights and out overlap in part")
        weights = weights.contiguous()
    elif weights is not None and not weights.is_contiguous():
        raise ValueError(f"{what}: weights that are also the result must be contiguous")
    return weights, out


@functools.lru_cache(maxsize=256)
def _decode_workspace(*sizes) -> int:
    return _lib.lib().pjx_attn_decode_weights_workspace_bytes(*sizes)


def decode_weights(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, weights: torch.Tensor | None = None, *, kv_lengths=None,
                   sm_scale: float | None = None, split_len: int = 0, return_lse: bool = False, out: torch.Tensor | None = None):
    """Split-KV decode (as :func:`decode_forward`) that also returns ``weights`` plus what every key received of this step's
    attention, summed over the query tokens and the heads of its group (``pjx_attn_decode_weights``): ``q [B, Lq, Hq, D]`` over
    ``k_cache``, ``v_cache`` ``[B, capacity, Hkv, D]``, ``weights`` float32 ``[B, Hkv, capacity]`` (``None``: zeros).
    ``out`` takes the sum and may be ``weights`` itself.  Returns ``(o, out)`` or ``(o, lse, out)``; no gradient (inputs that ask for one
    are refused)."""
    _require_gpu()
    for t in (q, k_cache, v_cache):
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise ValueError("decode_weights takes CUDA tensors")
    B, Lq, cap, Hq, Hkv, D, Dv = _check_call(q, k_cache, v_cache, what="decode_weights")
    dev = q.device
    _refuse_grad("decode_weights", q, k_cache, v_cache, weights)
    lengths = None if kv_lengths is None else _int32(kv_lengths, dev, (B,), "kv_lengths")
    given = out
    weights, out = _weights_args("decode_weights", weights, out, (B, Hkv, cap), dev)
    q, k_cache, v_cache = q.contiguous(), k_cache.contiguous(), v_cache.contiguous()
    o = torch.empty((B, Lq, Hq, Dv), dtype=q.dtype, device=dev)
    lse = torch.empty((B, Hq, Lq), dtype=torch.float32, device=dev) if return_lse else None
    if Lq == 0:  # no query looks at a key
        if weights is None:
            out.zero_()
        elif weights.data_ptr() != out.data_ptr():
            out.copy_(weights)
        return (o, lse, out) if return_lse else (o, out)
    ws = _workspace(dev, "decode_weights", _decode_workspace(B, Lq, Hq, Hkv, Dv, cap, int(split_len)))
    _launch(dev.index, _lib.lib().pjx_attn_decode_weights, _ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(lengths), _ptr(weights), _ptr(out),
            _ptr(o), _ptr(lse), B, Lq, Hq, Hkv, D, Dv, cap, _DTYPES[q.dtype], 1.0 / math.sqrt(D) if sm_scale is None else float(sm_scale),
            int(split_len), _ptr(ws), ws.numel(), _ptr(_status_word(dev)), _stream(dev))
    if given is not None:
        _written(given)
    return (o, lse, out) if return_lse else (o, out)


def key_weights(q: torch.Tensor, k: torch.Tensor, lse: torch.Tensor, *, weights: torch.Tensor | None = None, mask: AttentionMask | None = None,
                sm_scale: float | None = None, out: torch.Tensor | None = None, implementation: str | None = None) -> torch.Tensor:
    """What every key received of an attention call that has been made (``pjx_attn_key_weights``): ``weights`` (float32
    ``[B, Hkv, Lkv]``, ``None``: zeros) plus the sum over the queries that see it of ``exp(sm_scale q.k - lse)``, with the call's own
    ``mask``, ``sm_scale`` (default ``1/sqrt(D)``) and natural-log ``lse [B, Hq, Lq]``; a row with ``lse = +inf`` adds nothing, whatever
    its query holds.  ``mask`` may hold key lengths and bands
    (causal, windows, bottom-right causal).  ``out`` takes the sum and may be ``weights`` itself.  No gradient (inputs that ask for one
    are refused)."""
    _require_gpu()
    if implementation not in _IMPL:
        raise ValueError(f"implementation must be None or one of {sorted(x for x in _IMPL if x)}")
    for t in (q, k, lse):
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise ValueError("key_weights takes CUDA tensors")
    B, Lq, Lkv, Hq, Hkv, D, _ = _check_call(q, k, k, lse=lse, what="key_weights")
    dev = q.device
    _refuse_grad("key_weights", q, k, lse, weights)
    if lse.device != dev or lse.dtype != torch.float32:
        raise ValueError(f"key_weights: lse must be float32 on {dev}")
    lm, residual = split_mask(mask, B, Lq, Lkv)
    if residual is not None or lm.structured or lm.q_limit is not None:
        raise NotImplementedError("key_weights takes masks of key lengths and bands (causal, windows)")
    lengths = None if lm.kv_lengths is None else _as_tensor(lm.kv_lengths).to(device=dev, dtype=torch.int32).contiguous()
    if lengths is not None and lengths.numel() != B:
        raise ValueError(f"key_weights: key lengths must hold B={B} entries, got {lengths.numel()}")
    given = out
    weights, out = _weights_args("key_weights", weights, out, (B, Hkv, Lkv), dev)
    q, k, lse = q.contiguous(), k.contiguous(), lse.contiguous()
    band_lo, band_hi = _band_args(False, lm.band)
    _launch(dev.index, _lib.lib().pjx_attn_key_weights, _ptr(q), _ptr(k), _ptr(lse), _ptr(weights), _ptr(out), _ptr(lengths), B, Lq, Lkv, Hq,
            Hkv, D, _DTYPES[q.dtype], band_lo, band_hi, 1.0 / math.sqrt(D) if sm_scale is None else float(sm_scale), _IMPL[implementation],
            _ptr(_status_word(dev)), _stream(dev))
    if given is not None:
        _written(given)
    return out


@functools.lru_cache(maxsize=256)
def _evict_workspace(*sizes) -> int:
    return _lib.lib().pjx_kv_cache_evict_workspace_bytes(*sizes)


def evict(k_cache: torch.Tensor, v_cache: torch.Tensor, weights: torch.Tensor, kv_lengths, keep: int, *, recent: int = 0, out=None,
          lengths_out: torch.Tensor | None = None):
    """Cut every sequence of a cache to ``keep`` keys per KV head (``pjx_kv_cache_evict``): the ``recent`` last ones and, of the
    others, those with the largest ``weights`` (float32 ``[B, Hkv, capacity]``; ties go to the lowest index, NaN ranks last).  Shorter
    sequences keep all.  The kept rows move to the front in their order: in place, or into ``out = (k, v, weights)`` of the same layout
    and a capacity of at least ``keep`` (rows behind the kept ones stay as they were there; free weights become 0).

    Keys keep the angles that a rotary embedding gave them, and the new lengths no longer count the tokens seen: positions of further tokens
    follow a count of the caller's own.  Results share no memory with each other; in place, ``v_cache`` may be ``k_cache``.

    Returns ``(lengths, kept)``: the new lengths ``int32 [B]`` (``lengths_out`` takes them and may be the tensor of
    ``kv_lengths``) and the kept keys' former indices ``int32 [B, Hkv, keep]``, ``-1`` behind them."""
    _require_gpu()
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dim() != 4:
            raise ValueError(f"evict takes rank-4 CUDA tensors; {name} is not one")
    dev = k_cache.device
    if k_cache.dtype not in _DTYPES:
        raise ValueError(f"unsupported dtype {k_cache.dtype}; expected float32, bfloat16 or float16")
    B, cap, Hkv, D = k_cache.shape
    Dv = v_cache.shape[3]
    if v_cache.shape[:3] != (B, cap, Hkv) or v_cache.dtype is not k_cache.dtype or v_cache.device != dev:
        raise ValueError(f"evict: v_cache must be [B={B}, capacity={cap}, Hkv={Hkv}, Dv] of the keys' dtype and device, got {tuple(v_cache.shape)}")
    keep, recent = int(keep), int(recent)
    if keep < 1 or not 0 <= recent <= keep:
        raise ValueError(f"evict: keep must be positive and recent in [0, keep], got keep={keep}, recent={recent}")
    lengths = _int32(kv_lengths, dev, (B,), "kv_lengths")
    ko, vo, wo = (k_cache, v_cache, weights) if out is None else out
    cap_out = ko.shape[1] if ko.dim() == 4 else -1
    for name, t, shape, dtype in (("weights", weights, (B, Hkv, cap), torch.float32), ("out keys", ko, (B, cap_out, Hkv, D), k_cache.dtype),
                                  ("out values", vo, (B, cap_out, Hkv, Dv), k_cache.dtype), ("out weights", wo, (B, Hkv, cap_out), torch.float32)):
        if t.shape != shape or t.dtype is not dtype or t.device != dev or not t.is_contiguous():
            raise ValueError(f"evict: {name} must be a contiguous {dtype} {list(shape)} on {dev}, got {t.dtype} {tuple(t.shape)}")
    if not k_cache.is_contiguous() or not v_cache.is_contiguous():
        raise ValueError("evict: the caches must be contiguous")
    given = lengths_out
    if lengths_out is None:
        lengths_out = torch.empty_like(lengths)
    elif tuple(lengths_out.shape) != (B,) or lengths_out.dtype != torch.int32 or lengths_out.device != dev or not lengths_out.is_contiguous():
        raise ValueError(f"evict: lengths_out must be a contiguous int32 [{B}] on {dev}")
    kept = torch.empty((B, Hkv, keep), dtype=torch.int32, device=dev)
    ws = _workspace(dev, "evict", _evict_workspace(B, Hkv))
    _launch(dev.index, _lib.lib().pjx_kv_cache_evict, _ptr(k_cache), _ptr(v_cache), _ptr(weights), _ptr(lengths), _ptr(ko), _ptr(vo), _ptr(wo),
            _ptr(lengths_out), _ptr(kept), B, Hkv, D, Dv, cap, cap_out, keep, recent, _DTYPES[k_cache.dtype], _ptr(ws), ws.numel(), _stream(dev))
    _written(ko, vo, wo, given)
    return lengths_out, kept
