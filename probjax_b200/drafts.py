"""Drafted tokens over a KV cache: the verification step of speculative decoding.

A draft model proposes a tree of tokens behind every sequence's context; one call of :func:`decode_tree` attends for all of them
(each draft sees the cached context and its ancestors), and :func:`accept_drafts` moves the keys and values of the accepted path
into the cache.  The drafts' keys and values live beside the cache, so rejected ones leave nothing to undo.

The reference decodes one token at a time (probjax/nn/layers/attention.py:603-675); this is the several-token form of its
decode branch for a ragged batch.
"""

from __future__ import annotations

import functools
import math

import torch

from . import _lib
from .attention import _DTYPES, _IMPL, _launch, _ptr, _refuse_grad, _require_gpu, _status_word, _stream, _workspace, _written


def _token_rows(t: torch.Tensor):
    """``(tensor, sequence stride, token stride)`` of a ``[B, N, H, D]`` tensor whose heads are dense, in elements: a slice
    of a fused projection is taken as it is, anything the kernels cannot address is copied."""
    B, N, H, D = t.shape
    if t.is_contiguous() and t.data_ptr() % 16 == 0:
        return t, N * H * D, H * D
    es = t.element_size()
    bs, ts = t.stride(0), t.stride(1)
    dense = (t.stride(3) == 1 or D == 1) and (t.stride(2) == D or H == 1)
    if not dense or (N > 1 and (ts < H * D or ts * es % 16)) or (B > 1 and (bs < H * D or bs * es % 16)):
        t = t.contiguous()
        bs, ts = t.stride(0), t.stride(1)
    if t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
        bs, ts = t.stride(0), t.stride(1)
    return t, (bs if B > 1 else N * H * D), (ts if N > 1 else H * D)


def _int32(x, device, shape, what):
    if isinstance(x, torch.Tensor) and x.dtype is torch.int32 and x.shape == shape and x.device == device and x.is_contiguous():
        return x
    t = torch.as_tensor(x)
    if t.is_floating_point() or t.is_complex() or t.dtype == torch.bool:
        raise ValueError(f"{what} must hold integers, got {t.dtype}")
    if t.dtype not in (torch.int32, torch.int16, torch.int8, torch.uint8):  # (wrapped to 32 bits, a number far out of range might be in range)
        t = t.to(torch.int64).clamp(-2 ** 31, 2 ** 31 - 1)
    t = t.to(device=device, dtype=torch.int32).contiguous()
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{what} must be {list(shape)}, got {tuple(t.shape)}")
    return t


def _check_cache(name, k_new, v_new, k_cache, v_cache, block_table):
    """Shapes, types and devices of drafts beside a cache: ``(B, N, Hkv, D, Dv, capacity, page_size, max_pages, num_pages, table)``."""
    dtype = getattr(k_new, "dtype", None)
    for what, t in (("k_new", k_new), ("v_new", v_new), ("k_cache", k_cache), ("v_cache", v_cache)):
        if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dim() != 4:
            raise ValueError(f"{name} takes rank-4 CUDA tensors; {what} is not one")
        if t.dtype is not dtype or t.get_device() != k_new.get_device():
            raise ValueError(f"{name}: all tensors must share a dtype and a device")
    if dtype not in _DTYPES:
        raise ValueError(f"unsupported dtype {dtype}; expected float32, bfloat16 or float16")
    B, N, Hkv, D = k_new.shape
    vb, vn, vh, Dv = v_new.shape
    if (vb, vn, vh) != (B, N, Hkv):
        raise ValueError(f"{name}: v_new must be [B={B}, N={N}, Hkv={Hkv}, Dv], got {tuple(v_new.shape)}")
    rows, cap, kh, kd = k_cache.shape
    if (kh, kd) != (Hkv, D) or v_cache.shape != (rows, cap, Hkv, Dv):
        raise ValueError(f"{name}: caches must be [.., .., Hkv={Hkv}, D={D}] and [.., .., Hkv={Hkv}, Dv={Dv}] alike, got "
                         f"{tuple(k_cache.shape)} and {tuple(v_cache.shape)}")
    if block_table is None:
        if rows != B:
            raise ValueError(f"{name}: the cache holds {rows} sequences, the drafts {B}")
        return B, N, Hkv, D, Dv, cap, 0, 0, 0, None
    table = torch.as_tensor(block_table)
    if table.dim() != 2 or table.shape[0] != B:
        raise ValueError(f"block_table must be [B={B}, max_pages], got {tuple(table.shape)}")
    table = _int32(table, k_new.device, table.shape, "block_table")
    return B, N, Hkv, D, Dv, table.shape[1] * cap, cap, table.shape[1], rows, table


@functools.lru_cache(maxsize=256)
def _tree_workspace(*sizes) -> int:
    return _lib.lib().pjx_attn_decode_tree_workspace_bytes(*sizes)


def decode_tree(q: torch.Tensor, k_new: torch.Tensor, v_new: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, parents, *,
                kv_lengths, block_table=None, sm_scale: float | None = None, return_lse: bool = False,
                implementation: str | None = None):
    """Attention of drafted tokens ``q [B, N, Hq, D]`` over a cache (``pjx_attn_decode_tree``): draft ``i`` of a sequence
    sees its ``kv_lengths[b]`` cached keys, itself and its ancestors.  ``parents`` (``[N]`` shared, or ``[B, N]``) holds ``-1`` for
    a draft right behind the context, the index of an earlier draft otherwise, and any other value where there is none
    (padding: zero output, ``lse = +inf``).  ``k_new`` / ``v_new`` ``[B, N, Hkv, D]`` are the drafts' keys and values;
    the cache is contiguous ``[B, capacity, Hkv, D]`` or, with ``block_table [B, max_pages]``, a page pool
    ``[num_pages, page_size, Hkv, D]`` with a page size that is a multiple of 16.  At most 256 drafts a sequence.

    A chain of drafts is ``parents = arange(N) - 1``.  Positions for a rotary embedding (:func:`probjax_b200.rope_axes`) are the tokens that
    the sequence has seen plus ``depth``: ``kv_lengths + depth`` as long as no key has been evicted, a count of the caller's own after that.
    A NaN or an infinity in the value of a draft that is there reaches the others too (0 times it is NaN); absent drafts may hold anything.  Returns ``o [B, N, Hq, Dv]`` and, with ``return_lse``, ``lse [B, Hq, N]``; no gradient (inputs
    that ask for one are refused)."""
    _require_gpu()
    if implementation not in _IMPL:
        raise ValueError(f"implementation must be None or one of {sorted(k for k in _IMPL if k)}")
    B, N, Hkv, D, Dv, cap, page, max_pages, num_pages, table = _check_cache("decode_tree", k_new, v_new, k_cache, v_cache, block_table)
    dev = k_new.device
    if not isinstance(q, torch.Tensor) or q.dim() != 4 or q.device != dev or q.dtype is not k_new.dtype:
        raise ValueError("decode_tree: q must be a rank-4 tensor of the drafts' dtype and device")
    Hq = q.shape[2]
    if q.shape != (B, N, Hq, D):
        raise ValueError(f"decode_tree: q must be [B={B}, N={N}, Hq, D={D}], got {tuple(q.shape)}")
    if Hq < 1 or Hkv < 1 or Hq % Hkv != 0:
        raise ValueError(f"query heads ({Hq}) must be a multiple of key/value heads ({Hkv})")
    _refuse_grad("decode_tree", q, k_new, v_new, k_cache, v_cache)
    lengths = _int32(kv_lengths, dev, (B,), "kv_lengths")
    if not isinstance(parents, torch.Tensor):
        parents = torch.as_tensor(parents)
    tree = _int32(parents, dev, (N,) if parents.dim() == 1 else (B, N), "parents")
    q, qb, qt = _token_rows(q)
    k_new, kb, kt = _token_rows(k_new)
    v_new, vb, vt = _token_rows(v_new)
    k_cache, v_cache = k_cache.contiguous(), v_cache.contiguous()
    o = torch.empty((B, N, Hq, Dv), dtype=q.dtype, device=dev)
    lse = torch.empty((B, Hq, N), dtype=torch.float32, device=dev) if return_lse else None
    ws = _workspace(dev, "tree", _tree_workspace(B, N, Hq, Hkv, Dv, cap))
    _launch(dev.index, _lib.lib().pjx_attn_decode_tree, _ptr(q), qb, qt, _ptr(k_new), kb, kt, _ptr(v_new), vb, vt, _ptr(k_cache),
            _ptr(v_cache), _ptr(tree), 0 if tree.dim() == 1 else N, _ptr(lengths), _ptr(table), _ptr(o), _ptr(lse), B, N, Hq, Hkv, D, Dv, cap,
            page, max_pages, num_pages, _DTYPES[q.dtype], 1.0 / math.sqrt(D) if sm_scale is None else float(sm_scale), _IMPL[implementation],
            _ptr(ws), ws.numel(), _ptr(_status_word(dev)), _stream(dev))
    return (o, lse) if return_lse else o


def accept_drafts(k_new: torch.Tensor, v_new: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, path, counts, *, kv_lengths,
                  block_table=None, out: torch.Tensor | None = None, overflow: torch.Tensor | None = None) -> torch.Tensor:
    """Put the accepted drafts into the cache, in place (``pjx_kv_cache_accept``): draft ``path[b, i]`` of ``k_new`` /
    ``v_new`` becomes row ``kv_lengths[b] + i`` for ``i < counts[b]``.  Returns the new lengths ``int32 [B]`` (at most the
    capacity); ``out`` may be the tensor of ``kv_lengths`` itself, so that a captured step advances it on the device.
    ``overflow`` (int32, one entry) is set to 1 where a sequence ran past the capacity."""
    _require_gpu()
    B, N, Hkv, D, Dv, cap, page, max_pages, num_pages, table = _check_cache("accept_drafts", k_new, v_new, k_cache, v_cache, block_table)
    dev = k_new.device
    if not k_cache.is_contiguous() or not v_cache.is_contiguous():
        raise ValueError("accept_drafts writes the caches in place: they must be contiguous")
    lengths = _int32(kv_lengths, dev, (B,), "kv_lengths")
    if not isinstance(path, torch.Tensor):
        path = torch.as_tensor(path)
    if path.dim() != 2:
        raise ValueError(f"path must be [B={B}, P], got {tuple(path.shape)}")
    path = _int32(path, dev, (B, path.shape[1]), "path")
    counts = _int32(counts, dev, (B,), "counts")
    given = out
    if out is None:
        out = torch.empty_like(lengths)
    for what, t, n in (("out", given, B), ("overflow", overflow, 1)):
        if t is not None and (tuple(t.shape) != (n,) or t.dtype != torch.int32 or t.device != dev or not t.is_contiguous()):
            raise ValueError(f"accept_drafts: {what} must be a contiguous int32 [{n}] on {dev}")
    k_new, kb, kt = _token_rows(k_new)
    v_new, vb, vt = _token_rows(v_new)
    _launch(dev.index, _lib.lib().pjx_kv_cache_accept, _ptr(k_cache), _ptr(v_cache), _ptr(k_new), kb, kt, _ptr(v_new), vb, vt, _ptr(lengths),
            _ptr(path), _ptr(counts), _ptr(table), B, N, path.shape[1], Hkv, D, Dv, cap, page, max_pages, num_pages, _DTYPES[k_new.dtype],
            _ptr(out), _ptr(overflow), _stream(dev))
    _written(k_cache, v_cache, given, overflow)
    return out
