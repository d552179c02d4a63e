"""Autoregressive KV cache for decode steps.

Host-side mirror of the cache the reference's attention layer keeps
(probjax/nn/layers/attention.py: ``init_cache`` 727-757, decode branch 603-675):
``cached_key`` / ``cached_value`` ``[B, capacity, Hkv, D]`` and a write position.  The
reference shares one ``cache_index`` across the batch and masks with
``KeyPaddingMask(cur_index + 1)``; here every sequence has its own position (a ragged
batch), the update is one kernel launch (``pjx_kv_cache_append``) that also advances the
positions on the device, and attention over the filled prefix is the split-KV decode
kernel with ``kv_lengths = positions``.
"""

from __future__ import annotations

import ctypes
import functools
import math

import torch

from . import _lib
from .attention import _DTYPES, _IMPL, _launch, _ptr, _require_gpu, _scratch_bytes, _status_word, _stream, _wants_grad, _written, mha
from .drafts import accept_drafts, decode_tree
from .eviction import decode_weights, evict, key_weights
from .masks import CausalFromBottomRightMask, KVLenMask


class DecodeCache:
    """Keys and values of a batch of sequences, each with its own position.  ``track_weights`` also keeps, in ``key_weights``
    float32 ``[B, Hkv, capacity]``, the attention that every key has received so far, by which :meth:`evict` cuts the cache."""

    def __init__(self, batch: int, capacity: int, num_kv_heads: int, head_dim: int, v_head_dim: int | None = None,
                 dtype=torch.bfloat16, device=None, track_weights: bool = False):
        _require_gpu()
        device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        v_head_dim = head_dim if v_head_dim is None else v_head_dim
        self.batch, self.capacity = int(batch), int(capacity)
        self.cached_key = torch.zeros((batch, capacity, num_kv_heads, head_dim), dtype=dtype, device=device)
        self.cached_value = torch.zeros((batch, capacity, num_kv_heads, v_head_dim), dtype=dtype, device=device)
        # [0, B): positions; [B, 2B): scratch counters of the append kernel (zero between launches)
        self._positions = torch.zeros((2 * batch,), dtype=torch.int32, device=device)
        self._overflow = torch.zeros((1,), dtype=torch.int32, device=device)
        self.key_weights = torch.zeros((batch, num_kv_heads, capacity), dtype=torch.float32, device=device) if track_weights else None

    @property
    def cache_index(self) -> torch.Tensor:
        """``int32 [B]``: number of valid tokens per sequence (a view, updated on the device)."""
        return self._positions[: self.batch]

    def reset(self, lengths=None):
        self._positions.zero_()
        self._overflow.zero_()
        if self.key_weights is not None:
            self.key_weights.zero_()
        if lengths is not None:
            self._positions[: self.batch] = torch.as_tensor(lengths, dtype=torch.int32, device=self._positions.device)

    def overflowed(self) -> bool:
        """Whether an update ran past the capacity (synchronises)."""
        return bool(self._overflow.item())

    def update(self, key: torch.Tensor, value: torch.Tensor, advance: bool = True):
        """Append ``key [B, n, Hkv, D]`` / ``value [B, n, Hkv, Dv]`` at each sequence's position."""
        ck, cv = self.cached_key, self.cached_value
        if key.shape[0] != self.batch or key.shape[2:] != ck.shape[2:] or value.shape[2:] != cv.shape[2:] \
                or value.shape[:2] != key.shape[:2]:
            raise ValueError(
                f"Autoregressive cache shape error, expected key [B={self.batch}, n, {ck.shape[2]}, {ck.shape[3]}] and "
                f"value [B, n, {cv.shape[2]}, {cv.shape[3]}], got {tuple(key.shape)} and {tuple(value.shape)}."
            )
        if key.dtype != ck.dtype or value.dtype != cv.dtype:
            raise ValueError("key / value dtype differs from the cache dtype")
        key, value = key.contiguous(), value.contiguous()
        dev = ck.device
        with torch.cuda.device(dev):
            rc = _lib.lib().pjx_kv_cache_append(_ptr(ck), _ptr(cv), _ptr(key), _ptr(value), _ptr(self._positions),
                                                self.batch, self.capacity, key.shape[1], ck.shape[2], ck.shape[3],
                                                cv.shape[3], _DTYPES[ck.dtype], int(advance), _ptr(self._overflow),
                                                _stream(dev))
        _lib.check(rc)

    def attend(self, query: torch.Tensor, *, sm_scale: float | None = None, return_lse: bool = False,
               prefix_length: int | None = None, window: int | None = None):
        """Attention of ``query [B, n, Hq, D]`` over the filled prefix.  One query token per
        sequence is a decode step (split-KV kernel, ragged positions).  Several query tokens
        (a prefill chunk just appended) need ``prefix_length``: the common number of valid
        tokens after the append, for the bottom-right causal mask.

        With ``track_weights`` the attention that every key receives is added to ``key_weights``: of all queries, or of the last
        ``window`` ones (which costs one more pass over the keys for those queries)."""
        if sm_scale is None:
            sm_scale = 1.0 / math.sqrt(query.shape[-1])
        mask = KVLenMask(self.cache_index)
        n = query.shape[1]
        if n > 1:
            if prefix_length is None:
                raise ValueError("attend with several query tokens needs prefix_length (tokens valid after the append)")
            mask = mask & CausalFromBottomRightMask(n, int(prefix_length))
        if window is not None and (self.key_weights is None or window < 1):
            raise ValueError("window is a positive number of queries whose attention counts, with track_weights")
        if self.key_weights is None:
            return mha(query, self.cached_key, self.cached_value, mask=mask, sm_scale=sm_scale, return_lse=return_lse)
        if n == 1 and not _wants_grad(query, self.cached_key, self.cached_value):
            res = decode_weights(query, self.cached_key, self.cached_value, self.key_weights, kv_lengths=self.cache_index, sm_scale=sm_scale,
                                 return_lse=return_lse, out=self.key_weights)
            return res[:2] if return_lse else res[0]
        out, lse = mha(query, self.cached_key, self.cached_value, mask=mask, sm_scale=sm_scale, return_lse=True)
        q, part = query.detach(), lse.detach()
        if window is not None and window < n:
            q, part = q[:, n - window:], part[:, :, n - window:]
            mask = KVLenMask(self.cache_index) & CausalFromBottomRightMask(window, int(prefix_length))
        key_weights(q, self.cached_key.detach(), part, weights=self.key_weights, mask=mask, sm_scale=sm_scale, out=self.key_weights)
        return (out, lse) if return_lse else out

    def attend_tree(self, query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, parents, *, sm_scale: float | None = None,
                    return_lse: bool = False):
        """Attention of a tree of drafted tokens ``query [B, N, Hq, D]`` over the filled prefix and their ancestors among the
        drafts (:func:`decode_tree`); ``key`` / ``value`` ``[B, N, Hkv, D]`` are the drafts' own and do not enter the cache.

        Nothing is added to ``key_weights``.  For the accepted drafts that is, after :meth:`accept` and before an eviction, one call of
        :func:`key_weights` for every depth ``i`` of the path (a draft sees the keys up to its own, which is another end for every sequence
        and depth, and a call has one end a sequence): the queries and ``lse`` rows of drafts ``path[:, i]``, ``lse = +inf`` where
        ``i >= counts``, the cache's keys, ``mask=KVLenMask(lengths + i + 1)`` with the lengths before the acceptance, ``weights`` and
        ``out`` the cache's."""
        return decode_tree(query, key, value, self.cached_key, self.cached_value, parents, kv_lengths=self.cache_index, sm_scale=sm_scale,
                           return_lse=return_lse)

    def accept(self, key: torch.Tensor, value: torch.Tensor, path, counts):
        """Append the accepted drafts ``path[b, :counts[b]]`` of ``key`` / ``value`` and advance the positions on the device
        (:func:`accept_drafts`)."""
        accept_drafts(key, value, self.cached_key, self.cached_value, path, counts, kv_lengths=self.cache_index, out=self.cache_index,
                      overflow=self._overflow)

    def evict(self, keep: int, *, recent: int = 0) -> torch.Tensor:
        """Cut every sequence to ``keep`` keys per KV head, by ``key_weights`` and with the ``recent`` last ones kept
        (:func:`evict`), in place.  Returns the kept keys' former indices ``int32 [B, Hkv, keep]``.  ``cache_index`` counts the kept keys from
        then on, not the tokens seen: whoever rotates queries and keys to their positions counts tokens apart."""
        if self.key_weights is None:
            raise ValueError("evict needs a cache with track_weights=True")
        return evict(self.cached_key, self.cached_value, self.key_weights, self.cache_index, keep, recent=recent,
                     lengths_out=self.cache_index)[1]

    def step(self, query, key, value, *, sm_scale: float | None = None):
        """One decode step: append the token's key / value, then attend over the prefix."""
        self.update(key, value)
        return self.attend(query, sm_scale=sm_scale)


def rope_interleaved(x: torch.Tensor, positions=None, *, base: float = 10_000.0, rotary_dim: int | None = None,
                     offset: float = 0.0, out: torch.Tensor | None = None) -> torch.Tensor:
    """Interleaved rotary embedding of ``x [..., T, H, D]`` on the device (``pjx_rope_interleaved``):
    the reference's rotary layer (layers/encoding.py:171-211) with its ``rotary_dim`` / ``offset``
    options; ``positions`` is ``[T]`` or ``None`` (= ``arange(T) + offset``)."""
    _require_gpu()
    if not x.is_cuda or x.dim() < 3:
        raise ValueError("rope_interleaved takes a CUDA tensor [..., T, H, D]")
    x = x.contiguous()
    T, H, D = x.shape[-3:]
    outer = x.numel() // max(T * H * D, 1)
    rotary_dim = D if rotary_dim is None else int(rotary_dim)
    y = torch.empty_like(x) if out is None else out
    pos = None if positions is None else torch.as_tensor(positions).to(device=x.device, dtype=torch.float32).contiguous()
    if pos is not None and pos.numel() != T:
        raise ValueError(f"positions must have {T} entries, got {pos.numel()}")
    with torch.cuda.device(x.device):
        rc = _lib.lib().pjx_rope_interleaved(_ptr(x), _ptr(y), _ptr(pos), float(offset), outer, T, H, D, rotary_dim,
                                             float(base), _DTYPES[x.dtype], _stream(x.device))
    _lib.check(rc)
    return y


_POSITION_TYPES = {torch.float32: _lib.POS_F32, torch.int32: _lib.POS_I32, torch.int64: _lib.POS_I64}


def _rope_axes_call(x, positions, sections, base, shared, interleaved, inverse, out=None):
    """One ``pjx_rope_axes`` call: ``x [B, T, H, D]`` with any sequence and token stride, ``positions [B|1, T, axes]`` dense."""
    B, T, H, D = x.shape
    if (x.stride(3) != 1 and D > 1) or (x.stride(2) != D and H > 1):
        x = x.contiguous()
    y = torch.empty((B, T, H, D), dtype=x.dtype, device=x.device) if out is None else out
    _launch(x.get_device(), _lib.lib().pjx_rope_axes, _ptr(x), x.stride(0) if B > 1 else 0, x.stride(1) if T > 1 else 0, _ptr(y), _ptr(positions),
            _POSITION_TYPES[positions.dtype], 0 if positions.shape[0] == 1 else positions.stride(0), len(sections), _section_array(sections), B, T,
            H, D, int(shared), int(interleaved), int(inverse), float(base), _DTYPES[x.dtype], _stream(x.device))
    return y


@functools.lru_cache(maxsize=64)
def _section_array(sections):
    return (ctypes.c_int32 * len(sections))(*sections)


class _RopeAxesFunction(torch.autograd.Function):
    """A rotation.  Its gradient is the rotation by the opposite angles, its tangent the same rotation."""

    @staticmethod
    def forward(ctx, x, positions, args, inverse):
        # (an input that takes no gradient: kept with its version, which costs less per call than the saved-tensor machinery; a tensor
        # of inference mode has no version and is copied)
        ctx.positions = positions.clone() if positions.is_inference() else positions
        ctx.version, ctx.args, ctx.inverse = ctx.positions._version if not ctx.positions.is_inference() else None, args, inverse
        return _rope_axes_call(x, positions, *args, inverse)

    @staticmethod
    def backward(ctx, dy):
        if ctx.version is not None and ctx.positions._version != ctx.version:
            raise RuntimeError("rope_axes: positions were changed in place after the call whose gradient is wanted; pass a copy")
        if torch.is_grad_enabled():  # a gradient of the gradient is wanted
            return _RopeAxesFunction.apply(dy, ctx.positions, ctx.args, not ctx.inverse), None, None, None
        return _rope_axes_call(dy, ctx.positions, *ctx.args, not ctx.inverse), None, None, None

    @staticmethod
    def jvp(ctx, tx, *_):
        return _rope_axes_call(tx, ctx.positions, *ctx.args, ctx.inverse)


def rope_axes(x: torch.Tensor, positions, sections, *, base: float = 10_000.0, shared: bool = False, interleaved: bool = True,
              out: torch.Tensor | None = None) -> torch.Tensor:
    """Rotary embedding with several axes and positions of every sequence's own (``pjx_rope_axes``): ``x [..., T, H, D]``,
    ``positions [T, axes]`` or ``[..., T, axes]`` (float32, int32 or int64; other integers become int64, other floats float32; leading
    dimensions as ``x``), ``sections`` the
    elements of a head vector that each axis rotates (even; they follow one another, the rest is copied).  Pair ``i`` of an axis turns
    by ``position * base**(-2 i / section)``; with ``shared`` the frequencies run through all axes,
    ``base**(-2 p / sum(sections))`` for pair ``p``.  ``interleaved``: pairs are neighbours, otherwise the two halves of the rotated
    part.  A slice of a fused projection is read in place.  Differentiable with respect to ``x`` (``positions`` must not change in place until the
    gradient has been taken: the backward pass refuses then, except after :meth:`DecodeCache.update`, whose writes autograd does not see:
    pass a copy of ``cache_index``); ``out`` (dense, may be a dense ``x``) takes the result where no gradient is
    wanted.  One axis is :func:`rope_interleaved` with positions per sequence."""
    _require_gpu()
    if not isinstance(x, torch.Tensor) or not x.is_cuda or x.dim() < 3 or x.dtype not in _DTYPES:
        raise ValueError("rope_axes takes a CUDA tensor [..., T, H, D] of dtype float32, bfloat16 or float16")
    sections = tuple(int(s) for s in sections)
    T, H, D = x.shape[-3:]
    lead = tuple(x.shape[:-3])
    pos = positions if isinstance(positions, torch.Tensor) else torch.as_tensor(positions)
    if pos.dtype not in _POSITION_TYPES:
        if pos.is_complex() or pos.dtype == torch.bool:
            raise ValueError(f"positions must be numbers, got {pos.dtype}")
        pos = pos.to(torch.float32 if pos.is_floating_point() else torch.int64)
    if pos.device != x.device:
        pos = pos.to(x.device)
    if pos.shape == (T, len(sections)):
        pos = pos[None].contiguous()
    elif pos.shape == lead + (T, len(sections)):
        pos = (pos if pos.dim() == 3 else pos.reshape(math.prod(lead), T, len(sections))).contiguous()
    else:
        raise ValueError(f"positions must be [T={T}, axes={len(sections)}] or [..., T, axes] with the leading dimensions {list(lead)}, "
                         f"got {tuple(pos.shape)}")
    if torch.is_grad_enabled() and pos.requires_grad:
        raise NotImplementedError("rope_axes has no gradient with respect to positions: detach them")
    x4 = x[None] if x.dim() == 3 else x if x.dim() == 4 else x.reshape((math.prod(lead),) + tuple(x.shape[-3:]))
    if _wants_grad(x):
        if out is not None:
            raise ValueError("rope_axes: out cannot be given where a gradient is wanted")
        y = _RopeAxesFunction.apply(x4, pos, (sections, base, shared, interleaved), False)
        return y if x.dim() == 4 else y.reshape(x.shape)
    if out is not None:
        if tuple(out.shape) != tuple(x.shape) or out.dtype != x.dtype or out.device != x.device or not out.is_contiguous():
            raise ValueError("rope_axes: out must be a dense tensor like x")
        n = out.numel() * out.element_size()
        same = out.data_ptr() == x.data_ptr() and x.is_contiguous()
        if not same and x.numel() and out.untyped_storage().data_ptr() == x.untyped_storage().data_ptr():
            first, last = x.data_ptr(), x.data_ptr() + (sum((d - 1) * s for d, s in zip(x.shape, x.stride())) + 1) * x.element_size()
            if first < out.data_ptr() + n and out.data_ptr() < last:
                raise ValueError("rope_axes: out overlaps x without being it")
    y = _rope_axes_call(x4, pos, sections, base, shared, interleaved, False, out)
    if out is not None:
        _written(out)
    return y if x.dim() == 4 else y.reshape(x.shape)


def _check_layers(x, *weights) -> None:
    ok, k, dtype = x.is_cuda, x.shape[-1], x.dtype
    for w in weights:
        ok = ok and w.dim() == 2 and w.shape[-1] == k and w.dtype == dtype
    if not ok:
        raise ValueError("linear takes CUDA tensors x [..., K] and weight [N, K] of one dtype")


def _on(device, w):
    return w if w.device == device else w.to(device)


def linear(x: torch.Tensor, weight: torch.Tensor, *, implementation: str | None = None) -> torch.Tensor:
    """``x [..., K] @ weight[N, K]^T`` on the device (``pjx_linear``): the bias-free query / key /
    value / output projections around the attention call (layers/attention.py:591-594).  A fused
    QKV projection is one call with the three weights concatenated along ``N``."""
    _require_gpu()
    _check_layers(x, weight)
    if implementation not in _IMPL:
        raise ValueError(f"implementation must be None or one of {sorted(k for k in _IMPL if k)}")
    x2 = x.contiguous().view(-1, x.shape[-1])
    w = weight.to(x.device).contiguous()
    y = torch.empty((x2.shape[0], w.shape[0]), dtype=x.dtype, device=x.device)
    with torch.cuda.device(x.device):
        rc = _lib.lib().pjx_linear(_ptr(x2), _ptr(w), _ptr(y), x2.shape[0], w.shape[0], w.shape[1], _DTYPES[x.dtype],
                                   _IMPL[implementation], _ptr(_status_word(x.device)), _stream(x.device))
    _lib.check(rc)
    return y.view(*x.shape[:-1], w.shape[0])


def _linear_grads(x, weights, dys, want_dx: bool, want_dw):
    """``(dx, [dw, ..])`` of one or two layers ``y_p = x . w_p^T`` sharing ``x [M, K]``: one launch for ``dx`` (summed
    over the layers in fp32) and one for the weight gradients, on the operands as they are stored.  Operands the
    tensor-core kernel does not take go through :func:`linear` and transposed copies."""
    M, K = x.shape
    ns = [w.shape[0] for w in weights]
    ptrs = [x, *weights, *dys]
    if (x.dtype != torch.float32 and M >= 64 and K >= 64 and K % 8 == 0 and all(n >= 64 and n % 8 == 0 for n in ns)
            and all(t.data_ptr() % 16 == 0 for t in ptrs)):
        dx = torch.empty_like(x) if want_dx else None
        dws = [torch.empty_like(w) if need else None for w, need in zip(weights, want_dw)]
        w1, dy1, dw1 = (weights[1], dys[1], dws[1]) if len(ns) > 1 else (None, None, None)
        with torch.cuda.device(x.device):
            rc = _lib.lib().pjx_linear_pair_bwd(_ptr(x), _ptr(weights[0]), _ptr(w1), _ptr(dys[0]), _ptr(dy1), _ptr(dx),
                                                _ptr(dws[0]), _ptr(dw1), M, ns[0], ns[1] if len(ns) > 1 else 0, K,
                                                _DTYPES[x.dtype], _ptr(_status_word(x.device)), _stream(x.device))
        _lib.check(rc)
        return dx, dws
    dx = None
    if want_dx:
        parts = [linear(dy, w.t().contiguous()) for dy, w in zip(dys, weights)]      # [M, n] . [K, n]^T
        dx = parts[0] if len(parts) == 1 else parts[0] + parts[1]
    dws = [linear(dy.t().contiguous(), x.t().contiguous()) if need else None for dy, need in zip(dys, want_dw)]
    return dx, dws


class _LinearFunction(torch.autograd.Function):
    """``linear`` with its gradients: ``dx = dy . w`` and ``dw = dy^T . x``."""

    @staticmethod
    def forward(ctx, x, weight):
        ctx.save_for_backward(x, weight)
        return linear(x, weight)

    @staticmethod
    def backward(ctx, dy):
        x, weight = ctx.saved_tensors
        dy2 = dy.reshape(-1, dy.shape[-1]).to(x.dtype).contiguous()
        x2 = x.reshape(-1, x.shape[-1]).contiguous()
        dx, (dw,) = _linear_grads(x2, [weight.contiguous()], [dy2], ctx.needs_input_grad[0], [ctx.needs_input_grad[1]])
        return None if dx is None else dx.view(x.shape), dw


def linear_autograd(x: torch.Tensor, weight: torch.Tensor) -> torch.Tensor:
    """:func:`linear` that records itself for reverse-mode differentiation."""
    _require_gpu()
    _check_layers(x, weight)
    return _LinearFunction.apply(x, _on(x.device, weight))  # (a gradient goes back to the weight's device)


class _LinearPairFunction(torch.autograd.Function):
    """Two layers that share their input (keys and values of latent attention): one launch forward, and backward one
    for the gradient of the input and one for both weight gradients."""

    @staticmethod
    def forward(ctx, x, w0, w1):
        ctx.save_for_backward(x, w0, w1)
        x2, w0, w1 = x.contiguous().view(-1, x.shape[-1]), w0.contiguous(), w1.contiguous()
        y0, y1 = (torch.empty((x2.shape[0], w.shape[0]), dtype=x.dtype, device=x.device) for w in (w0, w1))
        with torch.cuda.device(x.device):
            rc = _lib.lib().pjx_linear_pair(_ptr(x2), _ptr(w0), _ptr(w1), _ptr(y0), _ptr(y1), x2.shape[0], w0.shape[0],
                                            w1.shape[0], x2.shape[1], _DTYPES[x.dtype], _ptr(_status_word(x.device)),
                                            _stream(x.device))
        _lib.check(rc)
        return y0.view(*x.shape[:-1], w0.shape[0]), y1.view(*x.shape[:-1], w1.shape[0])

    @staticmethod
    def backward(ctx, dy0, dy1):
        x, w0, w1 = ctx.saved_tensors
        dys = [dy.reshape(-1, dy.shape[-1]).to(x.dtype).contiguous() for dy in (dy0, dy1)]
        x2 = x.reshape(-1, x.shape[-1]).contiguous()
        dx, (dw0, dw1) = _linear_grads(x2, [w0.contiguous(), w1.contiguous()], dys, ctx.needs_input_grad[0],
                                       ctx.needs_input_grad[1:3])
        return None if dx is None else dx.view(x.shape), dw0, dw1


def linear_pair_autograd(x: torch.Tensor, w0: torch.Tensor, w1: torch.Tensor):
    """``(linear(x, w0), linear(x, w1))``, recorded for reverse-mode differentiation."""
    _require_gpu()
    _check_layers(x, w0, w1)
    return _LinearPairFunction.apply(x, _on(x.device, w0), _on(x.device, w1))


def decode_paged(q: torch.Tensor, k_pool: torch.Tensor, v_pool: torch.Tensor, block_table: torch.Tensor, kv_lengths,
                 *, sm_scale: float | None = None, split_len: int = 0, return_lse: bool = False):
    """Split-KV decode over a paged cache (``pjx_attn_decode_paged``): ``k_pool`` / ``v_pool``
    ``[num_pages, page_size, Hkv, D]``, ``block_table int32 [B, max_pages]`` (page of every logical
    block of a sequence), ``kv_lengths [B]``.  ``page_size`` must be a multiple of 64."""
    _require_gpu()
    if not q.is_cuda:
        raise ValueError("decode_paged takes CUDA tensors")
    dev = q.device
    if q.dim() != 4 or k_pool.dim() != 4 or v_pool.dim() != 4:
        raise ValueError("decode_paged: q must be [B, Lq, Hq, D] and the pools [num_pages, page_size, Hkv, D]")
    if k_pool.dtype != q.dtype or v_pool.dtype != q.dtype or k_pool.device != dev or v_pool.device != dev:
        raise ValueError("decode_paged: q and the page pools must share a dtype and a device")
    q, k_pool, v_pool = q.contiguous(), k_pool.contiguous(), v_pool.contiguous()
    B, Lq, Hq, D = q.shape
    page_size, Hkv, Dv = k_pool.shape[1], k_pool.shape[2], v_pool.shape[3]
    if k_pool.shape[3] != D or tuple(v_pool.shape[:3]) != tuple(k_pool.shape[:3]):
        raise ValueError(f"decode_paged: pools must be [P, page, Hkv, D={D}] / [P, page, Hkv, Dv], got "
                         f"{tuple(k_pool.shape)} and {tuple(v_pool.shape)}")
    if Hq % Hkv != 0:
        raise ValueError(f"query heads ({Hq}) must be a multiple of key/value heads ({Hkv})")
    bt = torch.as_tensor(block_table).to(device=dev, dtype=torch.int32).contiguous()
    if bt.dim() != 2 or bt.shape[0] != B:
        raise ValueError(f"block_table must be [B={B}, max_pages], got {tuple(bt.shape)}")
    max_pages = bt.shape[1]
    if sm_scale is None:
        sm_scale = 1.0 / math.sqrt(D)
    kvl = torch.as_tensor(kv_lengths).to(device=dev, dtype=torch.int32).contiguous()
    if kvl.numel() != B:
        raise ValueError(f"decode_paged: kv_lengths must hold B={B} entries, got {kvl.numel()}")
    L = _lib.lib()
    o = torch.empty((B, Lq, Hq, Dv), dtype=q.dtype, device=dev)
    lse = torch.empty((B, Hq, Lq), dtype=torch.float32, device=dev) if return_lse else None
    need = L.pjx_attn_decode_workspace_bytes(B, Lq, Hq, Hkv, Dv, max_pages * page_size, int(split_len))
    ws = _scratch_bytes(dev, "decode", need)
    with torch.cuda.device(dev):
        rc = L.pjx_attn_decode_paged(_ptr(q), _ptr(k_pool), _ptr(v_pool), _ptr(bt), _ptr(kvl), _ptr(o), _ptr(lse), B, Lq, Hq,
                                     Hkv, D, Dv, page_size, max_pages, _DTYPES[q.dtype], float(sm_scale), int(split_len),
                                     _ptr(ws), ws.numel(), _stream(dev))
    _lib.check(rc)
    return (o, lse) if return_lse else o
