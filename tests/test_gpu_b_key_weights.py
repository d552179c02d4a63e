"""Attention received by every key and eviction by it (``decode_weights``, ``key_weights``, ``evict``) against 64-bit references."""

import math

import pytest
import torch

from _operators_ref import HALF_STEP, attention_row, evict_reference, key_weights_reference

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def normal(seed, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def lse_of(q, k, lengths, lo=None, hi=None):
    """The call's natural log-sum-exp in 32 bits, +inf for rows without keys."""
    B, Lq, Hq, D = q.shape
    G = Hq // k.shape[2]
    s = torch.einsum("bqhd,bkhd->bhqk", q.double(), torch.nan_to_num(k.double()).repeat_interleave(G, 2)) / math.sqrt(D)
    t, j = torch.arange(Lq)[:, None], torch.arange(k.shape[1])[None]
    keep = torch.ones(B, 1, Lq, k.shape[1], dtype=torch.bool)
    if lengths is not None:
        keep &= (j < lengths[:, None, None])[:, None]
    if lo is not None:
        keep &= (j >= t + lo)
    if hi is not None:
        keep &= (j <= t + hi)
    l = torch.logsumexp(s.masked_fill(~keep, -math.inf), -1)
    return torch.where(torch.isinf(l), torch.full_like(l, math.inf), l).float()


TRACK = [  # B, Lq, Hq, Hkv, D, cap, lengths, dtype
    (1, 1, 8, 2, 128, 1500, [1500], torch.bfloat16),
    (3, 1, 8, 2, 64, 777, [777, 0, 1], torch.float16),
    (2, 4, 8, 2, 128, 640, [639, 65], torch.bfloat16),   # four tokens, sixteen rows
    (2, 1, 3, 1, 64, 130, [64, 129], torch.bfloat16),
    (2, 3, 16, 2, 64, 300, [300, 200], torch.float16),   # 24 rows: the regular kernels
    (2, 1, 4, 4, 96, 200, [190, 3], torch.bfloat16),     # a head width the streaming kernel does not take
    (2, 1, 4, 2, 64, 250, [250, 17], torch.float32),
    (130, 1, 2, 1, 64, 70, None, torch.bfloat16),
]


@pytest.mark.parametrize("B,Lq,Hq,Hkv,D,cap,lengths,dtype", TRACK)
def test_decode_weights(B, Lq, Hq, Hkv, D, cap, lengths, dtype):
    import probjax_b200 as pj

    q, k, v = normal(1, B, Lq, Hq, D, dtype=dtype), normal(2, B, cap, Hkv, D, dtype=dtype), normal(3, B, cap, Hkv, D, dtype=dtype)
    n = [cap] * B if lengths is None else lengths
    for b in range(B):
        k[b, n[b]:], v[b, n[b]:] = float("nan"), float("nan")
    old = normal(4, B, Hkv, cap).abs()
    kl = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=DEV)
    o, lse, w = pj.decode_weights(q.to(DEV), k.to(DEV), v.to(DEV), old.to(DEV), kv_lengths=kl, return_lse=True)
    pj.check_status(DEV)
    plain, plain_lse = pj.decode_forward(q.to(DEV), k.to(DEV), v.to(DEV), kv_lengths=kl, sm_scale=1 / math.sqrt(D), return_lse=True)
    if Lq * Hq // Hkv <= 16 and D in (64, 128) and dtype != torch.float32:
        assert torch.equal(o, plain) and torch.equal(lse, plain_lse)  # the decode itself is the same
    want, tol = torch.zeros(B, Hkv, cap, dtype=torch.float64), torch.zeros(B, Hkv, cap, dtype=torch.float64)
    for b in range(B):
        for h in range(Hq):
            g = h // (Hq // Hkv)
            for t in range(Lq):
                r, _, p, t_o, rel = attention_row(q[b, t, h], k[b, :n[b], g], v[b, :n[b], g], 1 / math.sqrt(D))
                want[b, g, :n[b]] += p
                tol[b, g, :n[b]] += p * rel
                u = HALF_STEP[dtype]
                bound = t_o + u * (p @ v[b, :n[b], g].double().abs() + r.abs())
                assert bool(((o[b, t, h].cpu().double() - r).abs() <= bound).all())
    total = old.double() + want
    assert bool(((w.cpu().double() - total).abs() <= tol + 2.0 ** -23 * total + 2.0 ** -22 * want).all())
    for b in range(B):
        assert torch.equal(w[b, :, n[b]:].cpu(), old[b, :, n[b]:])  # behind the valid keys nothing changes
    # in place, and from nothing
    buf = old.to(DEV)
    got = pj.decode_weights(q.to(DEV), k.to(DEV), v.to(DEV), buf, kv_lengths=kl, out=buf)
    assert got[1] is buf and torch.equal(buf, w)
    fresh = pj.decode_weights(q.to(DEV), k.to(DEV), v.to(DEV), kv_lengths=kl)[1].cpu().double()
    assert bool(((fresh - want).abs() <= tol + 2.0 ** -22 * want).all())


WINDOW = [  # B, Lq, Hq, Hkv, D, Lkv, lengths, mask, dtype
    (1, 1, 4, 1, 128, 1000, None, "none", torch.bfloat16),
    (2, 32, 8, 2, 128, 515, [515, 300], "right", torch.bfloat16),
    (2, 17, 6, 2, 64, 260, [259, 0], "none", torch.float16),
    (1, 100, 14, 2, 64, 300, None, "causal", torch.float16),    # 700 rows a KV head
    (1, 65, 4, 4, 128, 333, None, "band", torch.bfloat16),
    (1, 300, 8, 1, 64, 300, None, "causal", torch.bfloat16),    # 2400 rows
    (2, 9, 4, 2, 96, 130, [130, 77], "right", torch.bfloat16),
    (2, 21, 4, 2, 64, 200, [64, 200], "causal", torch.float32),
    (1, 3, 200, 1, 64, 140, None, "none", torch.bfloat16),      # 200 query heads on one KV head
    (1, 2, 300, 1, 64, 140, None, "none", torch.float16),
]


@pytest.mark.parametrize("B,Lq,Hq,Hkv,D,Lkv,lengths,mask,dtype", WINDOW)
def test_key_weights(B, Lq, Hq, Hkv, D, Lkv, lengths, mask, dtype):
    import probjax_b200 as pj

    q, k = normal(11, B, Lq, Hq, D, dtype=dtype), normal(12, B, Lkv, Hkv, D, dtype=dtype)
    lo, hi = {"none": (None, None), "right": (None, Lkv - Lq), "causal": (None, 0), "band": (-40, 5)}[mask]
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32)
    if n is not None:
        for b in range(B):
            k[b, lengths[b]:] = float("nan")
    lse = lse_of(q, k, n, lo, hi)
    m = {"none": pj.NoMask(), "right": pj.CausalFromBottomRightMask(Lq, Lkv), "causal": pj.CausalMask(), "band": pj.LocalWindowMask(40, 5)}[mask]
    if n is not None:
        m = pj.KVLenMask(n.to(DEV)) if mask == "none" else pj.KVLenMask(n.to(DEV)) & m
    old = normal(13, B, Hkv, Lkv).abs()
    w = pj.key_weights(q.to(DEV), k.to(DEV), lse.to(DEV), weights=old.to(DEV), mask=m)
    pj.check_status(DEV)
    want, tol = key_weights_reference(q, k, lse, n, lo, hi)
    assert bool(((w.cpu().double() - old - want).abs() <= tol + 2.0 ** -23 * (old + want)).all())
    again = pj.key_weights(q.to(DEV), k.to(DEV), lse.to(DEV), weights=old.to(DEV), mask=m)
    assert torch.equal(w, again)  # a fixed order of summation
    buf = old.to(DEV)
    pj.key_weights(q.to(DEV), k.to(DEV), lse.to(DEV), weights=buf, mask=m, out=buf)
    assert torch.equal(buf, w)
    fresh = pj.key_weights(q.to(DEV), k.to(DEV), lse.to(DEV), mask=m, implementation="b200:generic").cpu().double()
    assert bool(((fresh - want).abs() <= tol + 2.0 ** -23 * want).all())


def test_weights_of_an_attention_call_sum_to_its_rows():
    """With the forward's own lse every row's probabilities sum to one, so the weights of a KV head sum to rows x heads."""
    import probjax_b200 as pj

    B, L, Hq, Hkv, D = 2, 384, 8, 2, 128
    q, k, v = (normal(20 + i, B, L, h, D, dtype=torch.bfloat16).to(DEV) for i, h in enumerate((Hq, Hkv, Hkv)))
    _, lse = pj.mha(q, k, v, mask=pj.CausalMask(), sm_scale=1 / math.sqrt(D), return_lse=True)
    w = pj.key_weights(q, k, lse, mask=pj.CausalMask())
    total = w.double().sum(-1)
    assert float((total / (L * Hq // Hkv) - 1).abs().max()) <= 2.0 ** -14


@pytest.mark.parametrize("B,cap,Hkv,D,Dv,keep,recent,lengths,dtype", [
    (1, 300, 2, 128, 128, 100, 10, [300], torch.bfloat16),
    (4, 200, 3, 64, 64, 64, 64, [200, 64, 65, 0], torch.float16),   # only the recent ones; exactly the budget; one over; empty
    (2, 5000, 2, 64, 64, 1234, 0, [5000, 4097], torch.bfloat16),    # several CTAs a head
    (2, 40000, 1, 64, 64, 30001, 7, [40000, 35000], torch.bfloat16),
    (2, 150, 2, 20, 12, 33, 5, [150, 149], torch.float32),
    (2, 150, 2, 5, 7, 33, 5, [150, 90], torch.float16),             # rows that are no whole 16 bytes
    (3, 50, 2, 64, 128, 80, 3, [50, 10, 0], torch.bfloat16),        # a budget beyond the capacity
    (2, 90, 1, 64, 64, 1, 0, [90, 1], torch.bfloat16),
    (2, 90, 1, 64, 64, 1, 1, [90, 2], torch.bfloat16),
])
@pytest.mark.parametrize("place", ["in place", "other buffers"])
def test_evict(B, cap, Hkv, D, Dv, keep, recent, lengths, dtype, place):
    import probjax_b200 as pj

    k, v = normal(31, B, cap, Hkv, D, dtype=dtype), normal(32, B, cap, Hkv, Dv, dtype=dtype)
    w = normal(33, B, Hkv, cap).mul(2).exp()
    w[:, :, ::7] = 0.0
    w[:, :, 3::11] = 0.25
    w[..., 5::13] *= -1
    for b in range(B):
        w[b, :, lengths[b]:] = 0
    kept = evict_reference(k, v, w, lengths, keep, recent)
    n = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    kd, vd, wd = k.to(DEV), v.to(DEV), w.to(DEV)
    if place == "in place":
        out, (ko, vo, wo) = None, (kd, vd, wd)
        base = (k.clone(), v.clone(), w.clone())
    else:
        room = min(keep, cap) + 3
        ko, vo, wo = torch.full((B, room, Hkv, D), 7.0, dtype=dtype, device=DEV), torch.full((B, room, Hkv, Dv), 7.0, dtype=dtype, device=DEV), torch.full(
            (B, Hkv, room), 7.0, device=DEV)
        out, base = (ko, vo, wo), (ko.cpu(), vo.cpu(), torch.zeros(B, Hkv, room))
    new, idx = pj.evict(kd, vd, wd, n, keep, recent=recent, out=out)
    want_k, want_v, want_w = base
    want_i = torch.full((B, Hkv, keep), -1, dtype=torch.int32)
    for b in range(B):
        for h in range(Hkv):
            rows = kept[b][h]
            m = len(rows)
            want_i[b, h, :m] = torch.tensor(rows, dtype=torch.int32)
            want_k[b, :m, h], want_v[b, :m, h] = k[b, rows, h], v[b, rows, h]
            want_w[b, h, :m] = w[b, h, rows]
            if place == "in place":
                want_w[b, h, m:lengths[b]] = 0
    assert new.tolist() == [min(x, keep) for x in lengths]
    assert torch.equal(idx.cpu(), want_i)
    assert torch.equal(ko.cpu(), want_k) and torch.equal(vo.cpu(), want_v) and torch.equal(wo.cpu(), want_w)
    if place != "in place":
        assert torch.equal(kd.cpu(), k) and torch.equal(wd.cpu(), w)


def test_evict_orders_special_weights():
    """NaN ranks behind -inf, -0 ties with 0, +inf comes first; equal weights go by index."""
    import probjax_b200 as pj

    nan, inf = float("nan"), float("inf")
    row = [0.0, nan, -0.0, 1.0, -inf, inf, 0.0, 1.0, nan, -1.0, 3e-41, -3e-41]
    w = torch.tensor(row)[None, None].to(DEV)
    k = torch.arange(12.0).reshape(1, 12, 1, 1).expand(1, 12, 1, 64).contiguous().to(DEV)
    for keep, want in ((1, [5]), (3, [3, 5, 7]), (4, [3, 5, 7, 10]), (6, [0, 2, 3, 5, 7, 10]), (8, [0, 2, 3, 5, 6, 7, 10, 11]),
                       (10, [0, 2, 3, 4, 5, 6, 7, 9, 10, 11]), (11, [0, 1, 2, 3, 4, 5, 6, 7, 9, 10, 11])):
        out = tuple(torch.zeros(s, device=DEV) for s in ((1, keep, 1, 64), (1, keep, 1, 64), (1, 1, keep)))
        _, idx = pj.evict(k, k.clone(), w, [12], keep, out=out)
        assert idx[0, 0].tolist() == want
        assert out[0][0, :, 0, 0].tolist() == [float(x) for x in want]
    for same in (0.0, nan, 2.0):  # all equal: the first ones
        _, idx = pj.evict(k, k.clone(), torch.full_like(w, same), [12], 5, recent=2, out=tuple(
            torch.zeros(s, device=DEV) for s in ((1, 5, 1, 64), (1, 5, 1, 64), (1, 1, 5))))
        assert idx[0, 0].tolist() == [0, 1, 2, 10, 11]


def test_bounded_cache_loop():
    """Prompt, decode steps that track weights, eviction, further steps, captured and eager: attention over the kept keys is that of a
    cache which holds only them."""
    import probjax_b200 as pj

    B, Hq, Hkv, D, cap, L = 2, 8, 2, 64, 256, 200
    cache = pj.DecodeCache(B, cap, Hkv, D, track_weights=True)
    t = lambda s, *shape: normal(s, *shape, dtype=torch.bfloat16).to(DEV)
    q, k, v = t(50, B, L, Hq, D), t(51, B, L, Hkv, D), t(52, B, L, Hkv, D)
    cache.update(k, v)
    cache.attend(q, prefix_length=L, window=32)
    total = cache.key_weights.double().sum(-1)
    assert float((total / (32 * Hq // Hkv) - 1).abs().max()) <= 2.0 ** -7  # (the lse of a bf16 forward, P in 32 bits)
    steps = [(t(60 + i, B, 1, Hq, D), t(70 + i, B, 1, Hkv, D), t(80 + i, B, 1, Hkv, D)) for i in range(6)]
    for s in steps[:3]:
        cache.step(*s)
    before = cache.key_weights.clone()
    kept = cache.evict(64, recent=16)
    assert cache.cache_index.tolist() == [64, 64] and bool((kept[:, :, -16:] == torch.arange(187, 203, device=DEV)).all())
    at = kept.long()
    all_k = torch.cat([k] + [s[1] for s in steps[:3]], 1)
    for h in range(Hkv):
        for b in range(B):
            assert torch.equal(cache.cached_key[b, :64, h], all_k[b, at[b, h], h])
            assert torch.equal(cache.key_weights[b, h, :64], before[b, h, at[b, h]])
    assert bool((cache.key_weights[:, :, 64:] == 0).all())
    ref = pj.DecodeCache(B, cap, Hkv, D)
    ref.cached_key.copy_(cache.cached_key)
    ref.cached_value.copy_(cache.cached_value)
    ref.reset([64, 64])
    ins = [x.clone() for x in steps[3]]
    ref.update(*ins[1:])  # (caches this short attend on the regular forward; the split decode is asked for by name)
    want = pj.decode_forward(ins[0], ref.cached_key, ref.cached_value, kv_lengths=ref.cache_index, sm_scale=1 / math.sqrt(D))
    torch.cuda.synchronize()
    weights = cache.key_weights.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cache.step(*ins)
    cache.reset([64, 64])
    cache.key_weights.copy_(weights)
    graph.replay()
    torch.cuda.synchronize()
    assert cache.cache_index.tolist() == [65, 65]
    assert torch.equal(out, want)  # the decode itself does not change by tracking
    grown = (cache.key_weights - weights).double().sum(-1)
    assert float((grown / (Hq // Hkv) - 1).abs().max()) <= 2.0 ** -14
    pj.check_status(DEV)
