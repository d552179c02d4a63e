"""Corners of the decode loop's calls (drafted trees, key weights, eviction)."""

import math
import threading

import pytest
import torch

from _operators_ref import HALF_STEP, attention_row, evict_reference, key_weights_reference, tree_reference

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def normal(seed, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def natural_lse(q, k, hi=None, scale=None):
    """Log-sum-exp in 64 bits of every query over all keys, or over those up to its own plus ``hi``, rounded to 32."""
    G = q.shape[2] // k.shape[2]
    s = torch.einsum("bqhd,bkhd->bhqk", q.double(), k.double().repeat_interleave(G, 2)) * (1 / math.sqrt(q.shape[3]) if scale is None else scale)
    if hi is not None:
        s = s.masked_fill(torch.arange(k.shape[1])[None] > torch.arange(q.shape[1])[:, None] + hi, -math.inf)
    return torch.logsumexp(s, -1).float()


@pytest.mark.parametrize("impl", [None, "b200:generic"])
@pytest.mark.parametrize("Lq,Hq,Hkv,D,Lkv,causal,dtype", [
    (9, 8, 2, 128, 400, False, torch.bfloat16),
    (100, 4, 2, 64, 260, False, torch.float16),   # 200 rows a KV head: several chunks that stay
    (300, 8, 1, 64, 300, True, torch.bfloat16),   # 2400 rows: chunks that stream past the keys
    (70, 4, 4, 128, 70, True, torch.float16),
])
def test_rows_without_keys_add_nothing_whatever_they_hold(Lq, Hq, Hkv, D, Lkv, causal, dtype, impl):
    """Rows with lse = +inf hold NaN or infinite queries, and keys that only such rows see hold NaN: nothing of it reaches a weight."""
    import probjax_b200 as pj

    B = 2
    q, k = normal(1, B, Lq, Hq, D, dtype=dtype), normal(2, B, Lkv, Hkv, D, dtype=dtype)
    lse = natural_lse(q, k, 0 if causal else None)
    dead = torch.rand(B, Hq, Lq, generator=torch.Generator().manual_seed(3)) < 0.25
    dead[:, :, 0] = True      # a whole token,
    dead[:, :, -3:] = True    # the last ones,
    dead[1] = True            # and a whole sequence
    lse[dead] = math.inf
    at = dead.transpose(1, 2)
    clean = torch.where(at[..., None], torch.zeros_like(q), q)
    bad = torch.where(torch.arange(Lq)[None, :, None] % 3 == 0, math.inf, math.nan).expand(B, Lq, Hq)
    q = torch.where(at[..., None], bad[..., None].to(dtype), q)
    k[1, 5], k[1, 6, :, 0] = math.nan, math.inf
    if causal:
        k[0, Lq - 3:] = math.nan
    old = normal(4, B, Hkv, Lkv).abs()
    w = pj.key_weights(q.to(DEV), k.to(DEV), lse.to(DEV), weights=old.to(DEV), mask=pj.CausalMask() if causal else pj.NoMask(), implementation=impl).cpu()
    pj.check_status(DEV)
    want, tol = key_weights_reference(clean, k, lse, None, None, 0 if causal else None)
    assert bool(((w.double() - old - want).abs() <= tol + 2.0 ** -23 * (old + want)).all())
    assert torch.equal(w[1], old[1])
    if causal:
        assert torch.equal(w[0, :, Lq - 3:], old[0, :, Lq - 3:])


def test_absent_drafts_do_not_reach_the_key_weights():
    """``decode_tree`` gives absent drafts lse = +inf and lets their queries hold anything: its lse goes into ``key_weights`` as it is."""
    import probjax_b200 as pj

    B, N, Hq, Hkv, D, cap = 2, 6, 8, 2, 128, 384
    q, kn, vn = (normal(10 + i, B, N, h, D, dtype=torch.bfloat16) for i, h in enumerate((Hq, Hkv, Hkv)))
    k, v = normal(13, B, cap, Hkv, D, dtype=torch.bfloat16), normal(14, B, cap, Hkv, D, dtype=torch.bfloat16)
    parents, lengths = torch.tensor([[-1, 0, -9, 1, 2, 0], [-9, -1, 0, 1, 3, -9]], dtype=torch.int32), torch.tensor([300, 77], dtype=torch.int32)
    live = torch.tensor([[1, 1, 0, 1, 0, 1], [0, 1, 0, 1, 1, 0]], dtype=torch.bool)
    q[~live] = math.nan
    _, lse = pj.decode_tree(*(x.to(DEV) for x in (q, kn, vn, k, v, parents)), kv_lengths=lengths.to(DEV), return_lse=True)
    w = pj.key_weights(q.to(DEV), k.to(DEV), lse, mask=pj.KVLenMask(lengths.to(DEV))).cpu()
    pj.check_status(DEV)
    clean = torch.where(live[..., None, None], q, torch.zeros_like(q))
    want, tol = key_weights_reference(clean, k, lse.cpu(), lengths)
    assert bool(((w.double() - want).abs() <= tol + 2.0 ** -23 * want).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("Lq", [2, 700])  # (chunks that stay, chunks that stream)
def test_scores_and_log_sum_exps_of_many_millions(Lq, dtype):
    """q.k up to 2^29 with a scale of 2^-13, so that lse / scale passes what three 16-bit numbers carry in fp16.  All sums are exact in 32
    bits (2^29 plus multiples of 2^6), so the exponent scale q.k - lse is off by the roundings at |s| = 65536: the constant's, the lse's, the
    product's, each 2^-24 relative, and three 16-bit parts' 2^-24: below 2^-22 (|s| + |lse|)."""
    import probjax_b200 as pj

    B, Hq, Hkv, D, Lkv = 1, 4, 2, 64, 200
    q, k = torch.zeros(B, Lq, Hq, D), torch.zeros(B, Lkv, Hkv, D)
    q[..., 0], q[..., 1] = 2.0 ** 15, 64.0
    k[..., 0] = 2.0 ** 14
    k[..., 1] = torch.randint(0, 256, (B, Lkv, Hkv), generator=torch.Generator().manual_seed(5)).float()
    q[:, 0, 1] *= -1  # a row that is not among them
    q[:, 0, 0] = 0.0
    q, k, scale = q.to(dtype), k.to(dtype), 2.0 ** -13
    lse = natural_lse(q, k, scale=scale)
    assert float(lse.max()) / scale > 2.0 ** 28
    old = normal(6, B, Hkv, Lkv).abs()
    w = pj.key_weights(q.to(DEV), k.to(DEV), lse.to(DEV), weights=old.to(DEV), sm_scale=scale).cpu().double()
    pj.check_status(DEV)
    want, _ = key_weights_reference(q, k, lse, scale=scale)
    rel = math.expm1(2.0 ** -22 * 2 * (2.0 ** 16 + 8)) + Hq // Hkv * Lq * 2.0 ** -23 + 2.0 ** -20
    assert bool(((w - old - want).abs() <= rel * want + 2.0 ** -23 * (old + want)).all())


@pytest.mark.parametrize("Hkv,G,Lq,D", [(75, 2, 3, 64), (148, 1, 1, 64), (149, 1, 5, 128), (200, 2, 70, 64), (300, 1, 130, 64)])
def test_key_weights_of_many_heads(Hkv, G, Lq, D):
    """More KV heads than half of the SMs, as many, and more: rows that stay in shared memory (one to three chunks)."""
    import probjax_b200 as pj

    B, Lkv, Hq = 2, 200, Hkv * G
    q, k = normal(20, B, Lq, Hq, D, dtype=torch.bfloat16), normal(21, B, Lkv, Hkv, D, dtype=torch.bfloat16)
    n = torch.tensor([200, 131], dtype=torch.int32)
    k[1, 131:] = math.nan
    lse = torch.stack([natural_lse(q[b:b + 1], k[b:b + 1, :int(n[b])])[0] for b in range(B)])
    old = normal(22, B, Hkv, Lkv).abs()
    w = pj.key_weights(q.to(DEV), k.to(DEV), lse.to(DEV), weights=old.to(DEV), mask=pj.KVLenMask(n.to(DEV))).cpu()
    pj.check_status(DEV)
    want, tol = key_weights_reference(q, k, lse, n)
    assert bool(((w.double() - old - want).abs() <= tol + 2.0 ** -23 * (old + want)).all())
    assert torch.equal(w[1, :, 131:], old[1, :, 131:])


def test_decode_weights_of_many_heads_and_rows():
    """Rows above what the streaming kernel takes: the forward kernels, then the key weights, over 150 KV heads."""
    import probjax_b200 as pj

    B, Lq, Hkv, D, cap = 1, 20, 150, 64, 90
    q, k, v = (normal(23 + i, B, n, Hkv, D, dtype=torch.float16).to(DEV) for i, n in enumerate((Lq, cap, cap)))
    _, lse, w = pj.decode_weights(q, k, v, return_lse=True)
    pj.check_status(DEV)
    want, tol = key_weights_reference(q.cpu(), k.cpu(), lse.cpu())
    assert bool(((w.cpu().double() - want).abs() <= tol + 2.0 ** -23 * want).all())


def test_two_host_threads_on_one_stream():
    """Two threads evict, decode and verify on the default stream at once, with sizes of their own: each gets what it gets alone (a call of two
    launches hands over through memory that no other thread's call writes)."""
    import probjax_b200 as pj

    def job(seed, B, cap, keep, Hkv, N):
        D, Hq = 64, 4 * Hkv
        t = lambda i, *s: normal(seed + i, *s, dtype=torch.bfloat16).to(DEV)
        k, v, w = t(0, B, cap, Hkv, D), t(1, B, cap, Hkv, D), normal(seed + 2, B, Hkv, cap).abs().to(DEV)
        n = torch.tensor([cap - 13 * b for b in range(B)], dtype=torch.int32, device=DEV)
        q, kn, vn = t(3, B, N, Hq, D), t(4, B, N, Hkv, D), t(5, B, N, Hkv, D)
        parents = torch.arange(N, dtype=torch.int32, device=DEV) - 1
        out = tuple(torch.empty(s, dtype=x, device=DEV) for s, x in (((B, keep, Hkv, D), k.dtype), ((B, keep, Hkv, D), k.dtype), ((B, Hkv, keep), w.dtype)))

        def once():
            lengths, kept = pj.evict(k, v, w, n, keep, recent=3, out=out)
            o = pj.decode_tree(q, kn, vn, k, v, parents, kv_lengths=n)
            s = pj.decode_weights(q[:, :1], k, v, kv_lengths=n)
            d = pj.decode_forward(q[:, :1], k, v, kv_lengths=n, sm_scale=0.125)
            return [x.clone() for x in (lengths, kept, *out, o, *s, d)]
        return once

    jobs = [job(100, 2, 1500, 700, 2, 5), job(200, 3, 900, 64, 4, 9)]
    alone = [f() for f in jobs]
    torch.cuda.synchronize()
    wrong, start = [], threading.Barrier(2)

    def loop(f, want):
        try:
            start.wait(timeout=60)
            got = [f() for _ in range(150)]
            torch.cuda.synchronize()
            wrong.extend(i for g in got for i, (a, b) in enumerate(zip(g, want)) if not torch.equal(a, b))
        except Exception as e:
            wrong.append(e)

    threads = [threading.Thread(target=loop, args=a) for a in zip(jobs, alone)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong[:5]
    pj.check_status(DEV)


def test_calls_without_a_gradient_refuse_inputs_that_ask_for_one():
    import probjax_b200 as pj

    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device=DEV)
    q, kn, k = z(1, 3, 4, 64), z(1, 3, 2, 64), z(1, 8, 2, 64)
    par, lse = torch.tensor([-1, 0, 1], dtype=torch.int32), torch.zeros(1, 4, 3, device=DEV)
    calls = {
        "tree": (lambda a, b, c, d, e: pj.decode_tree(a, b, c, d, e, par, kv_lengths=[4]), (q, kn, kn, k, k)),
        "decode": (lambda a, b, c: pj.decode_weights(a[:, :1], b, c), (q, k, k)),
        "weights": (lambda a, b, c: pj.key_weights(a, b, c), (q, k, lse)),
        "attend_tree": (lambda a, b, c: pj.DecodeCache(1, 8, 2, 64).attend_tree(a, b, c, par), (q, kn, kn)),
    }
    for name, (f, args) in calls.items():
        f(*args)
        for i in range(len(args)):
            wanting = [x.clone().requires_grad_(j == i) for j, x in enumerate(args)]
            with pytest.raises(NotImplementedError, match="gradient"):
                f(*wanting)
            with torch.no_grad():
                f(*wanting)


def test_a_tracked_cache_still_differentiates():
    """``attend`` with tracked weights: gradients of the queries and of a cache that asks for them, weights as without."""
    import probjax_b200 as pj

    t = lambda i, *s: normal(60 + i, *s, dtype=torch.bfloat16).to(DEV)
    q, k, v, dy = t(0, 1, 5, 4, 64), t(1, 1, 40, 2, 64), t(2, 1, 40, 2, 64), t(3, 1, 5, 4, 64)
    weights = []
    for wants in (False, True):
        cache = pj.DecodeCache(1, 64, 2, 64, track_weights=True)
        cache.update(k, v)
        x = q.clone().requires_grad_(wants)
        cache.cached_key.requires_grad_(wants)
        o = cache.attend(x, prefix_length=40)
        if wants:
            dx, dk = torch.autograd.grad(o, (x, cache.cached_key), dy)
            assert bool(dx.any()) and bool(dk[:, :40].any()) and not bool(dk[:, 40:].any())
        weights.append(cache.key_weights)
    assert torch.equal(*weights)


@pytest.mark.parametrize("impl,dtype", [(None, torch.bfloat16), ("b200:generic", torch.bfloat16), (None, torch.float32)])
@pytest.mark.parametrize("N", [5, 70])  # (one row tile, two)
def test_a_key_that_is_not_a_number_shows_in_the_rows_that_see_it(N, impl, dtype):
    """NaN in a cached key, in a draft's key and in a query: the rows that see it are NaN in output and lse, the others are as without it."""
    import probjax_b200 as pj

    B, Hq, Hkv, D, cap = 2, 4, 2, 64, 1400
    q, kn, vn = (normal(30 + i, B, N, h, D, dtype=dtype) for i, h in enumerate((Hq, Hkv, Hkv)))
    k, v = normal(33, B, cap, Hkv, D, dtype=dtype), normal(34, B, cap, Hkv, D, dtype=dtype)
    parents, lengths = torch.tensor([[-1, 0, 0, 1, 2] + [3] * (N - 5)] * B, dtype=torch.int32), torch.tensor([1300, 900], dtype=torch.int32)
    want, want_l, tol, tol_l = tree_reference(q, kn, vn, k, v, parents, lengths)
    k[0, 700, 1] = math.nan    # sequence 0, KV head 1: every row of its heads
    kn[1, 2, 0] = math.nan     # sequence 1, KV head 0: drafts 2 and 4
    q[0, 3, 0] = math.nan      # sequence 0, query head 0, draft 3
    o, lse = pj.decode_tree(*(x.to(DEV) for x in (q, kn, vn, k, v, parents)), kv_lengths=lengths.to(DEV), return_lse=True, implementation=impl)
    pj.check_status(DEV)
    nan = torch.zeros(B, N, Hq, dtype=torch.bool)
    nan[0, :, 2:] = True
    nan[1, [2, 4], :2] = True
    nan[0, 3, 0] = True
    o, lse = o.cpu().double(), lse.cpu().double()
    assert bool(torch.isnan(o[nan]).all()) and bool(torch.isnan(lse.transpose(1, 2)[nan]).all())
    assert bool(((o - want).abs() <= tol)[~nan].all())
    assert bool(((lse - want_l).abs() <= tol_l).transpose(1, 2)[~nan].all())


def test_keys_and_values_that_are_one_tensor():
    """A cache whose values are its keys: the rows move once, in place and into a shared result; accepted rows are written once."""
    import probjax_b200 as pj

    B, cap, Hkv, D, keep, lengths = 2, 700, 2, 64, 200, [700, 431]
    k, w = normal(40, B, cap, Hkv, D, dtype=torch.bfloat16), normal(41, B, Hkv, cap).abs()
    kept = evict_reference(k, k, w, lengths, keep, 9)
    want = torch.stack([torch.stack([k[b, kept[b][h], h] for h in range(Hkv)], 1) for b in range(B)])
    kd, wd, n = k.to(DEV), w.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV)
    ko, wo = torch.zeros(B, keep, Hkv, D, dtype=torch.bfloat16, device=DEV), torch.zeros(B, Hkv, keep, device=DEV)
    _, idx = pj.evict(kd, kd, wd, n, keep, recent=9, out=(ko, ko, wo))
    assert torch.equal(idx.cpu(), torch.tensor(kept, dtype=torch.int32)) and torch.equal(ko.cpu(), want)
    pj.evict(kd, kd, wd, n, keep, recent=9)
    assert torch.equal(kd[:, :keep].cpu(), want) and torch.equal(wd[:, :, :keep], wo)
    kn = normal(42, B, 5, Hkv, D, dtype=torch.bfloat16).to(DEV)
    before = kd.clone()
    pj.accept_drafts(kn, kn, kd, kd, [[0, 3], [1, 2]], [2, 1], kv_lengths=[200, 200])
    before[0, 200], before[0, 201], before[1, 200] = kn[0, 0], kn[0, 3], kn[1, 1]
    assert torch.equal(kd, before)
    with pytest.raises(ValueError, match="share"):
        pj.accept_drafts(kn, kn.clone(), kd, kd, [[0, 3], [1, 2]], [2, 1], kv_lengths=[200, 200])
    both = torch.zeros(B * cap * Hkv * D + 64, dtype=torch.bfloat16, device=DEV)
    a, c = both[:-64].view(k.shape), both[64:].view(k.shape)
    with pytest.raises(ValueError, match="share"):
        pj.evict(a, c, wd, n, keep)
    with pytest.raises(ValueError, match="share"):
        pj.evict(kd, kd.clone(), wd, n, keep, out=(ko, ko, wo))


def test_a_status_word_first_needed_in_a_capture(monkeypatch):
    """The word that a captured call reports to is the one that ``check_status`` reads, also where the capture is the process's first call."""
    import probjax_b200 as pj
    from probjax_b200 import _lib
    from probjax_b200 import attention as A

    t = lambda i, *s: normal(50 + i, *s, dtype=torch.bfloat16).to(DEV)
    args = (t(0, 1, 3, 4, 64), t(1, 1, 3, 2, 64), t(2, 1, 3, 2, 64), t(3, 1, 256, 2, 64), t(4, 1, 256, 2, 64), torch.tensor([-1, 0, 0], dtype=torch.int32, device=DEV))
    n = torch.tensor([200], dtype=torch.int32, device=DEV)
    want = pj.decode_tree(*args, kv_lengths=n)
    monkeypatch.setattr(A, "_status_words", {})
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = pj.decode_tree(*args, kv_lengths=n)
    (word,) = A._status_words.values()
    pj.check_status(DEV)
    graph.replay()
    pj.check_status(DEV)
    assert torch.equal(o, want)
    word.fill_(_lib.PJX_ERR_DEVICE_TIMEOUT)  # what a kernel whose wait ran out writes
    with pytest.raises(_lib.KernelTimeout):
        pj.check_status(DEV)
    pj.check_status(DEV)
    del graph, o
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    assert int(word) == 0


def test_two_host_threads_with_different_head_widths():
    """One kernel serves many head widths with shared memory of the call's size: a call of another thread does not take it away."""
    import probjax_b200 as pj

    def job(seed, D):
        t = lambda i, *s: normal(seed + i, *s, dtype=torch.float32).to(DEV)
        q, kn, k = t(0, 1, 20, 4, D), t(1, 1, 20, 2, D), t(2, 1, 130, 2, D)
        lse, par = natural_lse(q.cpu(), k.cpu()).to(DEV), torch.arange(20, dtype=torch.int32, device=DEV) - 1

        def once():
            return pj.decode_tree(q, kn, kn, k, k, par, kv_lengths=[130]), pj.key_weights(q, k, lse)
        return once

    jobs = [job(300, 196), job(310, 256)]  # (both in the instantiation of 256 columns)
    alone = [f() for f in jobs]
    wrong, start = [], threading.Barrier(2)

    def loop(f, want):
        try:
            start.wait(timeout=60)
            for _ in range(100):
                if not all(torch.equal(a, b) for a, b in zip(f(), want)):
                    wrong.append("differs")
        except Exception as e:
            wrong.append(e)

    threads = [threading.Thread(target=loop, args=a) for a in zip(jobs, alone)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong[:3]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_the_exact_tree_kernel_rounds_only_its_result(dtype):
    """16-bit inputs of a head width that the tensor cores do not take: sums in 32 bits, one rounding at the end."""
    import probjax_b200 as pj

    B, N, Hq, Hkv, D, cap = 2, 7, 4, 2, 96, 500
    q, kn, vn = (normal(60 + i, B, N, h, D, dtype=dtype) for i, h in enumerate((Hq, Hkv, Hkv)))
    k, v = normal(63, B, cap, Hkv, D, dtype=dtype), normal(64, B, cap, Hkv, D, dtype=dtype)
    parents, n = [-1, 0, 0, 1, 3, -1, 5], [500, 33]
    o = pj.decode_tree(*(x.to(DEV) for x in (q, kn, vn, k, v)), parents, kv_lengths=n).cpu().double()
    chains = {0: [0], 2: [0, 2], 4: [0, 1, 3, 4], 6: [5, 6]}
    for b in range(B):
        for h in range(Hq):
            for i, c in chains.items():
                keys, vals = torch.cat([k[b, :n[b], h // 2], kn[b, c, h // 2]]), torch.cat([v[b, :n[b], h // 2], vn[b, c, h // 2]])
                r, _, _, tol, _ = attention_row(q[b, i, h], keys, vals, 1 / math.sqrt(D))
                assert bool(((o[b, i, h] - r).abs() <= tol + HALF_STEP[dtype] * (r.abs() + tol)).all())


def loop_inputs(seed, B, N, Hq, Hkv, D):
    return [normal(seed + i, B, N, h, D, dtype=torch.bfloat16).to(DEV) for i, h in enumerate((Hq, Hkv, Hkv))]


def test_accepted_drafts_of_a_ragged_batch_get_their_weights():
    """The recipe of ``DecodeCache.attend_tree``: one call a depth, with that depth's query of every sequence, the lengths up to it and
    lse = +inf where nothing was accepted so deep, adds for a ragged batch what the accepted drafts paid to every key."""
    import probjax_b200 as pj

    B, N, Hq, Hkv, D, cap = 3, 7, 8, 2, 64, 256
    cache = pj.DecodeCache(B, cap, Hkv, D, track_weights=True)
    k0, v0 = (normal(80 + i, B, cap, Hkv, D, dtype=torch.bfloat16).to(DEV) for i in range(2))
    lengths = [150, 64, 0]
    cache.cached_key.copy_(k0)
    cache.cached_value.copy_(v0)
    cache.reset(lengths)
    q, k, v = loop_inputs(82, B, N, Hq, Hkv, D)
    parents = torch.tensor([-1, 0, 0, 1, 2, 3, -9], dtype=torch.int32, device=DEV)
    path = torch.tensor([[0, 1, 3, 5], [0, 2, 4, 6], [0, 0, 0, 0]], dtype=torch.int32, device=DEV)
    counts = torch.tensor([4, 3, 1], dtype=torch.int32, device=DEV)
    old, before = cache.cache_index.clone(), cache.key_weights.clone()
    _, lse = cache.attend_tree(q, k, v, parents, return_lse=True)
    cache.accept(k, v, path, counts)
    for i in range(path.shape[1]):
        at = path[:, i].long()[:, None]
        q_i = q.gather(1, at[:, :, None, None].expand(B, 1, Hq, D))
        l_i = lse.gather(2, at[:, None].expand(B, Hq, 1)).masked_fill((i >= counts)[:, None, None], math.inf)
        pj.key_weights(q_i, cache.cached_key, l_i, weights=cache.key_weights, mask=pj.KVLenMask(old + i + 1), out=cache.key_weights)
    pj.check_status(DEV)
    grown = (cache.key_weights - before).cpu().double()
    want, tol = torch.zeros(B, Hkv, cap, dtype=torch.float64), torch.zeros(B, Hkv, cap, dtype=torch.float64)
    keys = cache.cached_key.cpu()
    for b in range(B):
        for i in range(int(counts[b])):
            n, node = lengths[b] + i + 1, int(path[b, i])
            for h in range(Hq):
                _, _, p, _, rel = attention_row(q[b, node, h].cpu(), keys[b, :n, h // 4], keys[b, :n, h // 4], 1 / math.sqrt(D))
                want[b, h // 4, :n] += p
                tol[b, h // 4, :n] += p * (2 * rel + 2.0 ** -20)  # (rel of the weight's own score and of the lse that the tree call gave)
    assert bool(((grown - want).abs() <= tol + 2.0 ** -22 * (want + before.cpu().double())).all())
    for b in range(B):  # every accepted draft paid one in all for each of its heads
        assert abs(float(grown[b].sum()) - Hq * int(counts[b])) <= 2.0 ** -12 * Hq * int(counts[b])


def test_draft_verify_accept_and_evict_in_one_graph():
    """A step of the loop -- verification, acceptance, a tracked decode step, eviction -- captured once and replayed for three steps of new
    inputs leaves what the same calls leave one by one."""
    import probjax_b200 as pj

    B, N, Hq, Hkv, D, cap, keep = 2, 6, 8, 2, 128, 160, 96
    caches = [pj.DecodeCache(B, cap, Hkv, D, track_weights=True) for _ in range(2)]
    k0, v0, w0 = (normal(90 + i, *s, dtype=x).to(DEV) for i, (s, x) in enumerate((((B, cap, Hkv, D), torch.bfloat16), ((B, cap, Hkv, D), torch.bfloat16),
                                                                                  ((B, Hkv, cap), torch.float32))))
    parents = torch.tensor([-1, 0, 0, 1, 2, 4], dtype=torch.int32, device=DEV)

    def start(c):
        c.cached_key.copy_(k0)
        c.cached_value.copy_(v0)
        c.reset([90, 60])
        c.key_weights.copy_(w0.abs() * (torch.arange(cap, device=DEV) < 60))

    def step(c, drafts, token, path, counts):
        o, lse = c.attend_tree(*drafts, parents, return_lse=True)
        c.accept(drafts[1], drafts[2], path, counts)
        s = c.step(*token)
        return o, lse, s, c.evict(keep, recent=8)

    ins = [(loop_inputs(100 + 10 * i, B, N, Hq, Hkv, D), loop_inputs(200 + 10 * i, B, 1, Hq, Hkv, D),
            torch.tensor([[0, 1, 3, 3], [0, 2, 4, 5]], dtype=torch.int32, device=DEV), torch.tensor([3, 4 - i], dtype=torch.int32, device=DEV)) for i in range(3)]
    for c in caches:
        start(c)
    held = [[x.clone() for x in part] if isinstance(part, list) else part.clone() for part in ins[0]]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(caches[0], *held)
    start(caches[0])
    for args in ins:
        for a, b in zip(held, args):
            for x, y in zip(a, b) if isinstance(a, list) else ((a, b),):
                x.copy_(y)
        graph.replay()
        want = step(caches[1], *args)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        for b in range(B):
            n = int(caches[1].cache_index[b])
            assert int(caches[0].cache_index[b]) == n
            assert torch.equal(caches[0].cached_key[b, :n], caches[1].cached_key[b, :n]) and torch.equal(caches[0].cached_value[b, :n], caches[1].cached_value[b, :n])
        assert torch.equal(caches[0].key_weights, caches[1].key_weights)
    assert int(caches[1].cache_index[0]) == keep  # (it was cut on the way)
    pj.check_status(DEV)


@pytest.mark.parametrize("cap,keep,recent", [(33_000, 5000, 7), (70_001, 20_000, 0), (140_000, 129_999, 50), (300_003, 1000, 50), (300_003, 262_145, 0)])
@pytest.mark.parametrize("place", ["in place", "other buffers"])
def test_eviction_from_long_caches_keeps_the_right_keys(cap, keep, recent, place):
    """Two, four and eight CTAs a head, and more weights than they hold in shared memory.  The kept keys against a stable sort of a copy of
    the weights, which take 4096 values and zero, so that the threshold cuts through ties."""
    import probjax_b200 as pj

    Hkv, D = 2, 8
    g = torch.Generator().manual_seed(cap + keep)
    k, v = normal(70, 1, cap, Hkv, D, dtype=torch.bfloat16), normal(71, 1, cap, Hkv, D, dtype=torch.bfloat16)
    w = torch.randint(0, 4096, (1, Hkv, cap), generator=g).float() / 64
    kd, vd, wd = k.to(DEV), v.to(DEV), w.to(DEV)
    out = None if place == "in place" else tuple(torch.zeros(s, dtype=x, device=DEV) for s, x in (
        ((1, keep, Hkv, D), k.dtype), ((1, keep, Hkv, D), k.dtype), ((1, Hkv, keep), w.dtype)))
    n, idx = pj.evict(kd, vd, wd, [cap], keep, recent=recent, out=out)
    ko, vo, wo = (kd, vd, wd) if out is None else out
    assert n.tolist() == [keep]
    for h in range(Hkv):
        order = torch.sort(w[0, h, :cap - recent], descending=True, stable=True).indices[:keep - recent]
        rows = torch.cat([order.sort().values, torch.arange(cap - recent, cap)])
        assert torch.equal(idx[0, h].cpu().long(), rows)
        assert torch.equal(ko[0, :keep, h].cpu(), k[0, rows, h]) and torch.equal(vo[0, :keep, h].cpu(), v[0, rows, h])
        assert torch.equal(wo[0, h, :keep].cpu(), w[0, h, rows])
    if out is None:
        assert not bool(wd[:, :, keep:].any())


def test_positions_count_tokens_and_not_kept_keys():
    """Decode steps with rotary positions over a cache that is cut on the way: a step's angles follow the tokens seen, the kept keys keep theirs,
    and attention is that of the kept tokens at their places in the text."""
    import probjax_b200 as pj

    B, Hq, Hkv, D, cap, keep = 2, 4, 2, 64, 64, 20
    cache = pj.DecodeCache(B, cap, Hkv, D, track_weights=True)
    seen = torch.zeros(B, dtype=torch.int32, device=DEV)
    places = [[[] for _ in range(Hkv)] for _ in range(B)]  # the tokens that every head holds
    k_all, v_all = [], []
    for i in range(60):
        q, k, v = (normal(400 + 3 * i + j, B, 1, h, D) for j, h in enumerate((Hq, Hkv, Hkv)))
        q, k, v = q.bfloat16().to(DEV), k.bfloat16().to(DEV), v.bfloat16().to(DEV)
        pos = seen[:, None, None]
        qr, kr = pj.rope_axes(q, pos, (D,)), pj.rope_axes(k, pos, (D,))
        o = cache.step(qr, kr, v)
        k_all.append(kr[:, 0].cpu())
        v_all.append(v[:, 0].cpu())
        seen += 1
        for b in range(B):
            for h in range(Hkv):
                places[b][h].append(i)
        if i % 25 == 24:
            kept = cache.evict(keep, recent=5).cpu()
            for b in range(B):
                for h in range(Hkv):
                    places[b][h] = [places[b][h][j] for j in kept[b, h].tolist()]
    assert cache.cache_index.tolist() == [30, 30] and seen.tolist() == [60, 60]
    for b in range(B):
        for h in range(Hq):
            at = places[b][h // 2]
            keys, vals = torch.stack([k_all[i][b, h // 2] for i in at]), torch.stack([v_all[i][b, h // 2] for i in at])
            r, _, p, tol, _ = attention_row(qr[b, 0, h].cpu(), keys, vals, 1 / math.sqrt(D))
            bound = tol + HALF_STEP[torch.bfloat16] * (p @ vals.double().abs() + r.abs())
            assert bool(((o[b, 0, h].cpu().double() - r).abs() <= bound).all())
    pj.check_status(DEV)


def test_two_host_threads_with_different_head_widths_in_training():
    """The same for the forward and backward kernels on CUDA cores."""
    import probjax_b200 as pj

    def job(seed, D):
        q, k, dy = (normal(seed + i, 1, n, 2, D).to(DEV) for i, n in enumerate((70, 90, 70)))
        o, lse = pj.attention_forward(q, k, k, sm_scale=0.07, return_lse=True)
        return lambda: (pj.attention_forward(q, k, k, sm_scale=0.07), *pj.attention.attention_backward(q, k, k, o, lse, dy, sm_scale=0.07))

    jobs = [job(320, 196), job(330, 256)]
    alone = [f() for f in jobs]
    wrong, start = [], threading.Barrier(2)

    def loop(f, want):
        try:
            start.wait(timeout=60)
            for _ in range(100):
                if not all(torch.equal(a, b) for a, b in zip(f(), want)):
                    wrong.append("differs")
        except Exception as e:
            wrong.append(e)

    threads = [threading.Thread(target=loop, args=a) for a in zip(jobs, alone)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong[:3]


def test_rope_axes_refuses_positions_that_ask_for_a_gradient():
    import probjax_b200 as pj

    x, pos = torch.zeros(1, 3, 2, 8, device=DEV), torch.zeros(3, 1, device=DEV, requires_grad=True)
    with pytest.raises(NotImplementedError, match="positions"):
        pj.rope_axes(x, pos, (8,))
    with torch.no_grad():
        pj.rope_axes(x, pos, (8,))
    pj.rope_axes(x, pos.detach(), (8,))


def test_results_written_in_place_are_seen_by_autograd():
    """A gradient that needs what a call has overwritten is refused: lengths that an acceptance or an eviction advances, as rotary positions,
    and tensors that take results."""
    import probjax_b200 as pj

    t = lambda i, *s: normal(500 + i, *s).to(DEV)
    x, k, v, kn, w = t(0, 2, 1, 2, 8).requires_grad_(True), t(1, 2, 32, 2, 8), t(2, 2, 32, 2, 8), t(3, 2, 3, 2, 8), t(4, 2, 2, 32).abs()
    n = torch.tensor([9, 20], dtype=torch.int32, device=DEV)
    lse, q = torch.zeros(2, 2, 1, device=DEV), t(5, 2, 1, 2, 8)
    calls = [
        (n, lambda: pj.accept_drafts(kn, kn, k, v, [[0, 1], [2, 0]], [2, 1], kv_lengths=n, out=n)),
        (n, lambda: pj.evict(k, v, w, n, 10, lengths_out=n)),
        (k, lambda: pj.evict(k, v, w, n, 10)),
        (v, lambda: pj.accept_drafts(kn, kn, k, v, [[0], [2]], [1, 1], kv_lengths=n)),
        (w, lambda: pj.decode_weights(q, k, v, w, out=w)),
        (w, lambda: pj.key_weights(q, k, lse, weights=w, out=w)),
        (k, lambda: pj.rope_axes(k, torch.zeros(32, 1, device=DEV), (8,), out=k)),
    ]
    for changed, call in calls:
        y = pj.rope_axes(x, n[:, None, None], (8,))
        leaf = torch.ones((), device=DEV, requires_grad=True)
        z = (leaf * changed).sum()  # (needs `changed` for the leaf's gradient)
        call()
        if changed is n:
            with pytest.raises(RuntimeError, match="changed in place"):
                y.sum().backward()
        with pytest.raises(RuntimeError, match="inplace"):
            z.backward()
    with torch.inference_mode():
        a, b, m = k.clone(), v.clone(), n.clone()
        pj.evict(a, b, w.clone(), m, 4, lengths_out=m)
        assert m.tolist() == [4, 4]
