"""The drafted-tree, key-weight and eviction calls on caches whose offsets pass 32 bits, on other streams, and captured with their
backward pass; refusals of the Python entry points."""

import math

import pytest
import torch

from _operators_ref import HALF_STEP, attention_row, rope_reference

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_offsets_beyond_32_bits():
    """2.2 million keys of 8 heads of 128: more than 2^31 elements.  All keys but the last 200 are zero, so that their score is zero and
    their values add nothing: the exact result needs the last rows and a count."""
    import probjax_b200 as pj

    cap, Hkv, Hq, D, N, live = 2_200_000, 8, 16, 128, 5, 200
    g = torch.Generator().manual_seed(1)
    t = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16)
    k, v = (torch.zeros((1, cap, Hkv, D), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    kl, vl = t(live, Hkv, D) * 3, t(live, Hkv, D)
    k[0, cap - live:], v[0, cap - live:] = kl.to(DEV), vl.to(DEV)
    q, kn, vn = t(1, N, Hq, D) * 2, t(1, N, Hkv, D), t(1, N, Hkv, D)
    parents = torch.tensor([-1, 0, 1, 0, -1], dtype=torch.int32)
    o, lse = pj.decode_tree(q.to(DEV), kn.to(DEV), vn.to(DEV), k, v, parents.to(DEV), kv_lengths=[cap], return_lse=True)
    step, w = pj.decode_weights(q[:, :1].to(DEV), k, v, kv_lengths=[cap])
    s_lse = pj.decode_forward(q[:, :1].to(DEV), k, v, sm_scale=1 / math.sqrt(D), return_lse=True)[1]
    w2 = pj.key_weights(q[:, :1].to(DEV), k, s_lse)
    pj.check_status(DEV)
    zeros = cap - live
    for h in range(Hq):
        gk = h // (Hq // Hkv)
        for i, chain in ((0, [0]), (2, [0, 1, 2]), (3, [0, 3])):
            keys, vals = torch.cat([kl[:, gk], kn[0, chain, gk]]), torch.cat([vl[:, gk], vn[0, chain, gk]])
            r, l, p, tol, rel = attention_row(q[0, i, h], keys, vals, 1 / math.sqrt(D))
            total = math.log(math.exp(l) + zeros)
            f = math.exp(l - total)  # the share of the keys that are not zero
            u = HALF_STEP[torch.bfloat16]
            bound = f * (tol + u * (p @ vals.double().abs() + r.abs())) + f * r.abs() * cap * 2.0 ** -23 / 64  # (each sum adds 64 and more at a time)
            assert bool(((o[0, i, h].cpu().double() - f * r).abs() <= bound).all())
            assert abs(float(lse[0, h, i]) - total) <= rel + cap * 2.0 ** -23 / 64 + 2.0 ** -18
    want = torch.zeros(Hkv, live, dtype=torch.float64)
    first = torch.zeros(Hkv, dtype=torch.float64)
    for h in range(Hq):
        s = kl[:, h // 2].double() @ q[0, 0, h].double() / math.sqrt(D)
        total = torch.logsumexp(s, 0).exp() + zeros
        want[h // 2] += s.exp() / total
        first[h // 2] += 1 / total
    # a thread's part of a row's sum is a chain of at most 4000 additions in 32 bits, 2^-24 each: below 2^-12; the scores' own error
    # (128 products, |s| below 60, as in attention_row) is below 2^-11
    for got in (w, w2):
        assert bool(((got[0, :, zeros:].cpu().double() - want).abs() <= 2.0 ** -10 * want).all())
        assert bool(((got[0, :, [0, zeros - 1]].cpu().double() - first[:, None]).abs() <= 2.0 ** -10 * first[:, None]).all())
    new, kept = pj.evict(k, v, w, [cap], 300, recent=50)
    assert new.tolist() == [300]
    for h in range(Hkv):
        idx = kept[0, h].long()
        assert bool((idx[1:] > idx[:-1]).all()) and idx[-50:].tolist() == list(range(cap - 50, cap))
        top = torch.topk(w[0, h], 1).values  # (the weights moved with their keys)
        assert float(w[0, h, :300].max()) == float(top)
        tail = idx >= zeros
        assert torch.equal(k[0, :300, h][tail].cpu(), kl[(idx[tail] - zeros).cpu(), h]) and bool((k[0, :300, h][~tail] == 0).all())
    del k, v
    torch.cuda.empty_cache()


def test_calls_on_a_side_stream():
    """Work queued on another stream than the current one of the test, behind the kernels that make its inputs."""
    import probjax_b200 as pj

    g = torch.Generator().manual_seed(2)
    t = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16).to(DEV)
    q, kn, vn, k, v = t(2, 6, 8, 128), t(2, 6, 2, 128), t(2, 6, 2, 128), t(2, 4096, 2, 128), t(2, 4096, 2, 128)
    parents, n = torch.tensor([-1, 0, 0, 1, 3, 2], dtype=torch.int32, device=DEV), torch.tensor([4000, 17], dtype=torch.int32, device=DEV)
    want = (pj.decode_tree(q, kn, vn, k, v, parents, kv_lengths=n), *pj.decode_weights(q[:, :1], k, v, kv_lengths=n))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        late = [x.clone() for x in (q, kn, vn, k, v)]  # produced on this stream just before
        got = (pj.decode_tree(*late, parents, kv_lengths=n), *pj.decode_weights(late[0][:, :1], late[3], late[4], kv_lengths=n))
    side.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a, b)


def test_captured_rotary_training_step():
    """Forward and gradient of the rotary embedding captured in one graph, while an eager graph of another leaf is alive."""
    import probjax_b200 as pj

    g = torch.Generator().manual_seed(3)
    x = torch.randn(2, 9, 4, 64, generator=g).to(DEV)
    pos = torch.randint(0, 99, (2, 9, 2), generator=g).to(DEV)
    other = x.clone().requires_grad_(True)
    eager = pj.rope_axes(other, pos, (32, 32))
    leaf, dy = x.clone().requires_grad_(True), torch.randn(2, 9, 4, 64, generator=g).to(DEV)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = pj.rope_axes(leaf, pos, (32, 32))
        (dx,) = torch.autograd.grad(y, leaf, dy)
    with torch.no_grad():
        leaf.copy_(2 * x)
    graph.replay()
    torch.cuda.synchronize()
    want, tol = rope_reference(2 * x.cpu(), pos.cpu(), (32, 32))
    assert bool(((y.detach().cpu().double() - want).abs() <= tol).all())
    want, tol = rope_reference(dy.cpu(), pos.cpu(), (32, 32), sign=-1)
    assert bool(((dx.cpu().double() - want).abs() <= tol).all())
    (g2,) = torch.autograd.grad(eager, other, dy)
    assert torch.equal(g2, dx)


def test_refusals_of_the_python_calls():
    import probjax_b200 as pj

    z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype, device=DEV)
    q, kn, k = z(2, 3, 4, 64), z(2, 3, 2, 64), z(2, 8, 2, 64)
    par = torch.zeros(3, dtype=torch.int32)
    ok = lambda **kw: pj.decode_tree(*[kw.get(n, d) for n, d in (("q", q), ("kn", kn), ("vn", kn), ("k", k), ("v", k), ("par", par))],
                                     kv_lengths=kw.get("n", [1, 1]), block_table=kw.get("table"), implementation=kw.get("impl"))
    ok()
    for kw in (dict(q=q.float()), dict(kn=kn.half()), dict(q=z(2, 3, 3, 64)), dict(q=z(2, 4, 4, 64)), dict(q=q[0]), dict(k=z(3, 8, 2, 64), v=z(3, 8, 2, 64)),
               dict(k=z(2, 8, 1, 64)), dict(vn=z(2, 3, 1, 64)), dict(par=torch.zeros(4, dtype=torch.int32)), dict(par=torch.zeros(3)), dict(n=[1]), dict(n=[1.0, 2.0]),
               dict(impl="x"), dict(table=torch.zeros(3, 1, dtype=torch.int32)), dict(table=[[0], [0]]), dict(q=q.cpu()), dict(k=k.double(), v=k.double())):
        with pytest.raises(ValueError):
            ok(**kw)
    with pytest.raises(NotImplementedError, match="256"):
        pj.decode_tree(z(1, 257, 2, 64), z(1, 257, 2, 64), z(1, 257, 2, 64), z(1, 8, 2, 64), z(1, 8, 2, 64), torch.zeros(257, dtype=torch.int32), kv_lengths=[0])
    with pytest.raises(NotImplementedError):
        ok(q=z(2, 3, 4, 64, dtype=torch.float32), kn=kn.float(), vn=kn.float(), k=k.float(), v=k.float(), impl="b200:tcgen05")
    path, cnt = torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="contiguous"):
        pj.accept_drafts(kn, kn, k.transpose(0, 1).contiguous().transpose(0, 1), k, path, cnt, kv_lengths=[0, 0])
    with pytest.raises(ValueError, match="inside the cache"):
        pj.accept_drafts(k[:, :3], kn, k, k.clone(), path, cnt, kv_lengths=[0, 0])
    for kw in (dict(out=torch.zeros(2, device=DEV)), dict(out=torch.zeros(3, dtype=torch.int32, device=DEV)), dict(overflow=torch.zeros(2, dtype=torch.int32, device=DEV))):
        with pytest.raises(ValueError):
            pj.accept_drafts(kn, kn, k, k.clone(), path, cnt, kv_lengths=[0, 0], **kw)
    w = z(2, 2, 8, dtype=torch.float32)
    for bad in (w.double(), w[:, :1], w[..., :7], w.cpu()):
        with pytest.raises(ValueError):
            pj.decode_weights(q[:, :1], k, k, bad)
        with pytest.raises(ValueError):
            pj.evict(k.clone(), k.clone(), bad, [8, 8], 2)
    both = torch.zeros(2 * 2 * 8 + 4, device=DEV)
    with pytest.raises(ValueError, match="overlap"):
        pj.decode_weights(q[:, :1], k, k, both[:32].view(2, 2, 8), out=both[4:36].view(2, 2, 8))
    lse = z(2, 4, 3, dtype=torch.float32)
    with pytest.raises(NotImplementedError):
        pj.key_weights(q, k, lse, mask=pj.PrefixLMMask(torch.tensor([2, 2])))
    with pytest.raises(ValueError):
        pj.key_weights(q, k, lse[:, :, :2])
    with pytest.raises(ValueError):
        pj.key_weights(q, k, lse.half())
    for kw in (dict(keep=0), dict(keep=2, recent=3), dict(keep=2, recent=-1), dict(keep=4, out=(z(2, 3, 2, 64), z(2, 3, 2, 64), z(2, 2, 3, dtype=torch.float32))),
               dict(keep=2, out=(z(2, 3, 2, 64), z(2, 4, 2, 64), z(2, 2, 3, dtype=torch.float32))), dict(keep=2, out=(k, z(2, 8, 2, 64), w))):
        with pytest.raises(ValueError):
            pj.evict(k, k.clone(), w, [8, 8], **kw)
    x, pos = z(2, 5, 2, 64), torch.zeros(2, 5, 2, dtype=torch.int32)
    for args in ((x, pos, (32, 31)), (x, pos, (64, 2)), (x, pos, (32,)), (x, pos[:, :4], (32, 32)), (x.cpu(), pos, (32, 32)), (x.double(), pos, (32, 32)),
                 (x, pos.bool(), (32, 32)), (x[0, 0], pos, (32, 32))):
        with pytest.raises(ValueError):
            pj.rope_axes(*args)
    with pytest.raises(ValueError, match="overlaps"):
        buf = z(21, 2, 64)
        pj.rope_axes(buf[:20].view(2, 10, 2, 64), torch.zeros(10, 1, dtype=torch.int32), (64,), out=buf[1:].view(2, 10, 2, 64))
    with pytest.raises(ValueError, match="gradient"):
        pj.rope_axes(z(1, 2, 1, 64, dtype=torch.float32).requires_grad_(True), torch.zeros(2, 1), (64,), out=z(1, 2, 1, 64, dtype=torch.float32))
    cache = pj.DecodeCache(1, 8, 1, 64)
    with pytest.raises(ValueError, match="track_weights"):
        cache.evict(2)
    with pytest.raises(ValueError, match="window"):
        cache.attend(z(1, 1, 1, 64), window=3)
    pj.check_status(DEV)
