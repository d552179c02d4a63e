"""Drafted trees over a cache (``decode_tree``, ``accept_drafts``) against 64-bit references."""

import math

import pytest
import torch

from _operators_ref import pages_to_rows, tree_reference

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def make(B, N, Hq, Hkv, D, cap, lengths, dtype, seed, page=0, Dv=None, garbage=float("nan")):
    """Inputs on the CPU; cache rows behind a sequence's length hold ``garbage``, and so do unused pages."""
    g = torch.Generator().manual_seed(seed)
    Dv = D if Dv is None else Dv
    t = lambda *s: torch.randn(*s, generator=g).to(dtype)
    q, kn, vn = t(B, N, Hq, D), t(B, N, Hkv, D), t(B, N, Hkv, Dv)
    table = None
    if page:
        pages = -(-cap // page)
        cap = pages * page
        table = torch.randperm(B * pages + 3, generator=g)[:B * pages].reshape(B, pages).to(torch.int32)
        k, v = torch.full((B * pages + 3, page, Hkv, D), garbage, dtype=dtype), torch.full((B * pages + 3, page, Hkv, Dv), garbage, dtype=dtype)
        for b in range(B):
            for j in range(lengths[b]):
                k[int(table[b, j // page]), j % page] = t(Hkv, D)
                v[int(table[b, j // page]), j % page] = t(Hkv, Dv)
    else:
        k, v = t(B, cap, Hkv, D), t(B, cap, Hkv, Dv)
        for b in range(B):
            k[b, lengths[b]:] = garbage
            v[b, lengths[b]:] = garbage
    parents = torch.full((B, N), -7, dtype=torch.int32)
    for b in range(B):
        n = N if b == 0 else max(1, N - b)
        for i in range(n):
            r = float(torch.rand((), generator=g))
            parents[b, i] = -1 if r < 0.2 or i == 0 else i - 1 - int(torch.randint(0, min(i, 5), (), generator=g))
    return q, kn, vn, k, v, parents, torch.tensor(lengths, dtype=torch.int32), table


def run(case, **kw):
    import probjax_b200 as pj

    q, kn, vn, k, v, parents, lengths, table = case
    d = [x.to(DEV) for x in (q, kn, vn, k, v, parents)]
    o, lse = pj.decode_tree(*d, kv_lengths=lengths.to(DEV), block_table=None if table is None else table.to(DEV), return_lse=True, **kw)
    pj.check_status(DEV)
    return o.cpu(), lse.cpu()


def check(case, o, lse, scale=None):
    want, want_l, tol, tol_l = tree_reference(*case, scale=scale)
    assert torch.isfinite(o).all()
    assert torch.equal(torch.isinf(lse), torch.isinf(want_l))
    err = (o.double() - want).abs()
    assert bool((err <= tol).all()), f"worst error / bound {float((err / tol.clamp(min=1e-30)).max()):.3f}"
    fin = torch.isfinite(want_l)
    assert bool(((lse.double() - want_l).abs()[fin] <= tol_l[fin]).all())


CASES = [  # B, N, Hq, Hkv, D, cap, lengths, dtype, page
    (1, 1, 4, 1, 128, 128, [0], torch.bfloat16, 0),           # one draft and an empty context
    (1, 1, 8, 2, 64, 300, [300], torch.float16, 0),           # one token over a full cache
    (3, 9, 8, 2, 128, 400, [127, 128, 129], torch.bfloat16, 0),
    (2, 33, 6, 2, 64, 700, [641, 0], torch.bfloat16, 0),      # 3 heads a group, 99 rows
    (2, 17, 14, 2, 128, 260, [255, 1], torch.float16, 0),     # 7 heads a group
    (1, 128, 4, 4, 64, 200, [77], torch.bfloat16, 0),         # no shared heads: as many rows as drafts
    (1, 256, 2, 1, 128, 640, [513], torch.bfloat16, 0),       # the most drafts
    (1, 129, 4, 2, 64, 256, [130], torch.float16, 0),         # drafts in two tiles
    (2, 20, 16, 1, 128, 512, [300, 511], torch.bfloat16, 0),  # one KV head, 320 rows
    (1, 3, 96, 1, 64, 256, [200], torch.float16, 0),          # one token of rows a tile
    (3, 12, 8, 2, 128, 512, [500, 16, 0], torch.bfloat16, 16),
    (2, 12, 8, 2, 64, 512, [479, 480], torch.float16, 48),    # a page size that is not a power of two
    (2, 40, 4, 1, 128, 1024, [1000, 64], torch.bfloat16, 64),
    (2, 5, 4, 2, 128, 768, [700, 300], torch.bfloat16, 256),
    (2, 9, 4, 2, 64, 256, [100, 3], torch.float32, 0),
    (2, 70, 3, 1, 80, 256, [100, 0], torch.float32, 32),
    (2, 9, 4, 2, 96, 256, [200, 64], torch.bfloat16, 0),      # a head width the tensor-core kernel does not take
]


@pytest.mark.parametrize("B,N,Hq,Hkv,D,cap,lengths,dtype,page", CASES)
def test_tree_matches_the_formula(B, N, Hq, Hkv, D, cap, lengths, dtype, page):
    case = make(B, N, Hq, Hkv, D, cap, lengths, dtype, seed=N * 1000 + D, page=page)
    check(case, *run(case))


@pytest.mark.parametrize("impl", ["b200:generic", None])
def test_both_kernels_and_unequal_head_widths(impl):
    case = make(2, 11, 8, 2, 128, 512, [333, 512], torch.bfloat16, seed=5)
    check(case, *run(case, implementation=impl, sm_scale=0.11), scale=0.11)
    case = make(1, 6, 4, 2, 64, 128, [90], torch.float16, seed=6, Dv=40)
    check(case, *run(case, implementation=impl))


def test_many_sequences():
    """More sequences than are dealt out from the lengths on the device."""
    lengths = [(37 * b) % 190 for b in range(150)]
    case = make(150, 3, 2, 1, 64, 192, lengths, torch.bfloat16, seed=8)
    check(case, *run(case))


def test_shared_tree_chain_and_invalid_parents():
    """One tree for all sequences; a chain; parents that point at themselves, forwards or nowhere are absent, with what hangs on them."""
    case = list(make(2, 6, 4, 2, 64, 128, [60, 128], torch.bfloat16, seed=9))
    for parents in ([-1, 0, 1, 2, 3, 4], [-1, 1, 0, 5, -1, -5], [-2, 0, 1, 2, 3, 4], [-1, 0, 2147483647, 2, -2147483648, 0]):
        case[5] = torch.tensor(parents, dtype=torch.int32)
        check(case, *run(case))


def test_absent_drafts_may_hold_anything():
    """Keys, values and queries of absent drafts are NaN or infinite; nobody's result changes, and theirs are zero."""
    q, kn, vn, k, v, parents, lengths, table = make(2, 10, 4, 2, 128, 256, [200, 100], torch.bfloat16, seed=10)
    parents = torch.tensor([[-1, 0, -9, 1, 2, 1, -9, 0, 3, 8]] * 2, dtype=torch.int32)
    for i in (2, 4, 6):
        kn[:, i], vn[:, i], q[:, i] = float("nan"), float("inf"), float("nan")
    case = (q, kn, vn, k, v, parents, lengths, table)
    o, lse = run(case)
    check(case, o, lse)
    assert (o[:, [2, 4, 6]] == 0).all()


def test_lengths_beyond_the_capacity_and_below_zero():
    case = list(make(2, 4, 4, 2, 64, 100, [100, 0], torch.bfloat16, seed=11))
    want = run(case)
    case[6] = torch.tensor([5000, -3], dtype=torch.int32)
    got = run(case)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_pages_outside_the_pool_read_as_zeros():
    case = list(make(1, 5, 4, 2, 64, 256, [200], torch.bfloat16, seed=12, page=64))
    bad = [x.clone() if isinstance(x, torch.Tensor) else x for x in case]
    page = int(bad[7][0, 1])
    bad[3][page], bad[4][page] = 0, 0
    want = run(bad)
    for number in (-1, 10 ** 6, 2 ** 31 - 1, -2 ** 31):
        case[7] = bad[7].clone()
        case[7][0, 1] = number
        got = run(case)
        assert torch.equal(got[0], want[0])


def test_an_empty_pool():
    """No page at all: nothing cached, or keys that all read as zeros."""
    case = list(make(1, 4, 4, 2, 64, 64, [0], torch.bfloat16, seed=15, page=64))
    want = run(case)
    case[3], case[4] = case[3][:0], case[4][:0]
    got = run(case)
    check(case, *got)
    assert float((got[0] - want[0]).abs().max()) <= 2.0 ** -7 * 4  # (the other kernel: a rounding of P and one of the result, |v| < 4)
    case[6] = torch.tensor([10], dtype=torch.int32)
    zeros = list(case)
    zeros[3], zeros[4], zeros[7] = torch.zeros(1, 64, 2, 64, dtype=torch.bfloat16), torch.zeros(1, 64, 2, 64, dtype=torch.bfloat16), torch.zeros(1, 1, dtype=torch.int32)
    check(zeros, *run(case))


def test_slices_of_a_fused_projection_and_unaligned_inputs():
    import probjax_b200 as pj

    q, kn, vn, k, v, parents, lengths, _ = make(2, 7, 8, 2, 64, 128, [100, 50], torch.bfloat16, seed=13)
    want = run((q, kn, vn, k, v, parents, lengths, None))
    fused = torch.cat([q, kn, vn], 2).to(DEV)
    o, lse = pj.decode_tree(fused[:, :, :8], fused[:, :, 8:10], fused[:, :, 10:], k.to(DEV), v.to(DEV), parents.to(DEV), kv_lengths=lengths.to(DEV),
                            return_lse=True)
    assert torch.equal(o.cpu(), want[0]) and torch.equal(lse.cpu(), want[1])
    flat = torch.empty(q.numel() + 1, dtype=q.dtype, device=DEV)
    odd = flat[1:].view(q.shape).copy_(q)
    heads_first = kn.to(DEV).transpose(1, 2).contiguous().transpose(1, 2)
    o = pj.decode_tree(odd, heads_first, vn.to(DEV), k.to(DEV), v.to(DEV), parents.to(DEV), kv_lengths=lengths.to(DEV))
    assert torch.equal(o.cpu(), want[0])
    odd_cache = torch.empty(k.numel() + 1, dtype=k.dtype, device=DEV)[1:].view(k.shape).copy_(k)
    got = pj.decode_tree(q.to(DEV), kn.to(DEV), vn.to(DEV), odd_cache, v.to(DEV), parents.to(DEV), kv_lengths=lengths.to(DEV), return_lse=True)
    check((q, kn, vn, k, v, parents, lengths, None), got[0].cpu(), got[1].cpu())  # (the exact kernel takes it)


def test_empty_calls():
    import probjax_b200 as pj

    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device=DEV)
    o = pj.decode_tree(z(0, 3, 4, 64), z(0, 3, 2, 64), z(0, 3, 2, 64), z(0, 8, 2, 64), z(0, 8, 2, 64), torch.zeros(3, dtype=torch.int32),
                       kv_lengths=torch.zeros(0, dtype=torch.int32))
    assert o.shape == (0, 3, 4, 64)
    o = pj.decode_tree(z(2, 0, 4, 64), z(2, 0, 2, 64), z(2, 0, 2, 64), z(2, 8, 2, 64), z(2, 8, 2, 64), torch.zeros((2, 0), dtype=torch.int32),
                       kv_lengths=[3, 3])
    assert o.shape == (2, 0, 4, 64)
    case = make(1, 4, 4, 2, 64, 0, [0], torch.bfloat16, seed=14)  # no cache at all
    check(case, *run(case))


def test_results_repeat_and_graphs_replay_side_by_side():
    """Bit-repeatable; two captured calls replayed at once on two streams do not share scratch memory."""
    import probjax_b200 as pj

    cases = [make(2, 16, 8, 2, 128, 2048, [2000, 1500], torch.bfloat16, seed=s) for s in (20, 21)]
    want = [run(c) for c in cases]
    again = [run(c) for c in cases]
    for a, b in zip(want, again):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    graphs, outs, keep = [], [], []
    for c in cases:
        d = [x.to(DEV) for x in c[:7]]
        keep.append(d)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(pj.decode_tree(*d[:6], kv_lengths=d[6], return_lse=True))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o[0].cpu(), w[0]) and torch.equal(o[1].cpu(), w[1])


# ------------------------------------------------------------------------------------------------ accept


def accept_reference(kn, vn, k, v, path, counts, lengths, table):
    k, v = k.clone(), v.clone()
    cap = k.shape[1] if table is None else table.shape[1] * k.shape[1]
    new = []
    for b in range(kn.shape[0]):
        n = max(0, int(lengths[b]))
        c = min(max(0, int(counts[b])), path.shape[1])
        for i in range(c):
            node, row = int(path[b, i]), n + i
            if 0 <= node < kn.shape[1] and row < cap:
                at = (b, row) if table is None else (int(table[b, row // k.shape[1]]), row % k.shape[1])
                if table is not None and not 0 <= at[0] < k.shape[0]:
                    continue
                k[at], v[at] = kn[b, node], vn[b, node]
        new.append(min(cap, n + c))
    return k, v, torch.tensor(new, dtype=torch.int32)


@pytest.mark.parametrize("dtype,page,Hkv,D,Dv", [(torch.bfloat16, 0, 8, 128, 128), (torch.float16, 16, 2, 64, 64), (torch.float32, 3, 1, 20, 12),
                                                 (torch.bfloat16, 64, 3, 80, 80)])
def test_accept_writes_the_path_and_nothing_else(dtype, page, Hkv, D, Dv):
    import probjax_b200 as pj

    B, N = 4, 19
    _, kn, vn, k, v, _, lengths, table = make(B, N, Hkv, Hkv, D, 90, [0, 40, 87, 5], dtype, seed=30, page=page, Dv=Dv, garbage=3.0)
    path = torch.tensor([[0, 3, 7, 18], [2, 2, 1, 0], [4, 5, 6, 7], [9, -1, 19, 3]], dtype=torch.int32)
    counts = torch.tensor([4, 3, 9, 4], dtype=torch.int32)  # (a count past the path's width is cut, row 2 ends at the capacity)
    want = accept_reference(kn, vn, k, v, path, counts, lengths, table)
    kd, vd, over = k.to(DEV), v.to(DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    new = pj.accept_drafts(kn.to(DEV), vn.to(DEV), kd, vd, path.to(DEV), counts.to(DEV), kv_lengths=lengths.to(DEV),
                           block_table=None if table is None else table.to(DEV), overflow=over)
    assert torch.equal(kd.cpu(), want[0]) and torch.equal(vd.cpu(), want[1]) and torch.equal(new.cpu(), want[2])
    cap = 90 if not page else -(-90 // page) * page
    assert int(over) == int(87 + 4 > cap)


def test_accept_in_place_lengths_bad_pages_and_strides():
    import probjax_b200 as pj

    _, kn, vn, k, v, _, lengths, table = make(3, 8, 2, 2, 64, 64, [10, 20, 64], torch.bfloat16, seed=31, page=16, garbage=0.0)
    table[1, 1] = 10 ** 8
    table[0, 0] = -1
    path = torch.tensor([[0, 1, 2]] * 3, dtype=torch.int32)
    counts = torch.tensor([3, 0, -4], dtype=torch.int32)
    want = accept_reference(kn, vn, k, v, path, counts, lengths, table)
    fused = torch.cat([kn, vn], 2).to(DEV)
    kd, vd, ln = k.to(DEV), v.to(DEV), lengths.to(DEV)
    out = pj.accept_drafts(fused[:, :, :2], fused[:, :, 2:], kd, vd, path.to(DEV), counts.to(DEV), kv_lengths=ln, block_table=table.to(DEV), out=ln)
    assert out is ln and torch.equal(ln.cpu(), want[2])
    assert torch.equal(kd.cpu(), want[0]) and torch.equal(vd.cpu(), want[1])


def test_speculative_loop_equals_token_by_token_decoding():
    """Drafts, verification and acceptance over a DecodeCache leave the cache that appending the accepted tokens one by one leaves, and
    the accepted drafts' attention is that of the plain decode steps."""
    import probjax_b200 as pj

    B, Hq, Hkv, D, cap = 3, 8, 2, 128, 512
    g = torch.Generator().manual_seed(40)
    t = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16).to(DEV)
    fast, slow = (pj.DecodeCache(B, cap, Hkv, D) for _ in range(2))
    k0, v0 = t(B, 200, Hkv, D), t(B, 200, Hkv, D)
    for c in (fast, slow):
        c.update(k0, v0)
        c.reset([200, 150, 0])
    parents = torch.tensor([-1, 0, 0, 1, 2, 3, 5, -1], dtype=torch.int32, device=DEV)
    paths = torch.tensor([[0, 1, 3, 5], [0, 2, 4, 4], [7, 7, 7, 7]], dtype=torch.int32, device=DEV)
    counts = torch.tensor([4, 3, 1], dtype=torch.int32, device=DEV)
    for step in range(3):
        q, k, v = t(B, 8, Hq, D), t(B, 8, Hkv, D), t(B, 8, Hkv, D)
        o = fast.attend_tree(q, k, v, parents)
        fast.accept(k, v, paths, counts)
        for i in range(4):
            rows = paths[:, i].long()
            pick = lambda x: x[torch.arange(B, device=DEV), rows][:, None]
            before = slow.cache_index.clone()
            slow.update(pick(k), pick(v))
            live = (counts > i)
            slow.cache_index.copy_(torch.where(live, slow.cache_index, before))
            got = slow.attend(pick(q))
            # two kernels of one formula: each within P's and the result's rounding of it, |v| below 5
            err = (got - pick(o)).float().abs()[live].max()
            assert float(err) <= 2 * (2 * 2.0 ** -8 * 5)
    assert torch.equal(fast.cache_index, slow.cache_index)
    for b, n in enumerate(fast.cache_index.tolist()):
        assert torch.equal(fast.cached_key[b, :n], slow.cached_key[b, :n]) and torch.equal(fast.cached_value[b, :n], slow.cached_value[b, :n])
    pj.check_status(DEV)
