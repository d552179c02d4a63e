"""Operators of a decode loop with drafted tokens and a bounded cache: their cases, inputs, plain forms and exact values.

A case is a dict of plain values; its ``op`` says which operator it runs:

* ``tree``     attention of a tree of drafted tokens over a KV cache, contiguous or paged (``decode_tree``): token ``i`` sees the
               cache and its ancestors among the drafts;
* ``accept``   the accepted path's keys and values go into the cache (``accept_drafts``);
* ``track``    a decode step that also adds up what every cached key received of attention (``decode_weights``);
* ``window``   the attention that the last queries of a prompt paid to every key (``key_weights``);
* ``evict``    the keys with the most accumulated attention, and the most recent ones, stay in the cache (``evict``);
* ``rope``     rotary positions with several axes (``rope_axes``), forward only or with the gradient.

``run`` computes them in plain torch operations in 32 bits, or, with ``own`` set, by the package's entry points.
"""

import math

import numpy as np
import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ------------------------------------------------------------------------------------------------ cases


def listed():
    return [
        # One user's chat: nine drafted tokens over a context of some 1500.  The smallest call: latency, launches, host work.
        dict(name="tree_chat", op="tree", B=1, N=9, Hq=32, Hkv=8, D=128, cap=4096, lo=1500, hi=1500, page=0, dtype="bf16"),
        # A serving batch over a paged cache with contexts of 1k to 32k tokens (the decode configuration of the benchmark), 64
        # drafts a sequence: the largest call, as much arithmetic as memory traffic.
        dict(name="tree_serving", op="tree", B=16, N=64, Hq=32, Hkv=8, D=128, cap=32768, lo=1024, hi=32768, page=128, dtype="bf16"),
        # Up to five of nine drafts accepted, one sequence.
        dict(name="accept_chat", op="accept", B=1, N=9, P=5, Hkv=8, D=128, cap=4096, lo=1500, hi=1500, page=0, dtype="bf16"),
        # Up to 16 of 64 drafts accepted in each sequence of a large paged batch, head width 64.
        dict(name="accept_serving", op="accept", B=64, N=64, P=16, Hkv=8, D=64, cap=4096, lo=1, hi=4000, page=64, dtype="f16"),
        # One user's decode step that keeps count of the keys' attention, at an odd length.
        dict(name="track_chat", op="track", B=1, Lq=1, Hq=16, Hkv=4, D=64, cap=4096, lo=1777, hi=1777, dtype="f16"),
        # The same for a serving batch of long, ragged contexts.
        dict(name="track_serving", op="track", B=16, Lq=1, Hq=32, Hkv=8, D=128, cap=32768, lo=1024, hi=32768, dtype="bf16"),
        # A few short prompts of unequal length, seventeen query tokens each, fp16.
        dict(name="window_short", op="window", B=3, Lq=17, Hq=16, Hkv=4, D=64, cap=777, lo=300, hi=777, dtype="f16"),
        # The last 64 queries of full 32k prompts decide what stays.
        dict(name="window_prompt", op="window", B=8, Lq=64, Hq=32, Hkv=8, D=128, cap=32768, lo=32768, hi=32768, dtype="bf16"),
        # One user's cache of 4000 tokens cut to 1024, 64 of them the most recent.
        dict(name="evict_chat", op="evict", B=1, Hkv=8, D=128, cap=4096, keep=1024, recent=64, lo=4001, hi=4001, dtype="bf16"),
        # Ragged prompts of up to 32k tokens cut to 8192; the short ones stay whole.
        dict(name="evict_serving", op="evict", B=16, Hkv=8, D=128, cap=32768, keep=8192, recent=257, lo=4096, hi=32768, dtype="bf16"),
        # Patches of an image, two axes, odd grid, fp32, halves layout.
        dict(name="rope_image", op="rope", B=2, T=1369, H=16, D=64, axes=2, shared=False, interleaved=False, fused=False,
             far=0, grad=False, dtype="f32"),
        # Training on video tokens behind a long text: time, height and width, queries out of a fused projection, with the gradient.
        dict(name="rope_video", op="rope", B=4, T=4096, H=32, D=128, axes=3, shared=True, interleaved=True, fused=True,
             far=200000, grad=True, dtype="bf16"),
    ]


_MOST = {  # the costs that no drawn case passes: those of the largest listed case of the operator
    "tree": "tree_serving", "accept": "accept_serving", "track": "track_serving", "window": "window_prompt",
    "evict": "evict_serving", "rope": "rope_video"}


def _size(rng, lo, hi):
    """A size spread over the logarithm of its range, odd about half of the time."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(lo, min(hi, n | 1 if rng.random() < 0.5 else n))


def _draw_once(rng):
    op = rng.choice(["tree", "tree", "tree", "accept", "track", "track", "window", "window", "evict", "evict", "rope", "rope"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    D = rng.choice([64, 128, 128])
    Hkv = rng.choice([1, 2, 4, 8])
    B = _size(rng, 1, 32)
    small = dtype == "f32"  # 32-bit caches are those of small models
    cap = _size(rng, 64, 2048 if small else 32768)
    lo = rng.choice([0, cap // 8, cap // 2, cap])
    page = rng.choice([0, 0, 16, 64, 256])
    if op == "tree":
        cap = -(-cap // page) * page if page else cap
        return dict(op=op, B=B, N=_size(rng, 1, 32 if small else 128), Hq=Hkv * rng.choice([1, 3, 4, 8]), Hkv=Hkv, D=D, cap=cap, lo=lo, hi=cap,
                    page=page, dtype=dtype)
    if op == "accept":
        cap = max(cap, 256)
        cap = -(-cap // page) * page if page else cap
        N = _size(rng, 1, 64)
        return dict(op=op, B=_size(rng, 1, 64), N=N, P=rng.randint(1, min(N, 16)), Hkv=Hkv, D=D, cap=min(cap, 4096), lo=1, hi=min(cap, 4096) - 16,
                    page=page, dtype=dtype)
    if op == "track":
        G, Lq = rng.choice([(1, 1), (4, 1), (8, 1), (4, 2), (4, 4), (3, 1)])
        return dict(op=op, B=B, Lq=Lq, Hq=Hkv * G, Hkv=Hkv, D=D, cap=cap, lo=lo, hi=cap, dtype=dtype)
    if op == "window":
        Lq = _size(rng, 1, 64)
        return dict(op=op, B=min(B, 8), Lq=Lq, Hq=Hkv * rng.choice([1, 3, 4, 8]), Hkv=Hkv, D=D, cap=max(cap, Lq), lo=max(lo, Lq), hi=max(cap, Lq),
                    dtype=dtype)
    if op == "evict":
        keep = _size(rng, 8, max(9, cap // 2))
        return dict(op=op, B=B, Hkv=Hkv, D=D, cap=cap, keep=keep, recent=rng.choice([0, 1, keep // 4, keep]), lo=lo, hi=cap, dtype=dtype)
    return dict(op=op, B=_size(rng, 1, 8), T=_size(rng, 1, 8192), H=rng.choice([1, 3, 8, 16, 32]), D=rng.choice([64, 80, 128]), axes=rng.choice([1, 2, 3]),
                shared=rng.random() < 0.5, interleaved=rng.random() < 0.5, fused=rng.random() < 0.5,
                far=rng.choice([0, 0, 131071, 1000000]), grad=rng.random() < 0.5, dtype=dtype)


def draw(rng):
    most = {c["name"]: work(c) for c in listed()}
    while True:
        case = _draw_once(rng)
        w, m = work(case), most[_MOST[case["op"]]]
        if w["bytes"] <= m["bytes"] and w["flops"] <= m["flops"]:
            return case


# ------------------------------------------------------------------------------------------------ what a pass cannot do without


def _lengths(case):
    """Valid tokens of every sequence: spread evenly from ``lo`` to ``hi``, the longest one first."""
    B, lo, hi = case["B"], case["lo"], case["hi"]
    return [hi - (hi - lo) * b // max(B - 1, 1) for b in range(B)]


def _kept(case):
    return [min(n, case["keep"]) for n in _lengths(case)]


def work(case):
    es = 4 if case["dtype"] == "f32" else 2
    op, B = case["op"], case["B"]
    if op == "rope":
        n = B * case["T"] * case["H"] * case["D"]
        passes = 2 if case["grad"] else 1
        return {"bytes": passes * (2 * n * es + B * case["T"] * case["axes"] * 4), "flops": passes * 3 * n}
    Hkv, D = case["Hkv"], case["D"]
    total = sum(_lengths(case))
    if op == "tree":
        N, Hq = case["N"], case["Hq"]
        keys = total + B * N
        return {"bytes": 2 * Hkv * D * es * keys + 2 * B * N * Hq * D * es + 4 * B * N, "flops": 4 * N * Hq * D * (total + B * (N + 1) // 2)}
    if op == "accept":
        rows = sum(_counts(case))
        return {"bytes": 4 * rows * Hkv * D * es + 4 * B * (case["P"] + 3), "flops": 0}
    if op == "track":
        rows = B * case["Lq"] * case["Hq"]
        return {"bytes": 2 * Hkv * D * es * total + 2 * rows * D * es + 8 * B * Hkv * case["cap"], "flops": 4 * case["Lq"] * case["Hq"] * D * total}
    if op == "window":
        rows = B * case["Lq"] * case["Hq"]
        return {"bytes": Hkv * D * es * total + rows * (D * es + 4) + 4 * B * Hkv * case["cap"], "flops": 2 * case["Lq"] * case["Hq"] * D * total}
    kept = sum(_kept(case))
    return {"bytes": 4 * Hkv * total + Hkv * kept * (4 * D * es + 4 + 4), "flops": 0}


# ------------------------------------------------------------------------------------------------ inputs


def _counts(case):
    """Accepted drafts of every sequence, 0 to ``P``, the first one ``P``."""
    return [(case["P"] * (b + 1) + b // 3) % (case["P"] + 1) if b else case["P"] for b in range(case["B"])]


def _parents(case, rng):
    """Trees in topological order: a draft hangs on the context (-1) or on one of the eight drafts before it.  All sequences of a
    batch but the first carry fewer drafts, and the rest of their row is absent (-2)."""
    B, N = case["B"], case["N"]
    p = np.full((B, N), -2, dtype=np.int32)
    for b in range(B):
        n = N if b == 0 else int(rng.integers(max(1, N // 2), N + 1))
        i = np.arange(n)
        back = np.minimum(rng.integers(1, 9, n), i + 1)
        p[b, :n] = np.where(rng.random(n) < 0.15, -1, i - back)
    return p


def _paths(case, rng):
    """An increasing list of draft indices for every sequence; entries past its count are not looked at."""
    B, N, P = case["B"], case["N"], case["P"]
    return np.stack([np.sort(rng.choice(N, P, replace=False)) for _ in range(B)]).astype(np.int32)


def _sections(case):
    """Elements of a head vector that every axis rotates: all for one axis, a quarter each for two (half of the vector stays as it
    is), a quarter for time and three eighths each for height and width."""
    D = case["D"]
    return {1: (D,), 2: (D // 4, D // 4), 3: (D // 4, 3 * D // 8, 3 * D // 8)}[case["axes"]]


def _positions(case):
    """Positions of a grid of tokens: (row, column), or (time, row, column), behind ``far`` tokens of text."""
    T, axes = case["T"], case["axes"]
    i = torch.arange(T)
    side = max(1, math.isqrt(T) if axes == 2 else round(T ** (1 / 3)))
    if axes == 1:
        p = i[:, None]
    elif axes == 2:
        p = torch.stack([i // side, i % side], 1)
    else:
        p = torch.stack([i // (side * side), i // side % side, i % side], 1)
    return (p + case["far"])[None] + 3 * torch.arange(case["B"])[:, None, None]


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(seed)
    rng = np.random.default_rng(seed)
    dt = _DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=g, device=dev, dtype=dt)

    def ints(a):
        return torch.as_tensor(np.asarray(a, dtype=np.int32)).to(dev)

    op, B = case["op"], case["B"]
    s = dict(case=case)
    if op == "rope":
        T, H, D = case["T"], case["H"], case["D"]
        if case["fused"]:  # the queries' part of a projection that also holds keys and values
            s["x"] = normal(B, T, H + 2, D)[:, :, :H]
        else:
            s["x"] = normal(B, T, H, D)
        s["positions"] = _positions(case).to(dev, torch.int32)
        s["sections"] = _sections(case)
        if case["grad"]:
            s["x"].requires_grad_(True)
            s["dy"] = normal(B, T, H, D)
        return s
    Hkv, D, cap = case["Hkv"], case["D"], case["cap"]
    s["lengths"] = ints(_lengths(case))
    page = case.get("page", 0)
    if op != "window":
        shape = (B * cap // page, page, Hkv, D) if page else (B, cap, Hkv, D)
        s["k"], s["v"] = normal(*shape), normal(*shape)
        s["table"] = ints(rng.permutation(B * cap // page).reshape(B, cap // page)) if page else None
    if op in ("tree", "accept"):
        N = case["N"]
        s["k_new"], s["v_new"] = normal(B, N, Hkv, D), normal(B, N, Hkv, D)
        if op == "tree":
            s["q"] = normal(B, N, case["Hq"], D)
            s["parents"] = ints(_parents(case, rng))
        else:
            s["path"], s["counts"] = ints(_paths(case, rng)), ints(_counts(case))
    elif op in ("track", "window"):
        s["q"] = normal(B, case["Lq"], case["Hq"], D)
        valid = torch.arange(cap, device=dev) < s["lengths"][:, None]
        if op == "track":  # what earlier steps left: some keys with much, most with little
            s["weights"] = torch.randn((B, Hkv, cap), generator=g, device=dev).mul_(2).exp_().mul_(valid[:, None])
        else:
            s["k"] = normal(B, cap, Hkv, D)
            s["lse"] = _window_lse(s)
    else:
        w = torch.randn((B, Hkv, cap), generator=g, device=dev).mul_(2).exp_()
        w = w * (torch.rand((B, Hkv, cap), generator=g, device=dev) > 0.05)  # some keys that no query looked at: ties
        s["weights"] = w * (torch.arange(cap, device=dev) < s["lengths"][:, None])[:, None]
        s["k_out"], s["v_out"] = (torch.zeros((B, case["keep"], Hkv, D), device=dev, dtype=dt) for _ in range(2))
        s["w_out"] = torch.zeros((B, Hkv, case["keep"]), device=dev)
    if own:
        import probjax_b200  # noqa: F401  (loaded before the first call)
    return s


# ------------------------------------------------------------------------------------------------ helpers of both forms


def _by_sequence(pool, table):
    """A paged cache as a contiguous one."""
    if table is None:
        return pool
    t = pool[table.long()]
    return t.reshape(t.shape[0], -1, *t.shape[3:])


def _ancestors(parents):
    """bool [B, N, N]: draft j is i or an ancestor of i; all false where i, or one of its ancestors, is absent."""
    B, N = parents.shape
    p = parents.long()
    j = torch.arange(N, device=p.device)
    up = ((p[..., None] == j) | (j[:, None] == j)).float()  # itself and its parent, then twice as far up each time
    for _ in range(max(N - 1, 0).bit_length()):
        up = (up @ up > 0).float()
    sees = up > 0
    return sees & ~(sees & (p < -1)[:, None]).any(-1, keepdim=True)


def _window_visible(case, lengths, cap):
    """bool [B, Lq, cap]: query t of the last Lq tokens sees the keys up to its own."""
    t = torch.arange(case["Lq"], device=lengths.device)
    j = torch.arange(cap, device=lengths.device)
    same = case["lo"] == case["hi"]
    if same:  # prompts of one length: the bottom-right causal mask
        return (j <= (case["hi"] - case["Lq"] + t)[:, None])[None].expand(case["B"], -1, -1)
    return (j < lengths[:, None, None]).expand(-1, case["Lq"], -1)  # ragged prompts: every valid key


def _window_lse(s):
    """Natural log-sum-exp of the window's scores, [B, Hq, Lq] in 32 bits: what the attention call before left."""
    case, q, k = s["case"], s["q"], s["k"]
    B, Lq, Hq, D = q.shape
    Hkv = k.shape[2]
    see = _window_visible(case, s["lengths"], k.shape[1])
    out = torch.empty((B, Hq, Lq), device=q.device)
    for b in range(B):
        qq = q[b].float().reshape(Lq, Hkv, Hq // Hkv, D).permute(1, 2, 0, 3)
        sc = qq @ k[b].float().permute(1, 2, 0)[:, None] / math.sqrt(D)
        out[b] = torch.logsumexp(sc.masked_fill(~see[b], -math.inf), -1).reshape(Hq, Lq)
    return out


def _softmax_parts(sc, see):
    """Probabilities over the visible keys, zero rows where there are none."""
    sc = sc.masked_fill(~see, -math.inf)
    top = sc.amax(-1, keepdim=True)
    e = torch.exp(sc - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total > 0, total, torch.ones_like(total))


# ------------------------------------------------------------------------------------------------ plain forms


def _tree_plain(s):
    case, q = s["case"], s["q"]
    B, N, Hq, D = q.shape
    k = torch.cat([_by_sequence(s["k"], s["table"]), s["k_new"]], 1).float()
    v = torch.cat([_by_sequence(s["v"], s["table"]), s["v_new"]], 1).float()
    cap, Hkv = case["cap"], case["Hkv"]
    tree = _ancestors(s["parents"])
    there = tree.any(-1)
    prefix = (torch.arange(cap, device=q.device) < s["lengths"][:, None])[:, None] & there[:, :, None]
    see = torch.cat([prefix, tree], 2)[:, None, None]                                       # [B, 1, 1, N, cap + N]
    qq = q.float().reshape(B, N, Hkv, Hq // Hkv, D).permute(0, 2, 3, 1, 4)                  # [B, Hkv, G, N, D]
    sc = (qq.reshape(B, Hkv, -1, D) @ k.permute(0, 2, 3, 1)).reshape(*qq.shape[:4], -1) / math.sqrt(D)
    p = _softmax_parts(sc, see)
    o = p.reshape(B, Hkv, -1, cap + N) @ v.permute(0, 2, 1, 3)
    return o.reshape(B, Hkv, Hq // Hkv, N, D).permute(0, 3, 1, 2, 4).reshape(B, N, Hq, D).to(q.dtype)


def _accept_plain(s):
    k, v, path, cap = s["k"], s["v"], s["path"].long(), s["case"]["cap"]
    B, P = path.shape
    i = torch.arange(P, device=k.device)
    rows = s["lengths"].long()[:, None] + i
    ok = (i < s["counts"][:, None]) & (rows < cap)
    b = torch.arange(B, device=k.device)[:, None].expand(B, P)
    for cache, new in ((k, s["k_new"]), (v, s["v_new"])):
        values = new[b, path]
        if s["table"] is None:
            cache[b[ok], rows[ok]] = values[ok]
        else:
            page = cache.shape[1]
            at = rows.clamp(max=cap - 1)
            pages = torch.gather(s["table"].long(), 1, at // page)
            cache[pages[ok], (at % page)[ok]] = values[ok]
    return dict(k=k, v=v, lengths=torch.clamp(s["lengths"] + s["counts"], max=cap))


def _track_plain(s):
    q, k, v = s["q"], s["k"], s["v"]
    B, Lq, Hq, D = q.shape
    Hkv = k.shape[2]
    see = (torch.arange(k.shape[1], device=q.device) < s["lengths"][:, None])[:, None, None]
    qq = q.float().reshape(B, Lq, Hkv, Hq // Hkv, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, D)
    p = _softmax_parts(qq @ k.float().permute(0, 2, 3, 1) / math.sqrt(D), see)
    o = (p @ v.float().permute(0, 2, 1, 3)).reshape(B, Hkv, Hq // Hkv, Lq, D).permute(0, 3, 1, 2, 4).reshape(B, Lq, Hq, D)
    return dict(o=o.to(q.dtype), weights=s["weights"] + p.sum(2))


def _window_plain(s):
    q, k = s["q"], s["k"]
    B, Lq, Hq, D = q.shape
    Hkv = k.shape[2]
    see = _window_visible(s["case"], s["lengths"], k.shape[1])[:, None, None]
    qq = q.float().reshape(B, Lq, Hkv, Hq // Hkv, D).permute(0, 2, 3, 1, 4)
    sc = (qq.reshape(B, Hkv, -1, D) @ k.float().permute(0, 2, 3, 1)).reshape(*qq.shape[:4], -1) / math.sqrt(D)
    p = torch.exp(sc - s["lse"].reshape(B, Hkv, Hq // Hkv, Lq, 1))
    return torch.where(see, p, torch.zeros_like(p)).sum((2, 3))


def _evict_plain(s):
    case, w, lengths = s["case"], s["weights"], s["lengths"].long()
    keep, recent = case["keep"], min(case["recent"], case["keep"])
    B, Hkv, cap = w.shape
    j = torch.arange(cap, device=w.device)
    n = lengths[:, None, None]
    rank = torch.where(j >= n, -math.inf, torch.where(j >= n - recent, math.inf, w))        # invalid last, the recent ones first
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices                  # (ties: the lowest index first)
    width = min(keep, cap)
    new = torch.clamp(lengths, max=keep)
    held = torch.arange(width, device=w.device) < new[:, None, None]
    kept = torch.sort(torch.where(held, order[..., :width], cap), dim=-1).values            # ascending, the missing ones last
    at = kept.clamp(max=cap - 1)
    for src, dst in ((s["k"], s["k_out"]), (s["v"], s["v_out"])):
        rows = torch.gather(src.permute(0, 2, 1, 3), 2, at[..., None].expand(-1, -1, -1, src.shape[3]))
        now = dst[:, :width].permute(0, 2, 1, 3)
        dst[:, :width] = torch.where(held[..., None], rows, now).permute(0, 2, 1, 3)
    s["w_out"][..., :width] = torch.where(held, torch.gather(w, 2, at), 0.0)
    index = torch.full((B, Hkv, keep), -1, dtype=torch.int32, device=w.device)
    index[..., :width] = torch.where(held, kept, -1).to(torch.int32)
    return dict(lengths=new.to(torch.int32), kept=index, k=s["k_out"], v=s["v_out"], weights=s["w_out"])


def _angles(case, positions, sections):
    """float64 [B, T, pairs]: the angle of every rotated pair."""
    parts, total = [], sum(sections)
    done = 0
    for a, width in enumerate(sections):
        i = torch.arange(width // 2, device=positions.device, dtype=torch.float64)
        e = (i + done // 2) * 2 / total if case["shared"] else i * 2 / max(width, 1)
        parts.append(positions[..., a, None].double() * 10000.0 ** -e)
        done += width
    return torch.cat(parts, -1)


def _rotate(case, x, angles, sign, dtype):
    """The rotation of x [B, T, H, D] by ``sign`` times the angles, computed in ``dtype``."""
    pairs = angles.shape[-1]
    c, n = torch.cos(angles).to(dtype)[:, :, None], (sign * torch.sin(angles)).to(dtype)[:, :, None]
    head, rest = x[..., :2 * pairs].to(dtype), x[..., 2 * pairs:].to(dtype)
    if case["interleaved"]:
        a, b = head[..., 0::2], head[..., 1::2]
        y = torch.stack([a * c - b * n, b * c + a * n], -1).flatten(-2)
    else:
        a, b = head[..., :pairs], head[..., pairs:]
        y = torch.cat([a * c - b * n, b * c + a * n], -1)
    return torch.cat([y, rest], -1)


def _rope_plain(s):
    case = s["case"]
    angles = _angles(case, s["positions"], s["sections"])
    x = s["x"].detach()
    y = _rotate(case, x, angles, 1, torch.float32).to(x.dtype)
    if not case["grad"]:
        return y
    return dict(y=y, dx=_rotate(case, s["dy"], angles, -1, torch.float32).to(x.dtype))


_PLAIN = {"tree": _tree_plain, "accept": _accept_plain, "track": _track_plain, "window": _window_plain, "evict": _evict_plain, "rope": _rope_plain}


# ------------------------------------------------------------------------------------------------ the package's calls


def _run_own(s):
    import probjax_b200 as pj

    case, op = s["case"], s["case"]["op"]
    if op == "tree":
        return pj.decode_tree(s["q"], s["k_new"], s["v_new"], s["k"], s["v"], s["parents"], kv_lengths=s["lengths"], block_table=s["table"])
    if op == "accept":
        lengths = pj.accept_drafts(s["k_new"], s["v_new"], s["k"], s["v"], s["path"], s["counts"], kv_lengths=s["lengths"],
                                   block_table=s["table"])
        return dict(k=s["k"], v=s["v"], lengths=lengths)
    if op == "track":
        o, weights = pj.decode_weights(s["q"], s["k"], s["v"], s["weights"], kv_lengths=s["lengths"])
        return dict(o=o, weights=weights)
    if op == "window":
        if case["lo"] == case["hi"]:
            mask = pj.KVLenMask(s["lengths"]) & pj.CausalFromBottomRightMask(case["Lq"], case["hi"])
        else:
            mask = pj.KVLenMask(s["lengths"])
        return pj.key_weights(s["q"], s["k"], s["lse"], mask=mask)
    if op == "evict":
        lengths, kept = pj.evict(s["k"], s["v"], s["weights"], s["lengths"], case["keep"], recent=case["recent"],
                                 out=(s["k_out"], s["v_out"], s["w_out"]))
        return dict(lengths=lengths, kept=kept, k=s["k_out"], v=s["v_out"], weights=s["w_out"])
    y = pj.rope_axes(s["x"], s["positions"], s["sections"], shared=case["shared"], interleaved=case["interleaved"])
    if not case["grad"]:
        return y
    (dx,) = torch.autograd.grad(y, s["x"], s["dy"])
    return dict(y=y.detach(), dx=dx)


def run(state):
    return _run_own(state) if own else _PLAIN[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------------------ exact values


def _attend64(q, k, v, see):
    """One head in 64 bits: (output, probabilities) of q [N, D] over the keys that ``see`` [N, L] leaves it."""
    sc = q.double() @ k.double().T / math.sqrt(q.shape[-1])
    sc = torch.where(see, sc, torch.full_like(sc, -math.inf))
    p = torch.nan_to_num(torch.softmax(sc, -1), nan=0.0)  # (a row without keys)
    return p @ v.double(), p


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    lengths = _lengths(case) if op != "rope" else None
    if op == "tree":
        q, par = s["q"], s["parents"].cpu().tolist()
        B, N, Hq, D = q.shape
        G = Hq // case["Hkv"]
        out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
        for b in range(B):
            see = torch.zeros((N, lengths[b] + N), dtype=torch.bool)
            for i in range(N):
                chain, j = [], i
                while j >= 0:
                    chain.append(j)
                    j = par[b][j]
                if j == -1:
                    see[i, :lengths[b]] = True
                    see[i, [lengths[b] + c for c in chain]] = True
            see = see.to(q.device)
            rows = s["k"][b] if s["table"] is None else s["k"][s["table"][b].long()].flatten(0, 1)
            vals = s["v"][b] if s["table"] is None else s["v"][s["table"][b].long()].flatten(0, 1)
            for h in range(Hq):
                k = torch.cat([rows[:lengths[b], h // G], s["k_new"][b, :, h // G]])
                v = torch.cat([vals[:lengths[b], h // G], s["v_new"][b, :, h // G]])
                out[b, :, h] = _attend64(q[b, :, h], k, v, see)[0]
        return out
    if op == "accept":
        k, v, path, counts = s["k"].clone(), s["v"].clone(), s["path"].cpu().tolist(), s["counts"].cpu().tolist()
        table = None if s["table"] is None else s["table"].cpu().tolist()
        new = []
        for b in range(case["B"]):
            for i in range(counts[b]):
                row = lengths[b] + i
                if row < case["cap"]:
                    at = (b, row) if table is None else (table[b][row // case["page"]], row % case["page"])
                    k[at], v[at] = s["k_new"][b, path[b][i]], s["v_new"][b, path[b][i]]
            new.append(min(lengths[b] + counts[b], case["cap"]))
        return dict(k=k, v=v, lengths=torch.tensor(new, dtype=torch.int32, device=k.device))
    if op in ("track", "window"):
        q, k = s["q"], s["k"]
        B, Lq, Hq, D = q.shape
        G = Hq // case["Hkv"]
        weights = torch.zeros((B, case["Hkv"], case["cap"]), dtype=torch.float64, device=q.device)
        if op == "window":
            see = _window_visible(case, s["lengths"], case["cap"])
            for b in range(B):
                for h in range(Hq):
                    sc = q[b, :, h].double() @ k[b, :, h // G].double().T / math.sqrt(D)
                    p = torch.exp(sc - s["lse"][b, h].double()[:, None])
                    weights[b, h // G] += torch.where(see[b], p, torch.zeros_like(p)).sum(0)
            return weights
        out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
        for b in range(B):
            n = lengths[b]
            for h in range(Hq):
                see = torch.ones((Lq, n), dtype=torch.bool, device=q.device)
                out[b, :, h], p = _attend64(q[b, :, h], k[b, :n, h // G], s["v"][b, :n, h // G], see)
                weights[b, h // G, :n] += p.sum(0)
        return dict(o=out, weights=s["weights"].double() + weights)
    if op == "evict":
        keep, recent = case["keep"], min(case["recent"], case["keep"])
        k, v, w = s["k_out"].clone(), s["v_out"].clone(), torch.zeros_like(s["w_out"])
        kept = torch.full((case["B"], case["Hkv"], keep), -1, dtype=torch.int32, device=w.device)
        for b, n in enumerate(lengths):
            for h in range(case["Hkv"]):
                if n <= keep:
                    index = torch.arange(n, device=w.device)
                else:
                    old = s["weights"][b, h, :n - recent].double()
                    top = torch.sort(old, descending=True, stable=True).indices[:keep - recent]
                    index = torch.cat([torch.sort(top).values, torch.arange(n - recent, n, device=w.device)])
                m = len(index)
                kept[b, h, :m] = index.to(torch.int32)
                k[b, :m, h], v[b, :m, h], w[b, h, :m] = s["k"][b, index, h], s["v"][b, index, h], s["weights"][b, h, index]
        new = torch.tensor([min(n, keep) for n in lengths], dtype=torch.int32, device=w.device)
        return dict(lengths=new, kept=kept, k=k, v=v, weights=w)
    # rope: pair after pair, as complex numbers
    x, widths = s["x"].detach(), s["sections"]
    total, done = sum(widths), 0
    pairs = [(a, (done_a + i) * 2 / total if case["shared"] else 2 * i / width)
             for a, (width, done_a) in enumerate(zip(widths, [sum(widths[:a]) // 2 for a in range(len(widths))])) for i in range(width // 2)]
    turn = torch.stack([s["positions"][..., a].double() * 10000.0 ** -e for a, e in pairs], -1)
    turn = torch.polar(torch.ones_like(turn), turn)[:, :, None]

    def turned(t, factor):
        t = t.double()
        n = len(pairs)
        first = t[..., 0:2 * n:2] if case["interleaved"] else t[..., :n]
        second = t[..., 1:2 * n:2] if case["interleaved"] else t[..., n:2 * n]
        z = torch.complex(first, second) * factor
        y = t.clone()
        if case["interleaved"]:
            y[..., 0:2 * n:2], y[..., 1:2 * n:2] = z.real, z.imag
        else:
            y[..., :n], y[..., n:2 * n] = z.real, z.imag
        return y

    y = turned(x, turn)
    return dict(y=y, dx=turned(s["dy"], turn.conj())) if case["grad"] else y
