"""64-bit references on the CPU of the drafted-tree, key-weight, eviction and multi-axis rotary operators, with error bounds."""

import math

import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def ancestors(parents):
    """Per draft the list of itself and its ancestors, ``None`` where it is absent."""
    out = []
    for i, p in enumerate(parents):
        if p == -1:
            out.append([i])
        elif 0 <= p < i and out[p] is not None:
            out.append([i] + out[p])
        else:
            out.append(None)
    return out


def pages_to_rows(pool, table, b, n):
    """The first ``n`` cached rows of sequence ``b`` of a page pool (or of a contiguous cache)."""
    if table is None:
        return pool[b, :n]
    page = pool.shape[1]
    return torch.stack([pool[int(table[b, j // page]), j % page] for j in range(n)]) if n else pool[:0, 0]


def attention_row(q, k, v, scale):
    """One row ``q [D]`` over ``k [L, D]``, ``v [L, Dv]`` in 64 bits: output, natural lse, probabilities, and per output element the bound of
    the error of a kernel that forms the scores and sums in 32 bits, in units that the caller scales: ``sum p |v|`` times

    * ``2 dS``, dS the error of a score: D products summed in 32 bits, each step at most 2^-23 of the sum of magnitudes (tensor cores may
      cut instead of rounding), twice because numerator and denominator move;
    * ``2^-20 + 2^-22 max|s|``: exp2 to 2^-22, its argument rounded at the size of the scores in the exp2 domain;
    * ``(L + 64) 2^-23``: the two sums over the keys and the joining of parts."""
    q, k, v = q.double(), k.double(), v.double()
    if k.shape[0] == 0:
        return torch.zeros(v.shape[1], dtype=torch.float64), math.inf, torch.zeros(0, dtype=torch.float64), torch.zeros(v.shape[1], dtype=torch.float64), 0.0
    s = k @ q * scale
    lse = float(torch.logsumexp(s, 0))
    p = torch.exp(s - lse)
    mag = float((k.abs() @ q.abs()).max()) * scale
    rel = 2 * q.shape[0] * 2.0 ** -23 * mag + 2.0 ** -20 + 2.0 ** -22 * float(s.abs().max()) + (k.shape[0] + 64) * 2.0 ** -23
    return p @ v, lse, p, (p @ v.abs()) * rel, rel


def tree_reference(q, k_new, v_new, k_cache, v_cache, parents, lengths, table=None, scale=None):
    """``(o, lse, tol_o, tol_lse)`` in 64 bits; the tolerances are the bound of ``attention_row`` plus the roundings to the
    inputs' type: P (relative to the sum of p |v|) and the result."""
    B, N, Hq, D = q.shape
    Hkv, Dv = k_new.shape[2], v_new.shape[3]
    scale = 1 / math.sqrt(D) if scale is None else scale
    u = HALF_STEP[q.dtype]
    o = torch.zeros((B, N, Hq, Dv), dtype=torch.float64)
    lse = torch.full((B, Hq, N), math.inf, dtype=torch.float64)
    tol, tol_l = torch.zeros_like(o), torch.zeros_like(lse)
    for b in range(B):
        par = parents if parents.dim() == 1 else parents[b]
        chains = ancestors(par.tolist())
        n = max(0, int(lengths[b]))
        kp, vp = pages_to_rows(k_cache, table, b, n), pages_to_rows(v_cache, table, b, n)
        for i, chain in enumerate(chains):
            if chain is None:
                continue
            for h in range(Hq):
                g = h // (Hq // Hkv)
                k = torch.cat([kp[:, g], k_new[b, chain, g]])
                v = torch.cat([vp[:, g], v_new[b, chain, g]])
                r, l, p, t, rel = attention_row(q[b, i, h], k, v, scale)
                o[b, i, h], lse[b, h, i] = r, l
                tol[b, i, h] = t + u * (p @ v.double().abs() + r.abs())
                tol_l[b, h, i] = rel + 2.0 ** -23 * abs(l) + 2.0 ** -20
    return o, lse, tol, tol_l


def key_weights_reference(q, k, lse, lengths=None, lo=None, hi=None, scale=None):
    """``(sum of exp(scale q.k - lse), tolerance)`` ``[B, Hkv, Lkv]`` in 64 bits from the given (32-bit) lse."""
    B, Lq, Hq, D = q.shape
    Lkv, Hkv = k.shape[1], k.shape[2]
    scale = 1 / math.sqrt(D) if scale is None else scale
    w = torch.zeros((B, Hkv, Lkv), dtype=torch.float64)
    tol = torch.zeros_like(w)
    t, j = torch.arange(Lq)[:, None], torch.arange(Lkv)[None]
    for b in range(B):
        keep = torch.ones((Lq, Lkv), dtype=torch.bool)
        if lo is not None:
            keep &= j >= t + lo
        if hi is not None:
            keep &= j <= t + hi
        if lengths is not None:
            keep &= j < int(lengths[b])
        for h in range(Hq):
            g = h // (Hq // Hkv)
            kk = torch.nan_to_num(k[b, :, g].double(), nan=0.0, posinf=0.0, neginf=0.0)
            s = q[b, :, h].double() @ kk.T * scale
            mag = q[b, :, h].double().abs() @ kk.abs().T * scale
            l = lse[b, h].double()[:, None]
            on = keep & torch.isfinite(l)
            p = torch.where(on, torch.exp(s - torch.where(torch.isfinite(l), l, torch.zeros_like(l))), torch.zeros_like(s))
            rel = D * 2.0 ** -23 * mag + 2.0 ** -20 + 2.0 ** -22 * (s.abs() + torch.nan_to_num(l, posinf=0.0).abs()) + (Hq // Hkv * Lq) * 2.0 ** -23
            w[b, g] += p.sum(0)
            tol[b, g] += (p * rel).sum(0)
    return w, tol + 2.0 ** -23 * w


def evict_reference(k, v, w, lengths, keep, recent):
    """Lists of kept indices per (sequence, head), by sorting in Python."""
    B, cap, Hkv, _ = k.shape
    kept = []
    for b in range(B):
        n = min(cap, max(0, int(lengths[b])))
        rows = []
        for h in range(Hkv):
            if n <= keep:
                rows.append(list(range(n)))
                continue
            score = [(-math.inf if math.isnan(x) else x) for x in w[b, h, :n - recent].tolist()]
            # (NaN ranks behind -inf: a second key)
            nan = [math.isnan(x) for x in w[b, h, :n - recent].tolist()]
            order = sorted(range(n - recent), key=lambda j: (nan[j], -score[j], j))
            rows.append(sorted(order[:keep - recent]) + list(range(n - recent, n)))
        kept.append(rows)
    return kept


def rope_reference(x, positions, sections, base=10000.0, shared=False, interleaved=True, sign=1):
    """``(y, tolerance)`` in 64 bits for ``x [B, T, H, D]`` and ``positions [B, T, axes]``: the sine and cosine of a kernel are off by at
    most 2^-22 (argument and function), each product and the sum by half a step of 32 bits, the result by half a step of its type."""
    total = sum(sections)
    y = x.double().clone()
    tol = torch.zeros_like(y)
    p = 0
    for a, width in enumerate(sections):
        for i in range(width // 2):
            e = 2 * p / total if shared else 2 * i / width
            ang = positions[..., a].double() * base ** -e
            c, s = torch.cos(ang)[..., None], sign * torch.sin(ang)[..., None]
            ia, ib = (2 * p, 2 * p + 1) if interleaved else (p, total // 2 + p)
            u, w = x[..., ia].double(), x[..., ib].double()
            y[..., ia], y[..., ib] = u * c - w * s, w * c + u * s
            for at in (ia, ib):
                tol[..., at] = (u.abs() + w.abs()) * (2.0 ** -22 + 2 * 2.0 ** -23) + HALF_STEP[x.dtype] * y[..., at].abs()
            p += 1
    return y, tol
