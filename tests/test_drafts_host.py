"""Refusals and host logic of the drafted-tree, key-weight, eviction and multi-axis rotary calls; no GPU is touched: every call is refused,
or has nothing to do, before anything is launched."""

import ctypes

import pytest
import torch

BAD, UNSUPPORTED, WORKSPACE = 1, 2, 3
P = 0x1000  # a pointer that is never followed


@pytest.fixture(scope="module")
def L(built_lib):
    from probjax_b200 import _lib

    return _lib.lib()


def tree(L, **kw):
    a = dict(q=P, qb=0, qt=0, kn=P, kb=0, kt=0, vn=P, vb=0, vt=0, k=P, v=P, parents=P, pb=0, lengths=P, table=None, o=P, lse=None, B=1, N=4, Hq=4,
             Hkv=2, D=64, Dv=64, cap=128, page=0, max_pages=0, num_pages=0, dtype=1, scale=1.0, impl=0, ws=P, wsb=0, status=None, stream=None)
    a.update(kw)
    return L.pjx_attn_decode_tree(*a.values())


@pytest.mark.parametrize("kw,rc,word", [
    (dict(dtype=5), BAD, "dtype"), (dict(B=-1), BAD, "dimension"), (dict(D=0), BAD, "dimension"), (dict(cap=-1), BAD, "dimension"),
    (dict(Hq=5), BAD, "multiple"), (dict(impl=3), BAD, "impl"), (dict(qt=-1), BAD, "stride"), (dict(pb=-4), BAD, "stride"),
    (dict(table=P, page=24, max_pages=2, num_pages=2), BAD, "multiple of 16"), (dict(table=P, page=0, max_pages=2, num_pages=2), BAD, "multiple of 16"),
    (dict(table=P, page=64, max_pages=1 << 25, num_pages=2), BAD, "2^30"), (dict(table=P, page=64, max_pages=1, num_pages=-1), BAD, "2^30"),
    (dict(q=None), BAD, "null"), (dict(parents=None), BAD, "null"), (dict(lengths=None), BAD, "null"), (dict(v=None), BAD, "null"),
    (dict(N=257), UNSUPPORTED, "256"), (dict(cap=1 << 30), UNSUPPORTED, "2^30"), (dict(B=65536), UNSUPPORTED, "65535"), (dict(B=60000, cap=1 << 29), UNSUPPORTED, "2^31"),
    (dict(Hq=32768, Hkv=32768), UNSUPPORTED, "16384"),
    (dict(wsb=0), WORKSPACE, "workspace"), (dict(ws=P + 4, wsb=1 << 40), WORKSPACE, "16-byte"),
    (dict(B=0), 0, None), (dict(N=0), 0, None),
])
def test_tree_refusals(L, kw, rc, word):
    from probjax_b200 import _lib

    assert tree(L, **kw) == rc
    if word:
        assert word in _lib.last_error()


def test_tree_workspace_sizes(L):
    f = L.pjx_attn_decode_tree_workspace_bytes
    assert f(0, 4, 4, 2, 64, 128) == 0 and f(1, 257, 4, 2, 64, 128) == 0 and f(1, 4, 5, 2, 64, 128) == 0
    for args in ((16, 64, 32, 8, 128, 32768), (200, 7, 8, 2, 64, 1000), (1, 256, 64, 1, 128, 1 << 20), (128, 1, 1, 1, 64, 1)):
        B, N, Hq, Hkv, Dv, _ = args
        assert f(*args) >= B * N * Hq * (Dv + 1) * 4  # a segment per sequence at least


def accept(L, **kw):
    a = dict(k=0x100000, v=0x200000, kn=P, kb=0, kt=0, vn=P, vb=0, vt=0, lengths=P, path=P, counts=P, table=None, B=1, N=4, Pw=2, Hkv=2, D=64, Dv=64, cap=128, page=0,
             max_pages=0, num_pages=0, dtype=1, out=P, overflow=None, stream=None)
    a.update(kw)
    return L.pjx_kv_cache_accept(*a.values())


@pytest.mark.parametrize("kw,rc", [
    (dict(dtype=9), BAD), (dict(N=-1), BAD), (dict(kt=-8), BAD), (dict(table=P, page=0), BAD), (dict(table=P, page=64, max_pages=1 << 24), BAD),
    (dict(lengths=None), BAD), (dict(counts=None), BAD), (dict(out=None), BAD), (dict(path=None), BAD), (dict(v=None), BAD),
    (dict(B=65536), UNSUPPORTED), (dict(D=1, Hkv=1), UNSUPPORTED), (dict(kt=4), UNSUPPORTED), (dict(vb=3), UNSUPPORTED), (dict(kn=P + 8), UNSUPPORTED),
    (dict(B=0), 0), (dict(kn=0x40000, k=0x40000 - 64), BAD), (dict(vn=0x40000, k=0x40000 + 64, v=0x90000), BAD)])
def test_accept_refusals(L, kw, rc):
    assert accept(L, **kw) == rc


def weights(L, **kw):
    a = dict(q=P, k=P, v=P, lengths=None, win=None, wout=P, o=P, lse=None, B=1, Lq=1, Hq=4, Hkv=2, D=64, Dv=64, cap=128, dtype=1, scale=1.0, split=0, ws=P,
             wsb=1 << 40, status=None, stream=None)
    a.update(kw)
    return L.pjx_attn_decode_weights(*a.values())


@pytest.mark.parametrize("kw,rc", [
    (dict(dtype=3), BAD), (dict(Hq=3), BAD), (dict(wout=None), BAD), (dict(q=None), BAD), (dict(split=100), WORKSPACE), (dict(ws=None), WORKSPACE),
    (dict(wsb=16), WORKSPACE), (dict(ws=P + 8), WORKSPACE), (dict(cap=1 << 30), UNSUPPORTED), (dict(B=0), 0), (dict(Lq=0), 0)])
def test_decode_weights_refusals(L, kw, rc):
    if "split" in kw:  # (a split length that is no multiple of 64 has no workspace size)
        assert L.pjx_attn_decode_weights_workspace_bytes(1, 1, 4, 2, 64, 128, 100) == 128 // 64 * 64 * 2 * 2 * 4
        kw = dict(kw, wsb=0)
    assert weights(L, **kw) == rc


def key_weights(L, **kw):
    a = dict(q=P, k=P, lse=P, win=None, wout=P, lengths=None, B=1, Lq=1, Lkv=8, Hq=4, Hkv=2, D=64, dtype=1, lo=-(1 << 30), hi=1 << 30, scale=1.0, impl=0,
             status=None, stream=None)
    a.update(kw)
    return L.pjx_attn_key_weights(*a.values())


@pytest.mark.parametrize("kw,rc", [
    (dict(dtype=3), BAD), (dict(Hq=3), BAD), (dict(impl=7), BAD), (dict(k=None), BAD), (dict(lse=None), BAD), (dict(wout=None), BAD), (dict(Lq=1 << 30), BAD),
    (dict(B=65536), UNSUPPORTED), (dict(Lq=1 << 29, Hq=16, Hkv=1), UNSUPPORTED), (dict(D=257), UNSUPPORTED), (dict(impl=2, dtype=0), UNSUPPORTED),
    (dict(impl=2, D=96), UNSUPPORTED), (dict(B=0), 0), (dict(Lkv=0), 0)])
def test_key_weights_refusals(L, kw, rc):
    assert key_weights(L, **kw) == rc


def evict(L, **kw):
    a = dict(k=0x10000, v=0x90000, w=0x20000, lengths=P, ko=0x10000, vo=0x90000, wo=0x20000, lo=P, kept=P, B=1, Hkv=1, D=64, Dv=64, cap=128, cap_out=128,
             keep=32, recent=4, dtype=1, ws=P, wsb=64, stream=None)
    a.update(kw)
    return L.pjx_kv_cache_evict(*a.values())


@pytest.mark.parametrize("kw,rc,word", [
    (dict(dtype=3), BAD, "dtype"), (dict(D=0), BAD, "dimension"), (dict(keep=0), BAD, "keep"), (dict(recent=33), BAD, "recent"), (dict(recent=-1), BAD, "recent"),
    (dict(lengths=None), BAD, "null"), (dict(kept=None), BAD, "null"), (dict(wo=None), BAD, "null"),
    (dict(cap_out=31, ko=0x50000, vo=0x60000, wo=0x70000), BAD, "fit"),
    (dict(vo=0x60000), BAD, "together"), (dict(wo=0x60000), BAD, "together"), (dict(cap_out=64), BAD, "together"),
    (dict(ko=0x10000 + 128, vo=0xb0000, wo=0x70000, cap_out=32), BAD, "overlap"), (dict(ko=0x50000, vo=0x90000 - 64, wo=0x70000, cap_out=32), BAD, "overlap"),
    (dict(cap=1 << 30, cap_out=1 << 30), UNSUPPORTED, "2^30"), (dict(B=8192), UNSUPPORTED, "8191"),
    (dict(wsb=4), WORKSPACE, "workspace"), (dict(ws=P + 4), WORKSPACE, "workspace"), (dict(B=0), 0, None)])
def test_evict_refusals(L, kw, rc, word):
    from probjax_b200 import _lib

    assert evict(L, **kw) == rc
    if word:
        assert word in _lib.last_error()


def rope(L, widths, **kw):
    a = dict(x=P, xb=0, xt=0, y=P, pos=P, ptype=0, pb=0, axes=len(widths), sections=(ctypes.c_int32 * max(1, len(widths)))(*widths), B=1, T=4, H=2, D=64,
             shared=0, interleaved=1, inverse=0, base=10000.0, dtype=1, stream=None)
    a.update(kw)
    return L.pjx_rope_axes(*a.values())


@pytest.mark.parametrize("widths,kw,rc", [
    ((32, 32), dict(dtype=4), BAD), ((32, 32), dict(ptype=3), BAD), ((32, 32), dict(T=-1), BAD), ((), {}, BAD), ((2,) * 9, {}, BAD), ((32, 32), dict(sections=None), BAD),
    ((31,), {}, BAD), ((-2,), {}, BAD), ((66,), {}, BAD), ((32, 34), {}, BAD), ((32, 32), dict(base=0.0), BAD), ((32, 32), dict(base=float("nan")), BAD),
    ((32, 32), dict(xt=-1), BAD), ((32, 32), dict(y=None), BAD), ((32, 32), dict(pos=None), BAD), ((514,), dict(D=600), UNSUPPORTED),
    ((32, 32), dict(T=0), 0), ((32, 32), dict(B=0), 0)])
def test_rope_axes_refusals(L, widths, kw, rc):
    assert rope(L, widths, **kw) == rc


def test_python_calls_need_a_gpu():
    import probjax_b200 as pj

    if torch.cuda.is_available():
        pytest.skip("a GPU is here")
    z = torch.zeros(1, 2, 2, 64)
    for f in (lambda: pj.decode_tree(z, z, z, z, z, [0, 0], kv_lengths=[0]), lambda: pj.accept_drafts(z, z, z, z, [[0]], [1], kv_lengths=[0]),
              lambda: pj.decode_weights(z, z, z), lambda: pj.key_weights(z, z, z), lambda: pj.evict(z, z, z, [0], 1), lambda: pj.rope_axes(z, [[0]], (64,))):
        with pytest.raises(RuntimeError):
            f()


def test_strides_of_drafts():
    """A slice of a fused projection is taken in place; what the kernels cannot address is copied."""
    from probjax_b200.drafts import _int32, _token_rows

    fused = torch.zeros(2, 5, 12, 64, dtype=torch.bfloat16)
    t, bs, ts = _token_rows(fused[:, :, :8])
    assert t.data_ptr() == fused.data_ptr() and (bs, ts) == (5 * 12 * 64, 12 * 64)
    for odd in (fused.transpose(1, 2), fused[..., ::2], fused[..., 1:], fused[:, :, :, :60], fused[:1, :1, :1].expand(2, 5, 8, 64),
                fused[:, :, ::2]):
        t, bs, ts = _token_rows(odd)
        N, H, D = odd.shape[1:]
        assert t.is_contiguous() and (bs, ts) == (N * H * D, H * D) and torch.equal(t, odd)
    t, bs, ts = _token_rows(torch.zeros(1, 1, 3, 8).as_strided((1, 1, 3, 8), (7, 7, 8, 1)))  # (strides of single entries mean nothing)
    assert (bs, ts) == (24, 24)
    with pytest.raises(ValueError, match="integers"):
        _int32([1.5], "cpu", (1,), "counts")
    with pytest.raises(ValueError, match="must be"):
        _int32([1, 2], "cpu", (3,), "counts")
