"""Host side of the decode loop's calls; no GPU is touched."""

import threading

import pytest
import torch

BAD = 1
P = 0x1000  # a pointer that is never followed


@pytest.fixture(scope="module")
def L(built_lib):
    from probjax_b200 import _lib

    return _lib.lib()


def test_threads_do_not_share_a_workspace(monkeypatch):
    """Calls of two launches hand over through a cached workspace: it is the thread's own, also on a shared stream."""
    from probjax_b200 import attention as A

    monkeypatch.setattr(A, "_stream", lambda device: 0)
    cpu, got = torch.device("cpu"), {}

    def take(name):
        got[name] = [A._scratch_bytes(cpu, "evict", 512), A._scratch_bytes(cpu, "evict", 300), A._scratch_bytes(cpu, "tree", 300)]

    take("here")
    other = threading.Thread(target=take, args=("there",))
    other.start()
    other.join()
    for a in got.values():
        assert a[0] is a[1] and a[0] is not a[2]
    assert not {x.data_ptr() for x in got["here"]} & {x.data_ptr() for x in got["there"]}
    assert A._scratch_bytes(cpu, "evict", 512) is got["here"][0]


def evict(L, **kw):
    a = dict(k=0x10000, v=0x90000, w=0x20000, lengths=P, ko=0x10000, vo=0x90000, wo=0x20000, lo=P, kept=P, B=1, Hkv=1, D=64, Dv=64, cap=128, cap_out=128,
             keep=32, recent=4, dtype=1, ws=P, wsb=0, stream=None)
    a.update(kw)
    return L.pjx_kv_cache_evict(*a.values())


OTHER = dict(ko=0x30000, vo=0x40000, wo=0x50000, cap_out=32)


@pytest.mark.parametrize("kw,word", [
    (dict(v=0x10000 + 128, vo=0x10000 + 128), "share"),              # values that begin inside the keys
    (dict(v=0x10000, vo=0x10000, Dv=32), "share"),                   # one address, other rows
    (dict(w=0x10000 + 256, wo=0x10000 + 256), "share"),              # weights inside the keys
    (dict(OTHER, vo=0x30000 + 64), "share"), (dict(OTHER, vo=0x30000), "share"), (dict(OTHER, wo=0x40000 + 64), "share"),
    (dict(OTHER, ko=0x90000), "overlap"), (dict(OTHER, vo=0x10000), "overlap"), (dict(OTHER, wo=0x90000 + 64), "overlap"), (dict(OTHER, ko=0x20000), "overlap"),
])
def test_evict_refuses_memory_that_its_results_share(L, kw, word):
    from probjax_b200 import _lib

    assert evict(L, **kw) == BAD
    assert word in _lib.last_error()


@pytest.mark.parametrize("kw", [{}, OTHER, dict(v=0x10000, vo=0x10000), dict(OTHER, v=0x10000, vo=0x30000), dict(OTHER, v=0x10000)])
def test_evict_takes_keys_that_are_the_values(L, kw):
    from probjax_b200 import _lib

    assert evict(L, **kw) == _lib.PJX_ERR_WORKSPACE  # (the check behind those of the memory)


def accept(L, **kw):
    a = dict(k=0x100000, v=0x200000, kn=P, kb=0, kt=0, vn=P, vb=0, vt=0, lengths=P, path=P, counts=P, table=None, B=1, N=4, Pw=2, Hkv=2, D=64, Dv=64, cap=128, page=0,
             max_pages=0, num_pages=0, dtype=1, out=P, overflow=None, stream=None)
    a.update(kw)
    return L.pjx_kv_cache_accept(*a.values())


@pytest.mark.parametrize("kw", [
    dict(v=0x100000 + 64), dict(v=0x100000, vn=0x2000), dict(v=0x100000, vt=8), dict(v=0x100000, Dv=32), dict(v=0x100000, kb=8),
    dict(table=P, page=64, max_pages=2, num_pages=9, v=0x100000 + 9 * 64 * 2 * 64 * 2 - 16)])
def test_accept_refuses_caches_that_share_memory(L, kw):
    from probjax_b200 import _lib

    assert accept(L, **kw) == BAD
    assert "share" in _lib.last_error()


def test_integers_beyond_32_bits_stay_out_of_range():
    """Parents, lengths, paths and pages of 64-bit tensors: what does not fit is cut to the nearest 32-bit number, which is as far out of range,
    and does not come back as a small one."""
    from probjax_b200.drafts import _int32

    big = torch.tensor([2 ** 32, 2 ** 32 - 1, -2 ** 40, 2 ** 63 - 1, -2 ** 63, 7, -1, 2 ** 31 - 1])
    want = [2 ** 31 - 1, 2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1, -2 ** 31, 7, -1, 2 ** 31 - 1]
    assert _int32(big, torch.device("cpu"), (8,), "parents").tolist() == want
    assert _int32(big.tolist(), torch.device("cpu"), (8,), "parents").tolist() == want
    for dtype in (torch.uint8, torch.int8, torch.int16):
        assert _int32(torch.tensor([3, 100], dtype=dtype), torch.device("cpu"), (2,), "path").tolist() == [3, 100]
    assert _int32(torch.tensor([5, 2 ** 32 - 1], dtype=torch.uint32), torch.device("cpu"), (2,), "path").tolist() == [5, 2 ** 31 - 1]
    assert _int32(torch.zeros((0, 3), dtype=torch.int64), torch.device("cpu"), (0, 3), "path").shape == (0, 3)


def test_rope_axes_refuses_an_infinite_base(L):
    """Its first frequency would be infinity to the power 0 by way of 0 times infinity."""
    import ctypes

    sections = (ctypes.c_int32 * 1)(64)
    for base, rc in ((float("inf"), BAD), (1e30, 0)):
        assert L.pjx_rope_axes(P, 0, 0, P, P, 0, 0, 1, sections, 0, 4, 2, 64, 0, 1, 0, base, 1, None) == rc  # (no sequence: nothing is launched)
