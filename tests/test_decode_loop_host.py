"""Host side of the decode loop's calls; no GPU is touched."""

import threading

import torch


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
