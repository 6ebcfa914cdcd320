"""Two threads on one HeadRotation or CacheAppend: each call hands the library its own operands (no GPU)."""
import ctypes
import threading
import types

import pytest

torch = pytest.importorskip("torch")

from paged_decode import _native, rotary
from paged_decode.layout import Layout


class Library:
    """Entry points with the library's signatures that meet another caller before they look at their operands."""

    def __init__(self):
        self.meet, self.seen = threading.Barrier(2), {}
        for name in ("pd_rotate_heads", "pd_cache_append"):
            restype, argtypes = _native.SIGNATURES[name]
            setattr(self, name, ctypes.CFUNCTYPE(restype, *argtypes)(getattr(self, "_" + name)))

    def _look(self, tokens, *rows):
        self.meet.wait(20)                                  # both threads are inside their call
        rows = [_native.Heads.from_address(r) for r in rows]
        self.seen[tokens] = [(r.data, r.token_stride, r.head_stride, r.heads) for r in rows] + [
            (r.out, r.out_token_stride, r.out_head_stride) for r in rows[:1]]
        self.meet.wait(20)
        return 0

    def _pd_rotate_heads(self, rotation, q, k, tokens, positions, dtype, error, device, stream):
        return self._look(tokens, q, k)

    def _pd_cache_append(self, layout, rotation, q, k, v, tokens, *rest):
        return self._look(tokens, q, k, v)


@pytest.fixture
def library(monkeypatch):
    library = Library()
    monkeypatch.setattr(rotary, "_cuda_device", lambda device: torch.device("cpu"))
    monkeypatch.setattr(rotary._native, "load", lambda: library)
    monkeypatch.setattr(rotary._native, "stream_of", lambda index: 0)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: types.SimpleNamespace(synchronize=lambda: None))
    return library


def together(*calls):
    failures = []

    def guarded(call):
        try:
            call()
        except BaseException as e:  # noqa: BLE001
            failures.append(e)

    threads = [threading.Thread(target=guarded, args=(c,)) for c in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures, failures


def described(out, *rows):
    return [(x.data_ptr(), x.stride(0), x.stride(1), x.shape[1]) for x in rows] + [
        (out.data_ptr(), out.stride(0), out.stride(1))]


def heads(tokens, *counts):
    packed = torch.zeros((tokens, sum(counts) + tokens % 3, 64))       # strides differ with the tokens
    return list(packed[:, : sum(counts)].split(counts, 1))


def test_rotations_keep_their_operands_apart(library):
    rotation = rotary.HeadRotation(64, device="cuda")
    rotation._index = -1                                    # what a CPU tensor's get_device() gives
    want, calls = {}, []
    for tokens, (hq, hk) in ((4, (8, 2)), (4096, (5, 1))):
        q, k = heads(tokens, hq, hk)
        out, k_out = torch.empty(q.shape), torch.empty(k.shape)
        want[tokens] = described(out, q, k)
        positions = torch.zeros(tokens, dtype=torch.int32)
        calls.append(lambda q=q, k=k, p=positions, o=out, ko=k_out: rotation.run(q, k, p, q_out=o, k_out=ko))
    together(*calls)
    assert library.seen == want


def test_appends_keep_their_operands_apart(library):
    layout = Layout(2, 4, 2, 64, 16, 8)
    append = rotary.CacheAppend(layout, device="cuda")
    append._index = -1
    caches = [torch.zeros((8, 16, 2, 64)) for _ in range(2)]
    table, lengths = torch.zeros((2, 4), dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    indptr = torch.zeros(3, dtype=torch.int32)
    want, calls = {}, []
    for tokens in (4, 60):
        q, k, v = heads(tokens, 4, 2, 2)
        out = torch.empty(q.shape)
        want[tokens] = described(out, q, k, v)
        calls.append(lambda q=q, k=k, v=v, o=out: append.run(k, v, *caches, table, lengths, q=q, indptr=indptr,
                                                            q_out=o))
    together(*calls)
    assert library.seen == want
