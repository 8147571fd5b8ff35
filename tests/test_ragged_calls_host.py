"""How the ragged-batch calls reach the library, without a GPU: the library and the device
queries are stand-ins, the tensors are on the host."""

import threading
import time

import pytest
import torch

from cvsa import _lib
from cvsa.kernels import chunk_attend, rope_append
from cvsa.runtime.kv_cache import PagedKVCache, SequenceKVManager

BYTES = 1000


class Library:
    """Records (call, current device, workspace) and what overlaps."""

    def __init__(self, pause=0.0):
        self.calls, self.inside, self.overlaps, self.pause = [], {}, 0, pause
        self.device, self.status = 0, _lib.OK
        self.guard = threading.Lock()

    def cvsa_chunk_attend_workspace_size(self, kv, rg, args):
        return BYTES

    def cvsa_chunk_attend(self, kv, rg, args, err, ws, nbytes, stream):
        with self.guard:
            self.calls.append(("chunk_attend", self.device, ws))
            self.overlaps += self.inside.get(ws, 0) > 0
            self.inside[ws] = self.inside.get(ws, 0) + 1
        time.sleep(self.pause)
        with self.guard:
            self.inside[ws] -= 1
        return self.status

    def cvsa_rope_append(self, kv, rg, args, err, stream):
        self.calls.append(("rope_append", self.device, None))
        return self.status

    def cvsa_paged_reserve(self, *args):
        self.calls.append(("reserve", self.device, None))
        return self.status


@pytest.fixture
def fake(monkeypatch):
    """A library and a CUDA runtime with two devices, of which 0 is current; every tensor
    passes for one of device `lib.tensors`."""
    lib = Library()
    lib.tensors, lib.capturing = 0, False

    class OnDevice:
        def __init__(self, index):
            self.index = getattr(index, "index", index)

        def __enter__(self):
            self.before, lib.device = lib.device, self.index

        def __exit__(self, *exc):
            lib.device = self.before

    monkeypatch.setattr(_lib, "load", lambda path=None: lib)
    monkeypatch.setattr(_lib, "same_device", lambda *t: lib.tensors)
    monkeypatch.setattr(_lib, "require_cuda", lambda *t: torch.device("cuda", lib.tensors))
    real_empty = torch.empty  # the tensors stay on the host
    monkeypatch.setattr(torch, "empty", lambda *a, **kw: real_empty(*a, **{**kw, "device": "cpu"}))
    monkeypatch.setattr(_lib, "raw_stream", lambda index: 0)
    monkeypatch.setattr(_lib, "stream_ptr", lambda device: 0)
    monkeypatch.setattr(_lib, "WORKSPACE", _lib.Workspace())
    monkeypatch.setattr(chunk_attend, "_ws_bytes", {})
    monkeypatch.setattr(torch.cuda, "current_device", lambda: lib.device)
    monkeypatch.setattr(torch.cuda, "device", OnDevice)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: lib.capturing)
    return lib


def tensors():
    q, k = torch.zeros(3, 4, 64), torch.zeros(3, 2, 64)
    pool = torch.zeros(4, 16, 2, 64)
    i = torch.zeros(2, dtype=torch.int32)
    return q, k, pool, i


def attend():
    q, _, pool, i = tensors()
    return chunk_attend.chunk_attention(q, pool, pool, i.view(1, 2), i[:1], i)


def test_threads_on_one_stream_share_a_workspace_one_call_at_a_time(fake, monkeypatch):
    """A call's kernels hand partials over in its workspace; first calls of several threads
    find one buffer, which stays."""
    fake.pause = 0.01
    made, real = [], torch.zeros

    def slow_zeros(*a, **kw):
        t = real(*a, **kw)
        if kw.get("dtype") is torch.uint8:
            made.append(t)
            time.sleep(0.02)
        return t

    monkeypatch.setattr(_lib.torch, "zeros", slow_zeros)
    threads = [threading.Thread(target=attend) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(fake.calls) == 4 and len(made) == 1
    assert len({ws for _, _, ws in fake.calls}) == 1
    assert fake.overlaps == 0
    assert all(ws % 256 == 0 for _, _, ws in fake.calls)


def test_a_captured_call_has_a_workspace_of_its_own(fake, monkeypatch):
    """Not the stream's: graphs captured on one stream may run at the same time."""
    attend()
    kept = fake.calls[-1][2]
    fake.capturing = True
    bufs, real = [], torch.empty

    def empty(*a, **kw):
        bufs.append(real(*a, **kw))
        return bufs[-1]

    monkeypatch.setattr(chunk_attend.torch, "empty", empty)
    attend()
    attend()
    own = [ws for _, _, ws in fake.calls[1:]]
    assert kept not in own and len(set(own)) == 2
    for ws, b in zip(own, bufs):
        assert ws % 256 == 0 and b.data_ptr() <= ws and ws + BYTES <= b.data_ptr() + b.numel()


def append():
    q, k, pool, i = tensors()
    return rope_append.rope_append(q, k, k, pool, pool, i.view(1, 2), i[:1], i)


def reserve():
    manager = SequenceKVManager(PagedKVCache(4, 16, 2, 64, device="cpu"), 1, 64)
    return manager.reserve(torch.tensor([0, 3]))


@pytest.mark.parametrize("call,name", [(attend, "chunk_attend"), (append, "rope_append"),
                                       (reserve, "reserve")])
def test_launches_go_to_the_tensors_device(fake, call, name):
    """The default stream's handle is the same on every device, so the tensors' device has to
    be current for the launch, and the caller's is current again afterwards."""
    for device in (0, 1):
        fake.tensors = device
        call()
        assert fake.calls[-1][:2] == (name, device)
        assert fake.device == 0


def test_checks_refuse_what_the_calls_refuse():
    """The check entry points answer as the calls do, whatever else the call would need."""
    lib = _lib.load()
    kv = _lib.KvDesc(256, 256, _lib.DTYPE_BF16, 10, 16, 2, 128, 0, 4096, 256, 128)
    rg = _lib.RaggedDesc(256, None, None, 256, 256, 2, 9, 2, 4)

    def rope(rot=128, hq=8, eps=1e-6):
        return _lib.RopeAppend(256, 256, 256, 256, _lib.DTYPE_BF16, hq, *[1024, 128] * 4, 256, 99,
                               rot, 0, _lib.DTYPE_BF16, None, 256, eps)

    def chunk(hq=8, scale=0.1, window=0):
        return _lib.ChunkAttend(256, 256, None, _lib.DTYPE_BF16, hq, 1024, 128, 1024, 128, scale,
                                1, window)

    assert lib.cvsa_rope_append_check(kv, rg, rope()) == _lib.OK
    assert lib.cvsa_chunk_attend_check(kv, rg, chunk()) == _lib.OK
    for bad in (rope(rot=48), rope(hq=0), rope(eps=-1.0), None):
        st = lib.cvsa_rope_append(kv, rg, bad, None, None)
        assert st != _lib.OK and lib.cvsa_rope_append_check(kv, rg, bad) == st
    for bad in (chunk(hq=7), chunk(hq=130), chunk(scale=-1.0), chunk(window=-1), None):
        st = lib.cvsa_chunk_attend(kv, rg, bad, None, 256, 1 << 40, None)
        assert st != _lib.OK and lib.cvsa_chunk_attend_check(kv, rg, bad) == st
    assert lib.cvsa_rope_append_check(None, rg, rope()) == _lib.ERR_INVALID
    assert lib.cvsa_chunk_attend_check(kv, None, chunk()) == _lib.ERR_INVALID


def test_arguments_past_their_type(fake):
    """A window of any size is a window; other numbers the library's structs cannot hold are
    a ValueError like every refused argument."""
    q, k, pool, i = tensors()
    where = (i.view(1, 2), i[:1], i)
    for window in (2 ** 31 - 1, 2 ** 31, 2 ** 63):
        chunk_attend.chunk_attention(q, pool, pool, *where, window=window)
        assert _lib.ARGS.chunk.window == 2 ** 31 - 1
    for bad in (dict(scale=1e39), dict(scale=-1e39), dict(window=-2 ** 31 - 1)):
        with pytest.raises(ValueError, match="out of range"):
            chunk_attend.chunk_attention(q, pool, pool, *where, **bad)
    with pytest.raises(ValueError, match="out of range"):
        rope_append.rope_append(q, k, k, pool, pool, *where, k_norm=torch.ones(64), eps=1e39)
