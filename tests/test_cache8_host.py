"""Argument checks of the 8-bit cache, the key weights and the eviction, without a GPU."""

import subprocess
import sys

import pytest
import torch

from cvsa import _lib
from cvsa.kernels import evict as evict_module
from cvsa.kernels.chunk_attend import chunk_attention
from cvsa.kernels.evict import evict
from cvsa.kernels.key_weights import key_weights
from cvsa.kernels.rope_append import rope_append
from cvsa.runtime.eviction import WeightedEviction
from cvsa.runtime.kv_cache import PagedKVCache, SequenceKVManager
from test_ragged_host import chunk, kv, ragged, rope

F8 = torch.float8_e4m3fn
E4M3, BF16 = _lib.DTYPE_E4M3, _lib.DTYPE_BF16
OK, INVALID, UNSUPPORTED = _lib.OK, _lib.ERR_INVALID, _lib.ERR_UNSUPPORTED


def weights(**kw):
    f = dict(q=256, lse=256, dt=BF16, hq=8, qs=1024, qh=128, scale=0.1, decay=1.0, causal=1,
             window=0, prior=256, out=256, stride=64)
    f.update(kw)
    return _lib.KeyWeights(f["q"], f["lse"], f["dt"], f["hq"], f["qs"], f["qh"], f["scale"],
                           f["decay"], f["causal"], f["window"], f["prior"], f["out"], f["stride"])


def cut(**kw):
    f = dict(w=256, ws=64, out=512, os=32, new=256, pages=2, kept=256, keep=32, sink=0, recent=0)
    f.update(kw)
    return _lib.Evict(f["w"], f["ws"], f["out"], f["os"], f["new"], f["pages"], f["kept"],
                      f["keep"], f["sink"], f["recent"])


def pages(**kw):
    f = dict(tables=256, lens=256, alloc=256, evicted=256, free=256, head=256, new=256, plan=256,
             S=2, W=4, bs=16, keep=32, n=10)
    f.update(kw)
    return _lib.EvictPages(f["tables"], f["lens"], f["alloc"], f["evicted"], f["free"], f["head"],
                           f["new"], f["plan"], f["S"], f["W"], f["bs"], f["keep"], f["n"])


def test_scales_go_with_pools_of_eight_bits():
    lib, r8, r16 = _lib.load(), kv(dt=E4M3), kv()
    assert lib.cvsa_rope_append_to_check(r8, 256, 256, ragged(), rope(), None) == OK
    assert lib.cvsa_rope_append_to_check(r16, None, None, ragged(), rope(), 256) == OK
    assert lib.cvsa_chunk_attend_q8_check(r8, 256, 256, ragged(), chunk()) == OK
    assert lib.cvsa_key_weights_check(r8, 256, ragged(), weights()) == OK
    assert lib.cvsa_key_weights_check(r16, None, ragged(), weights()) == OK
    for k, v in ((None, 256), (256, None), (None, None)):
        assert lib.cvsa_rope_append_to(r8, k, v, ragged(), rope(), None, None, None) == INVALID
        assert lib.cvsa_chunk_attend_q8(r8, k, v, ragged(), chunk(), None, 256, 1 << 40,
                                        None) == INVALID
        assert lib.cvsa_evict(r8, k, v, 256, 256, 2, 4, cut(), None, None) == INVALID
    assert lib.cvsa_rope_append_to(r16, 256, 256, ragged(), rope(), None, None, None) == INVALID
    assert lib.cvsa_chunk_attend_q8(r16, None, None, ragged(), chunk(), None, 256, 1 << 40,
                                    None) == INVALID
    assert lib.cvsa_key_weights(r8, None, ragged(), weights(), None, None) == INVALID
    assert lib.cvsa_key_weights(r16, 256, ragged(), weights(), None, None) == INVALID
    # the calls without scales take no pool of 8 bits
    assert lib.cvsa_chunk_attend(r8, ragged(), chunk(), None, 256, 1 << 40, None) == INVALID
    assert lib.cvsa_rope_append(r8, ragged(), rope(), None, None) == INVALID
    assert lib.cvsa_paged_gather(r8, 256, 1, 256, 256, None, None) == INVALID
    qd = _lib.QueryDesc(256, BF16, 2, 8, 4, 256, 256)
    assert lib.cvsa_score_pages(qd, r8, 256, None) == INVALID
    assert lib.cvsa_chunk_attend_q8_workspace_size(r8, None, None, ragged(), chunk()) == 0
    need = lib.cvsa_chunk_attend_q8_workspace_size(r8, 256, 256, ragged(), chunk())
    assert need > 0
    assert lib.cvsa_chunk_attend_q8(r8, 256, 256, ragged(), chunk(), None, 256, need - 1,
                                    None) == _lib.ERR_WORKSPACE
    assert lib.cvsa_chunk_attend_q8(r8, 256, 256, ragged(), chunk(), None, None, need,
                                    None) == _lib.ERR_WORKSPACE


@pytest.mark.parametrize("rg,args,kvd,status", [
    (None, weights(), kv(), INVALID), (ragged(), None, kv(), INVALID),
    (ragged(), weights(), None, INVALID), (ragged(B=-1), weights(), kv(), INVALID),
    (ragged(), weights(dt=9), kv(), INVALID), (ragged(), weights(dt=E4M3), kv(), INVALID),
    (ragged(), weights(hq=7), kv(), INVALID), (ragged(), weights(hq=0), kv(), INVALID),
    (ragged(), weights(q=None), kv(), INVALID), (ragged(), weights(lse=None), kv(), INVALID),
    (ragged(), weights(prior=None), kv(), INVALID), (ragged(), weights(out=None), kv(), INVALID),
    (ragged(), weights(scale=0.0), kv(), INVALID),
    (ragged(), weights(scale=float("nan")), kv(), INVALID),
    (ragged(), weights(decay=-0.5), kv(), INVALID),
    (ragged(), weights(decay=float("inf")), kv(), INVALID),
    (ragged(), weights(decay=float("nan")), kv(), INVALID),
    (ragged(), weights(window=-1), kv(), INVALID),
    (ragged(), weights(window=3, causal=0), kv(), INVALID),
    (ragged(), weights(stride=63), kv(), INVALID), (ragged(), weights(q=264), kv(), INVALID),
    (ragged(), weights(qs=1028), kv(), INVALID), (ragged(), weights(hq=130), kv(), UNSUPPORTED),
    (ragged(), weights(qh=192), kv(d=192), UNSUPPORTED),
    (ragged(W=1 << 30), weights(stride=1 << 40), kv(), UNSUPPORTED)])
def test_key_weights_refusals(rg, args, kvd, status):
    lib = _lib.load()
    assert lib.cvsa_key_weights(kvd, None, rg, args, None, None) == status
    assert lib.cvsa_key_weights_check(kvd, None, rg, args) == status


@pytest.mark.parametrize("kw", [
    dict(keep=0), dict(keep=-3), dict(sink=-1), dict(recent=-1), dict(sink=20, recent=13),
    dict(sink=2 ** 31 - 1, recent=2 ** 31 - 1), dict(pages=1), dict(pages=3), dict(ws=63),
    dict(os=31), dict(out=256, os=64, ws=80), dict(w=None), dict(new=None), dict(kept=None)])
def test_evict_refusals(kw):
    assert _lib.load().cvsa_evict(kv(), None, None, 256, 256, 2, 4, cut(**kw), None,
                                  None) == INVALID


def test_evict_refuses_other_shapes():
    lib = _lib.load()
    assert lib.cvsa_evict(None, None, None, 256, 256, 2, 4, cut(), None, None) == INVALID
    assert lib.cvsa_evict(kv(), None, None, 256, 256, 2, 4, None, None, None) == INVALID
    assert lib.cvsa_evict(kv(), None, None, 256, 256, -1, 4, cut(), None, None) == INVALID
    assert lib.cvsa_evict(kv(), None, None, 256, 256, 2, 0, cut(), None, None) == INVALID
    assert lib.cvsa_evict(kv(), None, None, None, 256, 2, 4, cut(), None, None) == INVALID
    assert lib.cvsa_evict(kv(), None, None, 256, 256, 2, 1 << 27, cut(ws=1 << 40), None,
                          None) == UNSUPPORTED
    assert lib.cvsa_evict(kv(), None, None, None, None, 0, 4, cut(), None, None) == OK
    for kw in (dict(S=-1), dict(W=0), dict(bs=0), dict(keep=0), dict(keep=65), dict(n=-1),
               dict(tables=None), dict(lens=None), dict(alloc=None), dict(evicted=None),
               dict(free=None), dict(head=None), dict(new=None), dict(plan=None)):
        assert lib.cvsa_evict_reserve(pages(**kw), None, None) == INVALID
        assert lib.cvsa_evict_commit(pages(**kw), None, None) == INVALID
    assert lib.cvsa_evict_reserve(None, None, None) == INVALID
    assert lib.cvsa_evict_commit(pages(S=0), None, None) == OK


class Recorder:
    """A library that records the calls it gets and the device current at each."""

    def __init__(self):
        self.calls, self.device = [], 0

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, self.device, args))
            return 1000 if name.endswith("size") else OK
        return call


@pytest.fixture
def fake(monkeypatch):
    """A library and a CUDA runtime with two devices, of which 0 is current; host tensors
    pass for tensors of device `lib.tensors`."""
    lib = Recorder()
    lib.tensors = 0

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
    real = torch.empty
    monkeypatch.setattr(torch, "empty", lambda *a, **kw: real(*a, **{**kw, "device": "cpu"}))
    monkeypatch.setattr(_lib, "raw_stream", lambda index: 0)
    monkeypatch.setattr(_lib, "stream_ptr", lambda device: 0)
    monkeypatch.setattr(_lib, "WORKSPACE", _lib.Workspace())
    monkeypatch.setattr(torch.cuda, "current_device", lambda: lib.device)
    monkeypatch.setattr(torch.cuda, "device", OnDevice)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    return lib


def args():
    f8 = torch.zeros(4, 16, 2, 64, dtype=F8)
    i = torch.zeros(2, dtype=torch.int32)
    return dict(q=torch.zeros(3, 4, 64), k=torch.zeros(3, 2, 64), f8=f8,
                wide=torch.zeros(4, 16, 2, 64), s=torch.ones(4, 2), tables=i.view(1, 2),
                lens=i[:1], cu=i, w=torch.zeros(1, 2, 32), lse=torch.zeros(3, 4),
                new=torch.zeros(1, 1, dtype=torch.int32))


def attend(a, **kw):
    return chunk_attention(a["q"], a["f8"], a["f8"], a["tables"], a["lens"], a["cu"],
                           **{**dict(k_scale=a["s"], v_scale=a["s"]), **kw})


def append(a, **kw):
    return rope_append(a["q"], a["k"], a["k"], a["f8"], a["f8"], a["tables"], a["lens"], a["cu"],
                       **{**dict(k_scale=a["s"], v_scale=a["s"]), **kw})


def weigh(a, **kw):
    f = dict(lse=a["lse"], weights=a["w"], k_scale=a["s"], cache=a["f8"])
    f.update(kw)
    return key_weights(a["q"], f.pop("lse"), f.pop("cache"), a["tables"], a["lens"], a["cu"],
                       f.pop("weights"), **f)


def drop(a, **kw):
    f = dict(new=a["new"], keep=16, weights=a["w"], k_scale=a["s"], v_scale=a["s"])
    f.update(kw)
    return evict(a["f8"], a["f8"], a["tables"], a["lens"], f.pop("weights"), f.pop("new"),
                 f.pop("keep"), **f)


@pytest.mark.parametrize("call,name", [(attend, "cvsa_chunk_attend_q8"),
                                       (append, "cvsa_rope_append_to"),
                                       (weigh, "cvsa_key_weights"), (drop, "cvsa_evict")])
def test_calls_reach_the_library_on_the_tensors_device(fake, call, name):
    for device in (0, 1):
        fake.tensors = device
        call(args())
        assert fake.calls[-1][:2] == (name, device)
        assert fake.device == 0


def test_a_shift_alone_goes_the_new_way(fake):
    a = args()
    shift = torch.zeros(1, dtype=torch.int32)
    rope_append(a["q"], a["k"], a["k"], a["wide"], a["wide"], a["tables"], a["lens"], a["cu"])
    assert fake.calls[-1][0] == "cvsa_rope_append"
    rope_append(a["q"], a["k"], a["k"], a["wide"], a["wide"], a["tables"], a["lens"], a["cu"],
                position_shift=shift)
    assert fake.calls[-1][0] == "cvsa_rope_append_to"
    assert fake.calls[-1][2][1:3] == (None, None) and fake.calls[-1][2][5] == shift.data_ptr()


def test_python_refusals(fake):
    a = args()
    bad_scales = (torch.ones(4, 3), torch.ones(4, 2).double(), torch.ones(2, 4).t(),
                  torch.ones(4, 2, 1))
    for call in (attend, append, drop):
        for s in bad_scales:
            with pytest.raises(ValueError):
                call(a, k_scale=s)
            with pytest.raises(ValueError):
                call(a, v_scale=s)
        with pytest.raises(ValueError, match="together"):
            call(a, v_scale=None)
        with pytest.raises(ValueError, match="8-bit"):
            call(a, k_scale=None, v_scale=None)
        with pytest.raises(ValueError, match="8-bit"):
            call({**a, "f8": a["wide"]})
    with pytest.raises(ValueError, match="8-bit"):
        weigh(a, k_scale=None)
    with pytest.raises(ValueError, match="8-bit"):
        weigh(a, cache=a["wide"])
    for bad in (torch.zeros(2, dtype=torch.int32), torch.zeros(1), torch.zeros(1, 1)):
        with pytest.raises(ValueError, match="position_shift"):
            append(a, position_shift=bad)
    for bad in (torch.zeros(3, 5), torch.zeros(3, 4).double(), torch.zeros(4, 3).t()):
        with pytest.raises(ValueError, match="lse"):
            weigh(a, lse=bad)
    for bad in (torch.zeros(1, 3, 32), torch.zeros(2, 2, 32), torch.zeros(1, 2, 32).double(),
                torch.zeros(1, 32, 2).transpose(1, 2), torch.zeros(2, 32)):
        with pytest.raises(ValueError, match="weights"):
            weigh(a, weights=bad)
        with pytest.raises(ValueError, match="weights"):
            weigh(a, out=bad)
        with pytest.raises(ValueError, match="weights"):
            drop(a, weights=bad)
    with pytest.raises(ValueError, match="out of range"):
        weigh(a, decay=1e39)
    for kw in (dict(keep=0), dict(keep=-1), dict(sink=-1), dict(sink=17), dict(sink=9, recent=8),
               dict(keep=2 ** 31)):
        with pytest.raises(ValueError, match="keep must be"):
            drop(a, **kw)
    with pytest.raises(ValueError, match="new_tables"):
        drop(a, keep=17)
    with pytest.raises(ValueError, match="new_tables"):
        drop(a, new=torch.zeros(1, 1))
    with pytest.raises(ValueError, match="kept"):
        drop(a, kept=torch.zeros(1, 2, 15, dtype=torch.int32))
    w = torch.zeros(100)
    with pytest.raises(ValueError, match="memory of its own"):
        drop(a, weights=w[:64].view(1, 2, 32), out_weights=w[32:96].view(1, 2, 32))
    with pytest.raises(ValueError, match="memory of its own"):
        drop(a, weights=w[:64].view(1, 2, 32), out_weights=w[:32].view(1, 2, 16))
    drop(a, weights=w[:64].view(1, 2, 32), out_weights=w[64:96].view(1, 2, 16))
    assert fake.calls[-1][0] == "cvsa_evict"


def test_overlap():
    w = torch.zeros(10)
    assert evict_module._overlap(w, w) and evict_module._overlap(w[:6], w[5:])
    assert not evict_module._overlap(w[:5], w[5:]) and not evict_module._overlap(w[5:], w[:5])


def test_manager_evicts_in_three_calls(fake):
    m = SequenceKVManager(PagedKVCache(8, 16, 2, 64, device="cpu"), 1, 64)
    assert m.evicted is None
    m.evict(torch.zeros(1, 2, 64), 20, 4, 8)
    assert [c[0] for c in fake.calls] == ["cvsa_evict_reserve", "cvsa_evict", "cvsa_evict_commit"]
    assert m.evicted.tolist() == [0]
    fake.calls.clear()
    for kw in (dict(keep=0), dict(keep=65), dict(keep=20, sink=21)):
        with pytest.raises(ValueError):
            m.evict(torch.zeros(1, 2, 64), **kw)
    assert "cvsa_evict_commit" not in [c[0] for c in fake.calls]


def test_eviction_refusals():
    m = SequenceKVManager(PagedKVCache(8, 16, 2, 64, device="cpu"), 1, 64)
    for kw in (dict(keep=0), dict(keep=4, sink=5), dict(keep=4, sink=2, recent=3),
               dict(keep=4, recent=-1)):
        with pytest.raises(ValueError):
            WeightedEviction(m, **kw)


def test_eight_bit_cache_has_scales():
    c = PagedKVCache(8, 16, 2, 64, dtype=F8, device="cpu")
    assert c.k_scale.shape == c.v_scale.shape == (8, 2) and c.k_cache.dtype is F8
    assert PagedKVCache(8, 16, 2, 64, device="cpu").k_scale is None


def test_key_weights_into_part_of_what_was_there(fake):
    a, w = args(), torch.zeros(128)
    for i in (1, 32, 63):
        with pytest.raises(ValueError, match="memory of its own"):
            weigh(a, weights=w[:64].view(1, 2, 32), out=w[i:i + 64].view(1, 2, 32))
    for out in (w[:64], w[64:]):
        weigh(a, weights=w[:64].view(1, 2, 32), out=out.view(1, 2, 32))
        assert fake.calls[-1][0] == "cvsa_key_weights"


def alone(code):
    """`code` in a process of its own, which may end badly."""
    code = f"import sys\nsys.path[:0] = {sys.path!r}\n" + code
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True)
    assert r.returncode == 0, (r.returncode, r.stdout[-200:], r.stderr[-500:])


def test_a_batch_without_tokens():
    """No tokens, any number of query heads a KV head: nothing to do. (The plan once divided by
    its groups' tokens, 0 of them, which ends the process.)"""
    alone(f"""
from cvsa import _lib
from test_ragged_host import chunk, kv, ragged
lib, r8 = _lib.load(), kv(dt={E4M3})
for hq in (2, 16, 18, 32, 64, 66, 128):
    for B in (0, 1, 5):
        for dt in ({BF16}, {_lib.DTYPE_F32}):
            print(hq, B, dt, flush=True)
            a = r8, 256, 256, ragged(T=0, B=B, S=5), chunk(hq=hq, dt=dt, q=None, out=None)
            assert lib.cvsa_chunk_attend_q8_check(*a) == 0
            assert lib.cvsa_chunk_attend_q8(*a, None, None, 0, None) == 0
            assert lib.cvsa_chunk_attend_q8_workspace_size(*a) > 0
""")


def test_few_token_grid_fits_its_workspace(tmp_path):
    """The descriptors ahead of the partial slots, and the merge's weights, hold 320 blocks: a
    device of more than 160 multiprocessors gets no more. (The library's function that counts
    them gives way to one of the same name that was loaded before it.)"""
    src, shim = tmp_path / "sms.cpp", str(tmp_path / "sms.so")
    src.write_text("int n_sms;\nnamespace cvsa { int num_sms() { return n_sms; } }\n")
    subprocess.run(["g++", "-shared", "-fPIC", "-o", shim, str(src)], check=True)
    alone(f"""
import ctypes
shim = ctypes.CDLL({shim!r}, ctypes.RTLD_GLOBAL)
from cvsa import _lib
from test_ragged_host import chunk, kv, ragged
lib, blocks = _lib.load(), ctypes.CDLL(_lib.LIB_PATH)._ZN4cvsa14chunk_few_ctasEv
for sms in (1, 148, 160, 161, 400):
    ctypes.c_int.in_dll(shim, "n_sms").value = sms
    assert blocks() == min(2 * sms, 320), (sms, blocks())
    # two slots of 32 rows a block fit behind the descriptors
    size = lib.cvsa_chunk_attend_q8_workspace_size(kv(dt={E4M3}), 256, 256, ragged(), chunk())
    assert size >= 320 * 16 + blocks() * 2 * 32 * (128 + 2) * 4, (sms, size)
""")
