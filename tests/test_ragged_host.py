"""Argument checks of the ragged-batch operators, without a GPU."""

import ctypes

import pytest
import torch

from cvsa import _lib
from cvsa.kernels.chunk_attend import chunk_attention
from cvsa.kernels.rope_append import rope_append, rope_table

BF16 = _lib.DTYPE_BF16


def kv(**kw):
    f = dict(k=256, v=256, dt=BF16, nb=10, bs=16, h=2, d=128)
    f.update(kw)
    return _lib.KvDesc(f["k"], f["v"], f["dt"], f["nb"], f["bs"], f["h"], f["d"], 0,
                       f["bs"] * f["h"] * f["d"], f["h"] * f["d"], f["d"])


def ragged(**kw):
    f = dict(cu=256, ids=None, starts=None, tables=256, lens=256, B=2, T=9, S=2, W=4)
    f.update(kw)
    return _lib.RaggedDesc(f["cu"], f["ids"], f["starts"], f["tables"], f["lens"], f["B"], f["T"],
                           f["S"], f["W"])


def chunk(**kw):
    f = dict(q=256, out=256, lse=None, dt=BF16, hq=8, qs=1024, qh=128, os=1024, oh=128, scale=0.1,
             causal=1, window=0)
    f.update(kw)
    return _lib.ChunkAttend(f["q"], f["out"], f["lse"], f["dt"], f["hq"], f["qs"], f["qh"],
                            f["os"], f["oh"], f["scale"], f["causal"], f["window"])


def rope(**kw):
    f = dict(q=256, k=256, v=256, qo=256, dt=BF16, hq=8, s=1024, h=128, cos=256, pos=99, rot=128,
             il=0, ndt=BF16, qn=None, kn=None, eps=1e-6)
    f.update(kw)
    return _lib.RopeAppend(f["q"], f["k"], f["v"], f["qo"], f["dt"], f["hq"], f["s"], f["h"],
                           f["s"], f["h"], f["s"], f["h"], f["s"], f["h"], f["cos"], f["pos"],
                           f["rot"], f["il"], f["ndt"], f["qn"], f["kn"], f["eps"])


INVALID, UNSUPPORTED, WORKSPACE = _lib.ERR_INVALID, _lib.ERR_UNSUPPORTED, _lib.ERR_WORKSPACE


@pytest.mark.parametrize("rg,args,kvd,status", [
    (None, chunk(), kv(), INVALID), (ragged(), None, kv(), INVALID),
    (ragged(), chunk(), None, INVALID), (ragged(B=-1), chunk(), kv(), INVALID),
    (ragged(T=-1), chunk(), kv(), INVALID), (ragged(W=0), chunk(), kv(), INVALID),
    (ragged(cu=None), chunk(), kv(), INVALID), (ragged(S=1), chunk(), kv(), INVALID),
    (ragged(), chunk(dt=9), kv(), INVALID), (ragged(), chunk(hq=7), kv(), INVALID),
    (ragged(), chunk(hq=0), kv(), INVALID), (ragged(), chunk(q=None), kv(), INVALID),
    (ragged(), chunk(scale=0.0), kv(), INVALID), (ragged(), chunk(scale=-1.0), kv(), INVALID),
    (ragged(), chunk(scale=float("nan")), kv(), INVALID),
    (ragged(), chunk(scale=float("inf")), kv(), INVALID),
    (ragged(), chunk(window=-1), kv(), INVALID),
    (ragged(), chunk(window=4, causal=0), kv(), INVALID),
    (ragged(), chunk(q=264), kv(), INVALID), (ragged(), chunk(oh=129), kv(), INVALID),
    (ragged(), chunk(), kv(d=96), UNSUPPORTED), (ragged(), chunk(hq=130), kv(), UNSUPPORTED),
    (ragged(), chunk(), kv(k=8), INVALID)])
def test_chunk_attend_refusals(rg, args, kvd, status):
    lib = _lib.load()
    assert lib.cvsa_chunk_attend(kvd, rg, args, None, 256, 1 << 40, None) == status
    assert lib.cvsa_chunk_attend_workspace_size(kvd, rg, args) == 0


def test_chunk_attend_workspace_and_empty():
    lib = _lib.load()
    need = lib.cvsa_chunk_attend_workspace_size(kv(), ragged(), chunk())
    assert need > 0
    for ws, n in ((None, need), (128, need), (256, need - 1)):
        assert lib.cvsa_chunk_attend(kv(), ragged(), chunk(), None, ws, n, None) == WORKSPACE
    # nothing to do: no launch, no workspace
    for rg in (ragged(B=0), ragged(T=0)):
        assert lib.cvsa_chunk_attend(kv(), rg, chunk(), None, None, 0, None) == _lib.OK


@pytest.mark.parametrize("rg,args,kvd,status", [
    (None, rope(), kv(), INVALID), (ragged(), None, kv(), INVALID),
    (ragged(), rope(), None, INVALID), (ragged(S=1), rope(), kv(), INVALID),
    (ragged(), rope(dt=7), kv(), INVALID), (ragged(), rope(hq=0), kv(), INVALID),
    (ragged(), rope(q=None), kv(), INVALID), (ragged(), rope(k=None), kv(), INVALID),
    (ragged(), rope(qo=None), kv(), INVALID), (ragged(), rope(rot=0), kv(), INVALID),
    (ragged(), rope(rot=48), kv(), INVALID), (ragged(), rope(rot=160), kv(), INVALID),
    (ragged(), rope(pos=0), kv(), INVALID), (ragged(), rope(h=129), kv(), INVALID),
    (ragged(), rope(cos=260), kv(), INVALID), (ragged(), rope(qn=256, ndt=1), kv(), INVALID),
    (ragged(), rope(kn=256, eps=-1.0), kv(), INVALID), (ragged(), rope(kn=264), kv(), INVALID),
    (ragged(), rope(), kv(d=96), UNSUPPORTED), (ragged(T=1 << 29), rope(), kv(), UNSUPPORTED)])
def test_rope_append_refusals(rg, args, kvd, status):
    assert _lib.load().cvsa_rope_append(kvd, rg, args, None, None) == status


def test_reserve_refusals():
    f = _lib.load().cvsa_paged_reserve
    assert f(0, 256, None, 2, 2, 256, 4, 256, 256, 256, 8, 256, None, None, None) == INVALID
    assert f(16, 256, None, -1, 2, 256, 4, 256, 256, 256, 8, 256, None, None, None) == INVALID
    assert f(16, None, None, 2, 2, 256, 4, 256, 256, 256, 8, 256, None, None, None) == INVALID
    assert f(16, 256, None, 2, 2, 256, 0, 256, 256, 256, 8, 256, None, None, None) == INVALID
    assert f(16, 256, None, 0, 2, 256, 4, 256, 256, 256, 8, 256, None, None, None) == _lib.OK


def test_descriptor_sizes_match_the_header():
    """LP64 sizes of the structs the header declares."""
    assert ctypes.sizeof(_lib.RaggedDesc) == 5 * 8 + 4 * 4
    assert ctypes.sizeof(_lib.RopeAppend) == 4 * 8 + 8 + 8 * 8 + 8 + 4 * 4 + 2 * 8 + 8
    assert ctypes.sizeof(_lib.ChunkAttend) == 3 * 8 + 8 + 4 * 8 + 16


def test_python_checks():
    q, k = torch.zeros(3, 4, 64), torch.zeros(3, 2, 64)
    pool = torch.zeros(4, 16, 2, 64)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        chunk_attention(q, pool, pool, i.view(1, 2), i[:1], i)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        rope_append(q, k, k, pool, pool, i.view(1, 2), i[:1], i)
    with pytest.raises(ValueError):
        rope_table(0, 64, device="cpu")
    with pytest.raises(ValueError):
        rope_table(8, 7, device="cpu")
    # the ragged description
    ok = dict(num_tokens=3, cu_tokens=i, block_tables=i.view(1, 2), context_lens=i[:1],
              seq_ids=None, start_positions=None)
    assert _lib.ragged_desc(**ok).batch == 1
    for bad in (dict(cu_tokens=i.long()), dict(context_lens=i), dict(seq_ids=i),
                dict(block_tables=i), dict(start_positions=i.float()[:1])):
        with pytest.raises(ValueError):
            _lib.ragged_desc(**{**ok, **bad})
    t = torch.zeros(3, 2, 9)[:, :, 1:]
    assert _lib.token_rows(t, "t").is_contiguous()
    s = torch.zeros(3, 4, 64)[:, 1:3]
    assert _lib.token_rows(s, "s").data_ptr() == s.data_ptr()
    with pytest.raises(ValueError):
        _lib.token_rows(torch.zeros(3, 2), "t")


def test_rope_table_values():
    t = rope_table(50, 32, base=500.0, device="cpu")
    assert t.shape == (50, 32) and t.dtype == torch.float32
    ang = 49 * 500.0 ** (-2 * 3 / 32)
    assert abs(float(t[49, 3]) - torch.cos(torch.tensor(ang, dtype=torch.float64))) < 1e-7
    assert abs(float(t[49, 19]) - torch.sin(torch.tensor(ang, dtype=torch.float64))) < 1e-7


def test_packed_arguments_are_the_structs():
    """One pack fills the per-thread structs as their constructors would."""
    mem = _lib.ARGS
    kvf = (11, 12, 2, 10, 16, 2, 128, 0, 4096, 256, 128)
    rgf = (21, 22, 23, 24, 25, 3, 9, 4, 7)
    chf = (31, 32, 0, 1, 8, 1024, 128, 2048, 256, 0.5, True, 40)
    rof = (41, 42, 43, 44, 2, 8, 1, 2, 3, 4, 5, 6, 7, 8, 45, 99, 64, True, 0, 46, 47, 0.25)

    def same(got, want):
        for name, _ in want._fields_:
            assert getattr(got, name) == getattr(want, name), name

    mem.pack_chunk(mem.buf, 0, *kvf, *rgf, *chf)
    same(mem.kv, _lib.KvDesc(*kvf))
    same(mem.rg, _lib.RaggedDesc(*rgf))
    same(mem.chunk, _lib.ChunkAttend(*chf))
    mem.pack_rope(mem.buf, 0, *kvf, *rgf, *rof)
    same(mem.rope, _lib.RopeAppend(*rof))
    k = torch.zeros(3, 16, 2, 64, dtype=torch.bfloat16)
    same(_lib.KvDesc(*_lib.kv_fields(k, k)), _lib.kv_desc(k, k))
    with pytest.raises(ValueError):
        _lib.kv_fields(k, k.float())
    with pytest.raises(ValueError):
        _lib.kv_fields(k.transpose(2, 3), k.transpose(2, 3))
