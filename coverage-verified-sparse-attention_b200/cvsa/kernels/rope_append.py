"""New tokens into the paged cache: query/key norms, position rotation, append.

`rope_append` takes the packed new tokens of a ragged batch (sequence b owns
tokens cu_tokens[b]..cu_tokens[b + 1]; q, k and v may be column ranges of one
projection output), norms and rotates the query and key rows in fp32, returns
the queries and writes the keys and values to the slots of their positions, in
one launch (csrc/rope_append.cu). The pages must have been reserved
(`cvsa.runtime.kv_cache.SequenceKVManager.reserve`). The reference leaves
norms and rotation to the model library and appends token by token
(cvsa/runtime/kv_cache.py:133-150).
"""

import struct
from typing import Callable, Optional

import torch

from cvsa import _lib


def rope_table(max_positions: int, rot_dim: int, base: float = 10000.0,
               device="cuda") -> torch.Tensor:
    """[max_positions, rot_dim] float32: cos(p * base^(-2i / rot_dim)), then the sines.

    The angles are formed in 64 bits: at position 131072 a 32-bit product is
    off by up to 4e-3 radians."""
    if max_positions <= 0 or rot_dim <= 0 or rot_dim % 2:
        raise ValueError("max_positions must be positive, rot_dim positive and even")
    freq = base ** (-torch.arange(0, rot_dim, 2, dtype=torch.float64, device=device) / rot_dim)
    ang = torch.arange(max_positions, dtype=torch.float64, device=device)[:, None] * freq
    return torch.cat([ang.cos(), ang.sin()], 1).float().contiguous()


def _weights(w: Optional[torch.Tensor], name: str, D: int) -> Optional[torch.Tensor]:
    if w is None:
        return None
    if w.shape != (D,):
        raise ValueError(f"{name} must be [head_dim]")
    w = w.contiguous()
    return w.clone() if w.data_ptr() % 16 else w


def rope_append(q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor,
                k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                context_lens: torch.Tensor, cu_tokens: torch.Tensor,
                cos_sin: Optional[torch.Tensor] = None, q_norm: Optional[torch.Tensor] = None,
                k_norm: Optional[torch.Tensor] = None, eps: float = 1e-6,
                interleaved: bool = False, seq_ids: Optional[torch.Tensor] = None,
                start_positions: Optional[torch.Tensor] = None,
                out: Optional[torch.Tensor] = None,
                dev_error: Optional[torch.Tensor] = None, *,
                k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None,
                position_shift: Optional[torch.Tensor] = None,
                _reserve: Optional[Callable[[], None]] = None) -> Optional[torch.Tensor]:
    """Normed and rotated queries [T, H_q, D] (None without q); keys and values are appended.

    q [T, H_q, D], k and v [T, H_kv, D] in one dtype (the pool may have
    another); context_lens count the new tokens; cos_sin is a `rope_table`
    (its width is the rotated part of a head, None: no rotation); q_norm and
    k_norm are RMS-norm weights [D]; interleaved pairs neighbouring elements
    instead of the halves of the rotated part. start_positions and seq_ids as
    returned by / given to `reserve`. `out` may be q itself.

    k_scale, v_scale [num_blocks, H_kv] float32: the scales of an 8-bit cache
    (float8_e4m3fn pools), which the call keeps (csrc/append8.cu): a page's is the
    least power of two, from 2^-15 to 2^7, with 448 times it at least the page's largest
    absolute value. position_shift [num_seqs] int32 is added to a token's
    position for the rotation: how many keys were evicted before it.
    """
    # _reserve, if given, makes the reservation when nothing can refuse the call any more
    # (it may not call an operator that packs its arguments into this thread's memory)
    dev = _lib.same_device(k, q, v, k_cache, v_cache, block_tables, context_lens, cu_tokens,
                           cos_sin, q_norm, k_norm, seq_ids, start_positions, out, dev_error,
                           k_scale, v_scale, position_shift)
    if dev != torch.cuda.current_device():  # a launch goes to the current device
        with torch.cuda.device(dev):
            return rope_append(q, k, v, k_cache, v_cache, block_tables, context_lens, cu_tokens,
                               cos_sin, q_norm, k_norm, eps, interleaved, seq_ids,
                               start_positions, out, dev_error, k_scale=k_scale,
                               v_scale=v_scale, position_shift=position_shift,
                               _reserve=_reserve)
    T, Hkv, D = k.shape
    if v.shape != k.shape or k_cache.dim() != 4 or tuple(k_cache.shape[2:]) != (Hkv, D):
        raise ValueError("k and v must be [T, H_kv, D] with the cache's H_kv and D")
    if v.dtype != k.dtype or (q is not None and q.dtype != k.dtype):
        raise ValueError("q, k and v dtypes differ")
    k, v = _lib.token_rows(k, "k"), _lib.token_rows(v, "v")
    Hq, qs, os_, qp, op = 0, (0, 0), (0, 0), 0, 0
    if q is not None:
        if q.dim() != 3 or q.shape[0] != T or q.shape[2] != D:
            raise ValueError("q must be [T, H_q, D]")
        Hq = q.shape[1]
        q = _lib.token_rows(q, "q")
        if out is None:
            out = q.new_empty((T, Hq, D))
        elif out.shape != q.shape or out.dtype != q.dtype or out.stride(2) != 1:
            raise ValueError("out must have q's shape and dtype and contiguous rows")
        qs, os_ = q.stride(), out.stride()
        qp, op = q.data_ptr(), out.data_ptr()
    elif out is not None or q_norm is not None:
        raise ValueError("out and q_norm need q")
    q_norm, k_norm = _weights(q_norm, "q_norm", D), _weights(k_norm, "k_norm", D)
    ndt = k.dtype
    for w in (q_norm, k_norm):
        if w is not None:
            ndt = w.dtype
    if q_norm is not None and k_norm is not None and q_norm.dtype != k_norm.dtype:
        raise ValueError("q_norm and k_norm dtypes differ")
    rot = pos = 0
    if cos_sin is not None:
        if cos_sin.dim() != 2 or cos_sin.dtype != torch.float32 or not cos_sin.is_contiguous():
            raise ValueError("cos_sin must be a contiguous float32 [max_positions, rot_dim]")
        pos, rot = cos_sin.shape
    scaled = k_scale is not None
    if scaled != (v_scale is not None):
        raise ValueError("k_scale and v_scale go together")
    if position_shift is not None and (
            position_shift.dtype is not torch.int32 or not position_shift.is_contiguous()
            or position_shift.shape != context_lens.shape):
        raise ValueError("position_shift must be a contiguous int32 [num_seqs]")
    ks, vs, mem = k.stride(), v.stride(), _lib.ARGS
    try:
        mem.pack_rope(mem.buf, 0, *_lib.kv_fields(k_cache, v_cache, scaled),
                      *_lib.ragged_fields(T, cu_tokens, block_tables, context_lens, seq_ids,
                                          start_positions),
                      qp, k.data_ptr(), v.data_ptr(), op, _lib.dtype_code(k.dtype), Hq,
                      qs[0], qs[1], ks[0], ks[1], vs[0], vs[1], os_[0], os_[1],
                      0 if cos_sin is None else cos_sin.data_ptr(), pos, rot, interleaved,
                      _lib.dtype_code(ndt), 0 if q_norm is None else q_norm.data_ptr(),
                      0 if k_norm is None else k_norm.data_ptr(), eps)
    except (struct.error, OverflowError) as e:
        raise ValueError(f"rope_append: an argument is out of range ({e})") from None
    lib = _lib.load()
    if scaled or position_shift is not None:
        args = (mem.kv, _lib.scale_ptr(k_scale, k_cache, "k_scale"),
                _lib.scale_ptr(v_scale, k_cache, "v_scale"), mem.rg, mem.rope,
                _lib.ptr(position_shift))
        if _reserve is not None:
            _lib.check(lib.cvsa_rope_append_to_check(*args), "cvsa_rope_append_to")
            _reserve()
        _lib.check(lib.cvsa_rope_append_to(*args, _lib.ptr(dev_error), _lib.raw_stream(dev)),
                   "cvsa_rope_append_to")
        return out
    if _reserve is not None:
        _lib.check(lib.cvsa_rope_append_check(mem.kv, mem.rg, mem.rope), "cvsa_rope_append")
        _reserve()
    st = lib.cvsa_rope_append(mem.kv, mem.rg, mem.rope, _lib.ptr(dev_error),
                              _lib.raw_stream(dev))
    if st:
        _lib.check(st, "cvsa_rope_append")
    return out
