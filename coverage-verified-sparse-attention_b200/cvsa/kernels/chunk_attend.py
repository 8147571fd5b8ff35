"""Attention of a ragged batch of new tokens over the paged cache.

`chunk_attention` serves a prompt, a chunk of one, drafted tokens to verify,
or one token for each sequence, in any mix: sequence b owns tokens
cu_tokens[b]..cu_tokens[b + 1] of q, and they attend to everything the
sequence has cached up to themselves (csrc/chunk_attend_tc.cu,
csrc/chunk_attend.cu). The reference computes prompts in the model library
(eval/latency_benchmark.py:376-420) and has no counterpart.
"""

import struct
from typing import Optional

import torch

from cvsa import _lib

_ALL = 2 ** 31 - 1  # keys: more than a sequence can hold
_ws_bytes = {}  # workspace bytes by (device, head_dim, dtypes)


def chunk_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                    block_tables: torch.Tensor, context_lens: torch.Tensor,
                    cu_tokens: torch.Tensor, causal: bool = True, window: int = 0,
                    scale: Optional[float] = None, seq_ids: Optional[torch.Tensor] = None,
                    start_positions: Optional[torch.Tensor] = None,
                    out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None,
                    dev_error: Optional[torch.Tensor] = None, *,
                    k_scale: Optional[torch.Tensor] = None,
                    v_scale: Optional[torch.Tensor] = None,
                    check_only: bool = False) -> torch.Tensor:
    """softmax(scale q K^T) V per new token and query head, [T, H_q, D] in q's dtype.

    q [T, H_q, D]; the pools, tables [num_seqs, max_pages] and lengths
    [num_seqs] are those of the decode step, with the new tokens already in
    (`rope_append`); scale defaults to D^-0.5. causal: a token sees its
    sequence up to itself, of which the last `window` keys if window > 0;
    otherwise all of it. lse, if given, is a float32 [T, H_q] tensor to fill
    with the log-sum-exp of each row's scaled scores (for a merge with
    attention over other keys). A row that sees no key gives 0 and -inf, as
    does a sequence that was refused or whose table row is out of range. Rows no sequence
    owns (padding, offsets out of range) are not written.
    k_scale, v_scale [num_blocks, H_kv]: the scales of an 8-bit cache
    (float8_e4m3fn pools, any q dtype; a value is its code times its page's scale).
    check_only raises what the call would be refused with and returns the output
    unfilled, without a launch.

    Threads may call on one stream. A captured call's workspace is memory of its
    graph's pool: graphs of different pools may be replayed at the same time.
    """
    dev = _lib.same_device(q, k_cache, v_cache, block_tables, context_lens, cu_tokens, seq_ids,
                           start_positions, out, lse, dev_error, k_scale, v_scale)
    if dev != torch.cuda.current_device():  # a launch goes to the current device
        with torch.cuda.device(dev):
            return chunk_attention(q, k_cache, v_cache, block_tables, context_lens, cu_tokens,
                                   causal, window, scale, seq_ids, start_positions, out, lse,
                                   dev_error, k_scale=k_scale, v_scale=v_scale,
                                   check_only=check_only)
    q = _lib.token_rows(q, "q")
    T, Hq, D = shape = q.shape
    if k_cache.dim() != 4 or k_cache.shape[3] != D:
        raise ValueError("q's head_dim does not match the cache")
    if out is None:
        out = q.new_empty(shape)
    elif out.shape != shape or out.dtype != q.dtype or out.stride(2) != 1:
        raise ValueError("out must have q's shape and dtype and contiguous rows")
    if lse is not None and (lse.shape != (T, Hq) or lse.dtype != torch.float32
                            or not lse.is_contiguous()):
        raise ValueError("lse must be a contiguous float32 [T, H_q]")
    scaled = k_scale is not None
    if scaled != (v_scale is not None):
        raise ValueError("k_scale and v_scale go together")
    qs, os_, mem = q.stride(), out.stride(), _lib.ARGS
    try:
        mem.pack_chunk(mem.buf, 0, *_lib.kv_fields(k_cache, v_cache, scaled),
                       *_lib.ragged_fields(T, cu_tokens, block_tables, context_lens, seq_ids,
                                           start_positions),
                       q.data_ptr(), out.data_ptr(), 0 if lse is None else lse.data_ptr(),
                       _lib.dtype_code(q.dtype), Hq, qs[0], qs[1], os_[0], os_[1],
                       D ** -0.5 if scale is None else scale, causal,
                       window if window < _ALL else _ALL)
    except (struct.error, OverflowError) as e:
        raise ValueError(f"chunk_attention: an argument is out of range ({e})") from None
    lib, stream = _lib.load(), _lib.raw_stream(dev)
    head, call = (mem.kv,), "cvsa_chunk_attend"
    if scaled:
        head = (mem.kv, _lib.scale_ptr(k_scale, k_cache, "k_scale"),
                _lib.scale_ptr(v_scale, k_cache, "v_scale"))
        call = "cvsa_chunk_attend_q8"
    if check_only:
        _lib.check(getattr(lib, call + "_check")(*head, mem.rg, mem.chunk), call)
        return out
    launch = getattr(lib, call)
    # the size depends on the head layout alone; 0 for what the call will refuse
    key = (dev, D, q.dtype, k_cache.dtype)
    nbytes = _ws_bytes.get(key)
    if nbytes is None:
        nbytes = getattr(lib, call + "_workspace_size")(*head, mem.rg, mem.chunk)
        if nbytes:
            _ws_bytes[key] = nbytes
    if nbytes and torch.cuda.is_current_stream_capturing():
        # memory of the graph, like its other tensors
        buf = torch.empty(nbytes + 256, dtype=torch.uint8, device=q.device)
        st = launch(*head, mem.rg, mem.chunk, _lib.ptr(dev_error),
                    buf.data_ptr() + (-buf.data_ptr()) % 256, nbytes, stream)
    else:
        with _lib.WORKSPACE.lock:
            ws = _lib.WORKSPACE.address(nbytes, q.device, stream, "chunk") if nbytes else None
            st = launch(*head, mem.rg, mem.chunk, _lib.ptr(dev_error), ws, nbytes, stream)
    if st:
        _lib.check(st, call)
    return out
