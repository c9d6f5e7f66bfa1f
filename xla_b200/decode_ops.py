"""Host-side front end of the decode-step operators: the dot with 4-bit weights, the append to the
8-bit paged cache of keys and values, and the attention over it.

They are custom calls like the scaled dots of `scaled_dot`: a `*Call` is one call site, bound to its
operand and result buffers and run stage by stage through the FFI, and each function beside it builds
such a site for torch tensors, runs it on the current stream of their device and drops it.  A program
that repeats a call keeps the site and uses `execute`; a recorded (CUDA graph) call wants the site, too,
with its buffers kept alive for the replays.
"""

from __future__ import annotations

from typing import Optional, Sequence

from . import _native
from .scaled_dot import (INVALID_ARGUMENT, S4, U4, Epilogue, FfiCall, XlaFfiError, _current_stream_and_device,
                         _torch)

TARGET_W4 = "b200$dot$w4"
TARGET_APPEND = "b200$kv_cache$append"
TARGET_ATTENTION = "b200$paged_attention$kv8"


class DotW4Call(FfiCall):
    """A `b200$dot$w4` call site: operands x [m, k], w u8[n, k / 2], scale [n, k / group], [zero u8[n, k / group]
    iff weight_type is U4], [bias [n] iff bias]; results D [m, n], [workspace].  The low four bits of a byte
    of w hold the even k."""

    def __init__(self, operands: Sequence, results: Sequence, *, weight_type: int = S4, bias: bool = False):
        super().__init__(TARGET_W4, operands, results, {
            "weight_type": ("i32", int(weight_type)),
            "epilogue": ("i32", int(Epilogue.BIAS if bias else Epilogue.DEFAULT)),
        })


class KvCacheAppendCall(FfiCall):
    """A `b200$kv_cache$append` call site: operands k_new, v_new [batch, new_tokens, kv_heads, head_dim], k_pages,
    v_pages [num_pages, kv_heads, page_tokens, head_dim], k_scale, v_scale f32[num_pages, kv_heads], page_table
    s32[batch, width], seq_lens s32[batch], [new_lens s32[batch]]; results k_pages, v_pages, k_scale, v_scale,
    in the operands' own buffers."""

    def __init__(self, operands: Sequence, results: Sequence):
        super().__init__(TARGET_APPEND, operands, results, {})


class PagedAttentionKv8Call(FfiCall):
    """A `b200$paged_attention$kv8` call site: operands q [batch, new_tokens, heads, head_dim], then the cache, table
    and lengths of `KvCacheAppendCall`; results out (as q), [lse f32[batch, new_tokens, heads] iff emit_lse],
    workspace s8[`paged_attention_workspace_bytes`]."""

    def __init__(self, operands: Sequence, results: Sequence, *, softmax_scale: float, window: int = 0, emit_lse: bool = False):
        super().__init__(TARGET_ATTENTION, operands, results, {
            "softmax_scale": float(softmax_scale), "window": int(window), "emit_lse": bool(emit_lse),
        })


def _run(call: FfiCall, tensors: Sequence) -> None:
    torch = _torch()
    try:
        device = tensors[0].device
        if device.type != "cuda" or any(t.device != device for t in tensors):
            raise XlaFfiError(INVALID_ARGUMENT, "all operands must be on one CUDA device")
        with torch.cuda.device(device):
            stream, index = _current_stream_and_device(tensors[0])
            call.run(stream, index)
    finally:
        call.close()


def dot_w4(x, w, scale, *, zero=None, bias=None, out_dtype=None, out=None):
    """x [m, k] times the transpose of 4-bit weights: out[m, n] = sum_k x[m, k] (w[n, k] - zero[n, k / group])
    scale[n, k / group] + bias[n].

    w is uint8 [n, k / 2], the even k in a byte's low four bits.  Without `zero` the weights are two's
    complement (-8 .. 7), with it (uint8 [n, k / group], low four bits) they are 0 .. 15.  The group size is
    k divided by scale's columns: 32, 64 or a multiple of 128.  m is at most 64.  The result has x's type, or float32
    with `out_dtype`."""
    torch = _torch()
    d = out if out is not None else torch.empty((x.shape[0], w.shape[0]), dtype=out_dtype or x.dtype, device=x.device)
    operands = [x, w, scale] + [t for t in (zero, bias) if t is not None]
    call = DotW4Call(operands, [d], weight_type=S4 if zero is None else U4, bias=bias is not None)
    _run(call, operands + [d])
    return d


def kv_cache_append(k_new, v_new, k_pages, v_pages, k_scale, v_scale, page_table, seq_lens, *, new_lens=None):
    """Rounds new keys and values [batch, new_tokens, kv_heads, head_dim] to the cache's 8-bit type and stores them at
    positions seq_lens - new_lens onwards of their sequences; the pages and scales are updated in place.

    seq_lens counts the tokens after the call, new_lens (all of new_tokens where it is not given) those of them
    that the call brings.  A page's scale is the least power of two that holds its new values, and no smaller than
    before where the page has earlier tokens; their codes are rounded to it again where it grows."""
    cache = [k_pages, v_pages, k_scale, v_scale]
    operands = [k_new, v_new] + cache + [page_table, seq_lens] + ([new_lens] if new_lens is not None else [])
    _run(KvCacheAppendCall(operands, cache), operands)


def paged_attention_workspace_bytes(batch: int, new_tokens: int, heads: int, kv_heads: int, head_dim: int) -> int:
    """Bytes of scratch that one attention call of this size needs."""
    return int(_native.product.b200sd_paged_attention_workspace_bytes(batch, new_tokens, heads, kv_heads, head_dim))


def paged_attention_kv8(q, k_pages, v_pages, k_scale, v_scale, page_table, seq_lens, *, new_lens=None,
                        softmax_scale: Optional[float] = None, window: int = 0, return_lse: bool = False, out=None,
                        workspace=None):
    """Attention of each sequence's last new_lens tokens over its pages, themselves included; returns the
    output, or (output, lse) with `return_lse`.

    q is [batch, new_tokens, heads, head_dim]; query i of sequence b stands at position p = seq_lens[b] -
    new_lens[b] + i and sees the positions up to p, the last `window` of them where window > 0.  Rows that see
    nothing get zeros and an lse of -inf.  softmax_scale is head_dim ** -0.5 where it is not given."""
    torch = _torch()
    batch, new, heads, dim = q.shape
    scale = dim ** -0.5 if softmax_scale is None else softmax_scale
    o = out if out is not None else torch.empty_like(q)
    lse = torch.empty((batch, new, heads), dtype=torch.float32, device=q.device) if return_lse else None
    if workspace is None:
        workspace = torch.empty(paged_attention_workspace_bytes(batch, new, heads, k_pages.shape[1], dim), dtype=torch.int8, device=q.device)
    operands = [q, k_pages, v_pages, k_scale, v_scale, page_table, seq_lens] + ([new_lens] if new_lens is not None else [])
    results = [o] + ([lse] if return_lse else []) + [workspace]
    _run(PagedAttentionKv8Call(operands, results, softmax_scale=scale, window=window, emit_lse=return_lse), operands + results)
    return (o, lse) if return_lse else o
