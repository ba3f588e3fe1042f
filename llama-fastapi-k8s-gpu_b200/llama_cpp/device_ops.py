"""Operators over device tensors that the caller owns: appending to a paged cache, attention of a batch over a shared prefix, log probabilities.

They are the C entry points b2_kv_append, b2_attention_shared_prefix and b2_token_logprobs (include/b200_gguf.h says what each computes), for hosts that keep
caches and logits of their own: score or continue several answers to one prompt by appending every answer's keys and values to pages of its own,
attending to the prompt's pages once for all of them, and reading the log probabilities off the logits.

A tensor is a torch tensor on a CUDA device, or anything with its `data_ptr()`, `shape`, `stride()`, `dtype`, `get_device()` and `is_contiguous()` (this
package does not import torch itself); results go into tensors of the caller's, nothing is allocated. `stream` is a stream object with `cuda_stream`, its
handle, or None for the default stream; the call only enqueues work there, so tensors that other streams use must be ordered by the caller. Wrong
shapes, types or devices raise ValueError before anything is enqueued. Waits inside the attention kernels are bounded: `error(device)` says
whether one ran out since it was last asked, after which results are not to be used.

A call is made by native code where that has been built (csrc/py_tensors.cpp: a single token's call is a few microseconds of device time, and reading a dozen
tensors in Python takes more). What it does not take comes back here, where the same checks say what is wrong: one condition a tensor, and what was
wrong with it is only looked for once it fails.
"""
from __future__ import annotations

import ctypes
import math
import struct

from . import _cabi
from ._cabi import check

_TYPES = {"float32": _cabi.B2_TYPE_F32, "float16": _cabi.B2_TYPE_F16, "bfloat16": _cabi.B2_TYPE_BF16, "int32": _cabi.B2_TYPE_I32}
_F32, _F16, _BF16, _I32 = (_TYPES[n] for n in ("float32", "float16", "bfloat16", "int32"))
_NAMES = {v: k for k, v in _TYPES.items()}
_ROWS, _CACHE = (_F32, _F16, _BF16), (_F16, _BF16)
_LAYOUTS = {"pairs": _cabi.B2_ROTATE_PAIRS, "halves": _cabi.B2_ROTATE_HALVES}


def _entry(name):
    """The native call and the address of the C entry point that it is to call, or two None."""
    calls = _cabi.load_calls()
    return (None, None) if calls is None else (getattr(calls, name), ctypes.cast(getattr(_cabi.load_library(), "b2_" + name), ctypes.c_void_p).value)


_entries = {}        # name -> _entry(name), once it has been called


class _Codes(dict):
    """dtype object -> type id (-1: none of ours); filled as dtypes are met."""

    def __missing__(self, dtype):
        code = self[dtype] = _TYPES.get(str(dtype).rpartition(".")[2], -1)
        calls = _cabi.load_calls()
        if calls is not None and code >= 0:
            calls.add_type(dtype, code)
        return code


_code = _Codes()


def _packer(structure):
    """The C structure's fields as bytes in one call (a ctypes structure takes twice as long to fill)."""
    letter = {ctypes.c_void_p: "P", ctypes.c_int64: "q", ctypes.c_int32: "i", ctypes.c_float: "f"}
    p = struct.Struct("@" + "".join(letter[t] for _, t in structure._fields_) + "0q")
    assert p.size == ctypes.sizeof(structure)
    return p.pack


_ragged_pages, _kv_append, _shared_prefix = (_packer(s) for s in (_cabi.B2RaggedPages, _cabi.B2KvAppend, _cabi.B2SharedPrefix))


def _wrong(what, t, shape, types, device, dense):
    """Raises what is wrong with a tensor that failed its check. `shape`: None where a length is free."""
    names = " or ".join(_NAMES[c] for c in types)
    if _code[t.dtype] not in types:
        raise ValueError(f"{what}: dtype {t.dtype}, expected {names}")
    if t.get_device() < 0:
        raise ValueError(f"{what} is not on a CUDA device")
    if t.get_device() != device:
        raise ValueError(f"{what} is on CUDA device {t.get_device()}, expected {device}")
    if len(t.shape) != len(shape) or any(e is not None and e != n for e, n in zip(shape, t.shape)):
        raise ValueError(f"{what}: shape {tuple(t.shape)}, expected ({', '.join('*' if e is None else str(e) for e in shape)})")
    raise ValueError(f"{what} must be contiguous" if dense else f"{what}: the last dimension must be contiguous")


def _dense(what, t, shape, types, device):
    """Pointer of a contiguous tensor of exactly this shape."""
    if t.shape != shape or _code[t.dtype] not in types or t.get_device() != device or not t.is_contiguous():
        _wrong(what, t, shape, types, device, True)
    return t.data_ptr()


def _rows(what, t, shape, types, device):
    """Pointer and strides of a tensor of this shape whose last dimension is contiguous."""
    stride = t.stride()
    if t.shape != shape or _code[t.dtype] not in types or t.get_device() != device or (stride[-1] != 1 and shape[-1] > 1):
        _wrong(what, t, shape, types, device, False)
    return t.data_ptr(), stride


def _begin(what, t, dims, types):
    """Device, shape and type of a call's first tensor."""
    device, shape, code = t.get_device(), t.shape, _code[t.dtype]
    if device < 0 or len(shape) != dims or code not in types:
        _wrong(what, t, (None,) * dims, types, device, False)
    return device, shape, code


def _where(n_rows, k_pool, v_pool, pages, row_start, lengths, device):
    """Pointers of the pools, their shape and type, and the packed b2_ragged_pages"""
    if len(lengths.shape) != 1 or len(pages.shape) != 2:
        raise ValueError(f"lengths must have one dimension and pages two, not {tuple(lengths.shape)} and {tuple(pages.shape)}")
    _, pool, cache = _begin("k_pool", k_pool, 4, _CACHE)
    n_seqs, width = pages.shape
    table, stride = _rows("pages", pages, (n_seqs, width), (_I32,), device)
    kp, vp = _dense("k_pool", k_pool, pool, (cache,), device), _dense("v_pool", v_pool, pool, (cache,), device)
    start, held = _dense("row_start", row_start, (n_seqs + 1,), (_I32,), device), _dense("lengths", lengths, (n_seqs,), (_I32,), device)
    return kp, vp, pool, cache, _ragged_pages(start, held, table, stride[0] if n_seqs > 1 else width, pool[0], width, n_seqs, n_rows, pool[2])


def kv_append(k, v, k_pool, v_pool, pages, row_start, lengths, *, freqs=None, layout="pairs", first_pos=0, amplitude=1.0, q=None, q_out=None, stream=None):
    """Append rows of keys and values to a paged cache, rotated by their positions (b2_kv_append).

    k, v [rows, kv heads, dim] (float32, float16 or bfloat16); pools [pages, kv heads, page tokens, dim] (float16 or bfloat16); pages [sequences, n],
    row_start [sequences + 1], lengths [sequences] int32: rows row_start[s] .. row_start[s + 1] - 1 are the newest of sequence s's lengths[s] tokens.
    `freqs` (float32 [rotated entries / 2], None: no rotation) are radians per position, `first_pos` the position of a sequence's first own token.
    `q` [rows, heads, dim] of k's type is rotated into `q_out` of the cache's type."""
    stream = getattr(stream, "cuda_stream", stream)
    call, entry = _entries.get("kv_append") or _entries.setdefault("kv_append", _entry("kv_append"))
    if call is not None and layout in _LAYOUTS:
        code = call(entry, k, v, k_pool, v_pool, pages, row_start, lengths, freqs, q, q_out, _LAYOUTS[layout], first_pos, amplitude, stream)
        if code is not None:
            if code:
                check(code, "b2_kv_append")
            return
    device, shape, rows = _begin("k", k, 3, _ROWS)
    n, n_kv, dim = shape
    kp, vp, pool, cache, where = _where(n, k_pool, v_pool, pages, row_start, lengths, device)
    if n_kv != pool[1] or dim != pool[3]:
        raise ValueError(f"k {tuple(shape)} and pools {tuple(pool)} do not go together")
    pk, sk = _rows("k", k, shape, (rows,), device)
    pv, sv = _rows("v", v, shape, (rows,), device)
    if layout not in _LAYOUTS:
        raise ValueError(f"layout must be 'pairs' or 'halves', not {layout!r}")
    if (q is None) != (q_out is None):
        raise ValueError("q and q_out go together")
    pq = po = heads = 0
    sq = so = (0, 0)
    if q is not None:
        shape_q = q.shape
        if len(shape_q) != 3 or shape_q[0] != n or shape_q[2] != dim:
            raise ValueError(f"q {tuple(shape_q)} and k {tuple(shape)} do not go together")
        pq, sq = _rows("q", q, shape_q, (rows,), device)
        po, so = _rows("q_out", q_out, shape_q, (cache,), device)
        heads = shape_q[1]
    pf, rot = 0, 0
    if freqs is not None:
        pf, rot = _dense("freqs", freqs, freqs.shape if len(freqs.shape) == 1 else (None,), (_F32,), device), 2 * freqs.shape[0]
    args = _kv_append(pk, pv, pq, kp, vp, po, pf, sk[0], sk[1], sv[0], sv[1], sq[0], sq[1], so[0], so[1], first_pos, rows, cache, heads, n_kv, dim, rot,
                      _LAYOUTS[layout], amplitude)
    check(_cabi.load_library().b2_kv_append(device, where, args, stream), "b2_kv_append")


def attention_shared_prefix_workspace(rows, n_head, n_kv, head_dim) -> int:
    """Bytes of workspace that attention_shared_prefix needs for so many rows, whatever the lengths."""
    for name, n in (("rows", rows), ("n_head", n_head), ("n_kv", n_kv), ("head_dim", head_dim)):
        if not 0 <= n < 1 << 31:                                 # (ctypes would drop the upper bits)
            raise ValueError(f"{name} must be a number of 31 bits, not {n}")
    out = ctypes.c_int64()
    check(_cabi.load_library().b2_attention_shared_prefix_workspace(rows, n_head, n_kv, head_dim, ctypes.byref(out)), "b2_attention_shared_prefix_workspace")
    return out.value


def attention_shared_prefix(q, k_pool, v_pool, prefix_pages, n_prefix, pages, row_start, lengths, out, workspace, *, max_rows=None, scale=None, stream=None):
    """Attention of a ragged batch whose sequences share their first `n_prefix` tokens (b2_attention_shared_prefix).

    q, out [rows, heads, dim] and the pools [pages, kv heads, page tokens, dim] all float16 or all bfloat16; prefix_pages [n], pages [sequences, m],
    row_start, lengths int32 as for kv_append: lengths count a sequence's own tokens, those behind the prefix. `workspace`: a contiguous tensor of at
    least attention_shared_prefix_workspace bytes, which no other call on another stream uses meanwhile (None when n_prefix is 0). `max_rows`: most
    rows of a sequence (None: all rows may be one sequence's; 1 for a batched step of single tokens is much faster than leaving it open)."""
    stream = getattr(stream, "cuda_stream", stream)
    call, entry = _entries.get("attention_shared_prefix") or _entries.setdefault("attention_shared_prefix", _entry("attention_shared_prefix"))
    if call is not None:
        code = call(entry, q, k_pool, v_pool, pages, row_start, lengths, prefix_pages, n_prefix, out, workspace, max_rows, scale, stream)
        if code is not None:
            if code:
                check(code, "b2_attention_shared_prefix")
            return
    device, shape, kind = _begin("q", q, 3, _CACHE)
    n, heads, dim = shape
    kp, vp, pool, cache, where = _where(n, k_pool, v_pool, pages, row_start, lengths, device)
    if cache != kind:
        raise ValueError(f"q is {_NAMES[kind]}, the cache {_NAMES[cache]}")
    if dim != pool[3] or pool[1] == 0 or heads % pool[1]:
        raise ValueError(f"q {tuple(shape)} and pools {tuple(pool)} do not go together")
    pq, sq = _rows("q", q, shape, (kind,), device)
    po, so = _rows("out", out, shape, (kind,), device)
    pp = pw = size = 0
    if n_prefix:
        held = prefix_pages.shape
        pp = _dense("prefix_pages", prefix_pages, held if len(held) == 1 else (None,), (_I32,), device)
        if n_prefix < 0 or n_prefix > held[0] * pool[2]:
            raise ValueError(f"a prefix of {n_prefix} tokens does not fit {held[0]} pages of {pool[2]}")
        if workspace is None or workspace.get_device() != device or not workspace.is_contiguous():
            raise ValueError("workspace must be a contiguous tensor on the same device")
        pw, size = workspace.data_ptr(), workspace.nbytes
    args = _shared_prefix(pq, kp, vp, pp, po, pw, size, sq[0], sq[1], so[0], so[1], n_prefix, max(1, n) if max_rows is None else max_rows, heads, pool[1], dim,
                          kind, 1.0 / math.sqrt(dim) if scale is None else scale)
    check(_cabi.load_library().b2_attention_shared_prefix(device, where, args, stream), "b2_attention_shared_prefix")


def token_logprobs(logits, tokens=None, logprob=None, entropy=None, top_logprob=None, top_id=None, *, stream=None):
    """Log probabilities of `tokens` (int32 [rows]), entropy, and the most likely tokens of logits [rows, vocab] (b2_token_logprobs).

    logits float32, float16 or bfloat16; logprob, entropy float32 [rows]; top_logprob float32 and top_id int32 [rows, n], n <= 64. A result whose tensor is None is
    left out."""
    stream = getattr(stream, "cuda_stream", stream)
    call, entry = _entries.get("token_logprobs") or _entries.setdefault("token_logprobs", _entry("token_logprobs"))
    if call is not None:
        code = call(entry, logits, tokens, logprob, entropy, top_logprob, top_id, stream)
        if code is not None:
            if code:
                check(code, "b2_token_logprobs")
            return
    device, shape, kind = _begin("logits", logits, 2, _ROWS)
    n, vocab = shape
    p, stride = _rows("logits", logits, shape, (kind,), device)
    pt = pl = pe = ptl = pti = None
    n_top = 0
    if (tokens is None) != (logprob is None):
        raise ValueError("tokens and logprob go together")
    if tokens is not None:
        pt, pl = _dense("tokens", tokens, (n,), (_I32,), device), _dense("logprob", logprob, (n,), (_F32,), device)
    if entropy is not None:
        pe = _dense("entropy", entropy, (n,), (_F32,), device)
    if (top_logprob is None) != (top_id is None):
        raise ValueError("top_logprob and top_id go together")
    if top_id is not None:
        if len(top_id.shape) != 2:
            _wrong("top_id", top_id, (n, None), (_I32,), device, True)
        n_top = top_id.shape[1]
        pti, ptl = _dense("top_id", top_id, (n, n_top), (_I32,), device), _dense("top_logprob", top_logprob, (n, n_top), (_F32,), device)
    check(_cabi.load_library().b2_token_logprobs(device, p, kind, stride[0] if n > 1 else vocab, n, vocab, pt, pl, pe, n_top, ptl, pti,
                                                 stream), "b2_token_logprobs")


def error(device) -> int:
    """Code of the first wait of attention_shared_prefix's kernels that ran out on this CUDA device since the last time that this was asked (0: none;
    b2_device_op_error): results of the calls in between are not to be used. Waits for all work on the device; not while a stream is being captured."""
    code = ctypes.c_uint32()
    check(_cabi.load_library().b2_device_op_error(device, ctypes.byref(code)), "b2_device_op_error")
    return code.value
