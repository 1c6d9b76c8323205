"""spmm_amd.attention -- attention under a sliding window with first keys that stay visible, its gradients, the form for
one new token over keys and values in pages, and the write of new rows into the pages (include/spmm_attn.h,
lib/libspmm_attn.so).

Beside ``spmm_amd.pipeline`` (SDDMM -> softmax -> SpMM under any CSR mask) these take the mask that long inputs use, a
band plus the first columns, as two numbers.  A query at position p sees key j if ``j <= p`` and (``window == 0`` or
``p - j < window`` or ``j < sinks``); the queries of a sequence are the last of its keys' positions.

Arguments are torch tensors on one HIP device, float32, float16 or bfloat16 alike, with the head width (1 to 128) as
their innermost, contiguous dimension and any other strides.  Work is ordered on ``stream`` (an integer hipStream_t; by
default the device's current stream), results and workspaces that a call allocates belong to that stream, and calls can
be captured in a graph.  What a call writes must not overlap what it reads.  There is no CPU path.

The calls are not recorded by autograd, and one that would lose a gradient is refused: outside ``torch.no_grad()`` their
operands may not require gradients.  To train, call ``window_attention`` and ``window_attention_backward`` in the two
methods of a ``torch.autograd.Function``, which run with gradients off; there are no second derivatives.
"""
from __future__ import annotations

import contextlib
import ctypes as C
import operator

import torch

from . import SpmmHipError, _open

F32, F16, BF16 = 1, 2, 3
MAX_DIM = 128
_DTYPES = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}


class _Desc(C.Structure):
    _fields_ = [("device", C.c_int32), ("dtype", C.c_int32), ("heads", C.c_int32), ("kv_heads", C.c_int32),
                ("dim", C.c_int32), ("window", C.c_int32), ("sinks", C.c_int32), ("scale", C.c_float),
                ("batch", C.c_int64), ("q_len", C.c_int64), ("k_len", C.c_int64), ("zero_rest", C.c_int32),
                ("reserved", C.c_int32)]


class _Rows(C.Structure):
    _fields_ = [("ptr", C.c_void_p), ("seq", C.c_int64), ("row", C.c_int64), ("head", C.c_int64)]


class _Pages(C.Structure):
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("pages", C.c_int64), ("page_rows", C.c_int64),
                ("k_page", C.c_int64), ("k_row", C.c_int64), ("k_head", C.c_int64),
                ("v_page", C.c_int64), ("v_row", C.c_int64), ("v_head", C.c_int64),
                ("table", C.c_void_p), ("table_cols", C.c_int64), ("table_stride", C.c_int64), ("lengths", C.c_void_p)]


def _bind(L: C.CDLL) -> C.CDLL:
    d, r, g, vp, i64 = C.POINTER(_Desc), C.POINTER(_Rows), C.POINTER(_Pages), C.c_void_p, C.c_int64
    L.spmm_attn_window.argtypes = [d, r, r, r, vp, vp, r, vp, vp]
    L.spmm_attn_window_work.argtypes = [d, C.c_int32, C.POINTER(C.c_size_t)]
    L.spmm_attn_window_grad.argtypes = [d, r, r, r, r, r, vp, vp, vp, r, r, r, vp, C.c_size_t, vp]
    L.spmm_attn_paged_work.argtypes = [d, i64, C.POINTER(C.c_size_t)]
    L.spmm_attn_paged.argtypes = [d, r, g, i64, r, vp, vp, C.c_size_t, vp]
    L.spmm_attn_append.argtypes = [d, r, r, vp, g, vp]
    L.spmm_attn_last_error_detail.restype = C.c_char_p
    return L


lib = _bind(_open("libspmm_attn.so"))


def _check(where: str, st: int) -> None:
    if st != 0:
        raise SpmmHipError(where, st, (lib.spmm_attn_last_error_detail() or b"").decode())


def _tensor(name: str, t, dtype=None, device: int | None = None, shape=None, contiguous: bool = False) -> tuple:
    """t is a tensor on a HIP device (the given one), of the given dtype and shape, its innermost dimension (or all of it)
    contiguous: its strides."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} is on {t.device}: there is no CPU path")
    if dtype is not None and t.dtype is not dtype:
        raise TypeError(f"{name} is {t.dtype}, expected {dtype}")
    if device is not None and t.get_device() != device:
        raise ValueError(f"{name} is on {t.device}, expected HIP device {device}")
    if shape is not None and t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    s = t.stride()
    if contiguous:
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
    elif s and s[-1] != 1 and t.shape[-1] > 1 and t.numel():
        raise ValueError(f"the innermost dimension of {name} must be contiguous")
    return s


def _lost(**operands) -> None:
    """Refuses operands whose gradient a call would lose."""
    for name, t in operands.items():
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{name} requires a gradient, which this call would lose: call it under torch.no_grad(), or in "
                             "the forward method of a torch.autograd.Function")


def _rows(t, s: tuple, packed: bool = False) -> _Rows:
    """[batch, rows, heads, d], or [rows, heads, d] with offsets, of strides s."""
    return _Rows(t.data_ptr(), 0, s[0], s[1]) if packed else _Rows(t.data_ptr(), s[0], s[1], s[2])


def _int(name: str, x, lo: int, hi: int = 2 ** 31 - 1) -> int:
    if isinstance(x, bool):
        raise TypeError(f"{name} must be an integer")
    x = operator.index(x)
    if not lo <= x <= hi:
        raise ValueError(f"{name} = {x} is not in {lo} .. {hi}")
    return x


def _place(device: int, stream):
    """(stream handle, context in which allocations belong to that stream, None where they do already)."""
    if stream is None:
        return torch._C._cuda_getCurrentRawStream(device), None
    return stream, torch.cuda.stream(_stream(device, stream))


def _stream(device: int, stream: int):
    """torch's stream of that handle.  0 is the null stream, of which ExternalStream would make a new one."""
    if isinstance(stream, bool) or not isinstance(stream, int):
        raise TypeError("stream must be an integer hipStream_t")
    return torch.cuda.ExternalStream(stream, device=device) if stream else torch.cuda.default_stream(device)


_HERE = contextlib.nullcontext()


def _desc(q, device: int, kv_heads: int, window, sinks, scale, batch: int, q_len: int, k_len: int, zero_rest: bool = False) -> _Desc:
    heads, dim = q.shape[-2:]
    dtype = _DTYPES.get(q.dtype)
    if dtype is None:
        raise TypeError(f"element type {q.dtype}: float32, float16 or bfloat16")
    if not 1 <= dim <= MAX_DIM:
        raise ValueError(f"head width {dim} is not in 1 .. {MAX_DIM}")
    if kv_heads < 1 or heads < 1 or heads % kv_heads:
        raise ValueError(f"{heads} heads are not a multiple of {kv_heads} key heads")
    return _Desc(device, dtype, heads, kv_heads, dim, _int("window", window, 0), _int("sinks", sinks, 0),
                 dim ** -0.5 if scale is None else scale, batch, q_len, k_len, zero_rest, 0)


def _window_operands(q, k, v, window, sinks, scale, cu_q, cu_k, zero_rest):
    """(packed, description, addresses of the offsets, rows of q, k, v, device, dtype)"""
    packed = cu_q is not None
    if not packed and cu_k is not None:
        raise ValueError("cu_k without cu_q")
    qs = _tensor("q", q)
    dev, dt = q.get_device(), q.dtype
    ks, vs = _tensor("k", k, dt, dev), _tensor("v", v, dt, dev)
    nd = 3 if packed else 4
    if len(qs) != nd or len(ks) != nd or len(vs) != nd:
        raise ValueError(f"q, k and v need {nd} dimensions: " + ("[rows, heads, d]" if packed else "[batch, rows, heads, d]"))
    qd, kd = q.shape, k.shape
    if kd != v.shape or kd[-1] != qd[-1] or (not packed and kd[0] != qd[0]):
        raise ValueError(f"q {tuple(qd)}, k {tuple(kd)} and v {tuple(v.shape)} do not fit")
    batch, pq, pk = qd[0], None, None
    if packed:
        cu_k = cu_q if cu_k is None else cu_k
        _tensor("cu_q", cu_q, torch.int32, dev, None, True)
        if cu_k is not cu_q:
            _tensor("cu_k", cu_k, torch.int32, dev, None, True)
        size = cu_q.shape
        if len(size) != 1 or size[0] < 1 or size != cu_k.shape:
            raise ValueError("cu_q and cu_k must be vectors of the number of sequences + 1")
        batch, pq, pk = size[0] - 1, cu_q.data_ptr(), cu_k.data_ptr()
    d = _desc(q, dev, kd[-2], window, sinks, scale, batch, qd[-3], kd[-3], zero_rest and packed)
    return packed, d, pq, pk, _rows(q, qs, packed), _rows(k, ks, packed), _rows(v, vs, packed), dev, dt


def window_attention(q, k, v, window: int = 0, sinks: int = 0, scale: float | None = None, cu_q=None, cu_k=None,
                     out=None, lse=None, stream: int | None = None):
    """Causal attention: (out, lse).

    q [batch, rows, heads, d], k and v [batch, key rows, key heads, d]; or, with int32 offsets ``cu_q`` and ``cu_k``
    ([sequences + 1], on the device; cu_k defaults to cu_q), [rows, heads, d] and [key rows, key heads, d].
    ``scale`` defaults to d ** -0.5.  out is like q, lse float32 with q's shape less its last dimension (the log of the sum
    of the exponentials, -inf where a query sees nothing).  With offsets, rows behind the last sequence are 0 in an out and
    -inf in an lse that the call allocates, and left as they are in one that is given."""
    whole = out is None and lse is None
    packed, d, pq, pk, qr, kr, vr, dev, dt = _window_operands(q, k, v, window, sinks, scale, cu_q, cu_k, whole)
    if q.requires_grad or k.requires_grad or v.requires_grad:
        _lost(q=q, k=k, v=v)
    fill = packed and not whole
    st, where = _place(dev, stream)
    with where or _HERE:
        if out is None:
            out = q.new_empty(q.shape)
            os = out.stride()
            if fill:
                out.zero_()
        else:
            os = _tensor("out", out, dt, dev, q.shape)
        if lse is None:
            lse = q.new_empty(q.shape[:-1], dtype=torch.float32)
            if fill:
                lse.fill_(float("-inf"))
        else:
            _tensor("lse", lse, torch.float32, dev, q.shape[:-1], True)
    _check("window_attention", lib.spmm_attn_window(d, qr, kr, vr, pq, pk, _rows(out, os, packed), lse.data_ptr(), st))
    return out, lse


def window_attention_backward(dout, q, k, v, out, lse, window: int = 0, sinks: int = 0, scale: float | None = None,
                              cu_q=None, cu_k=None, dq=None, dk=None, dv=None, stream: int | None = None):
    """Gradients (dq, dk, dv) of ``window_attention`` for the gradient ``dout`` of its out; out, lse: what it returned
    (for these keys, not joined with others'), the other arguments as they were.  With offsets, rows behind the last sequence are 0 in gradients that the call
    allocates and left as they are in those that are given."""
    whole = dq is None and dk is None and dv is None
    packed, d, pq, pk, qr, kr, vr, dev, dt = _window_operands(q, k, v, window, sinks, scale, cu_q, cu_k, whole)
    dr = _rows(dout, _tensor("dout", dout, dt, dev, q.shape), packed)
    if dout.requires_grad or q.requires_grad or k.requires_grad or v.requires_grad:
        _lost(dout=dout, q=q, k=k, v=v)
    outr = _rows(out, _tensor("out", out, dt, dev, q.shape), packed)
    _tensor("lse", lse, torch.float32, dev, q.shape[:-1], True)
    st, where = _place(dev, stream)
    need = C.c_size_t()
    _check("window_attention_backward", lib.spmm_attn_window_work(d, packed, need))
    with where or _HERE:
        res, rows = [], []
        for name, g, t in (("dq", dq, q), ("dk", dk, k), ("dv", dv, v)):
            if g is None:
                g = t.new_empty(t.shape)
                s = g.stride()
                if packed and not whole:
                    g.zero_()
            else:
                s = _tensor(name, g, dt, dev, t.shape)
            res.append(g)
            rows.append(_rows(g, s, packed))
        work = q.new_empty(need.value, dtype=torch.uint8)
    _check("window_attention_backward", lib.spmm_attn_window_grad(d, dr, qr, kr, vr, outr, lse.data_ptr(), pq, pk, *rows,
                                                                  work.data_ptr(), need.value, st))
    return tuple(res)


def _pages(k_pages, v_pages, page_table, lengths, dim: int, dt, dev: int, batch: int) -> _Pages:
    ks, vs = _tensor("k_pages", k_pages, dt, dev), _tensor("v_pages", v_pages, dt, dev)
    shape = k_pages.shape
    if len(ks) != 4 or shape != v_pages.shape or shape[3] != dim:
        raise ValueError(f"pages {tuple(shape)} and {tuple(v_pages.shape)}: [pages, rows, key heads, {dim}] expected")
    if shape[1] < 1:
        raise ValueError("pages without rows")
    ts = _tensor("page_table", page_table, torch.int32, dev)
    if len(ts) != 2 or page_table.shape[0] != batch:
        raise ValueError(f"page_table {tuple(page_table.shape)}: one row for each of {batch} sequences expected")
    _tensor("lengths", lengths, torch.int32, dev, (batch,), True)
    return _Pages(k_pages.data_ptr(), v_pages.data_ptr(), shape[0], shape[1], ks[0], ks[1], ks[2], vs[0], vs[1], vs[2],
                  page_table.data_ptr(), page_table.shape[1], ts[0], lengths.data_ptr())


def paged_attention(q, k_pages, v_pages, page_table, lengths, window: int = 0, sinks: int = 0,
                    scale: float | None = None, max_length: int | None = None, out=None, lse=None,
                    stream: int | None = None):
    """Attention of one new token a sequence, the last of its ``lengths`` positions in the cache: (out, lse).

    q [batch, heads, d]; k_pages, v_pages [pages, rows of a page, key heads, d]; page_table int32 [batch, columns]: page
    of positions 0 .. rows - 1, and so on; lengths int32 [batch], the new token counted (its row is written by
    ``cache_append`` before).  A sequence of length 0 gets out 0 and lse -inf.  ``max_length``: an upper bound of the
    lengths (by default what the table can hold); a tight one gives the better split of the work.  A sequence whose
    visible positions need a page that is not there, or whose length is negative, above max_length or above what the table
    can hold, gets NaN."""
    qs = _tensor("q", q)
    if len(qs) != 3:
        raise ValueError(f"q {tuple(q.shape)}: [batch, heads, d] expected")
    dev, dt, batch = q.get_device(), q.dtype, q.shape[0]
    pages = _pages(k_pages, v_pages, page_table, lengths, q.shape[2], dt, dev, batch)
    if q.requires_grad or k_pages.requires_grad or v_pages.requires_grad:
        _lost(q=q, k_pages=k_pages, v_pages=v_pages)
    d = _desc(q, dev, k_pages.shape[2], window, sinks, scale, batch, 1, 0)
    room = min(pages.table_cols * pages.page_rows, 2 ** 30 - 1)
    longest = room if max_length is None else min(_int("max_length", max_length, 0), room)
    st, where = _place(dev, stream)
    need = C.c_size_t()
    _check("paged_attention", lib.spmm_attn_paged_work(d, longest, need))
    with where or _HERE:
        if out is None:
            out = q.new_empty(q.shape)
            os = out.stride()
        else:
            os = _tensor("out", out, dt, dev, q.shape)
        if lse is None:
            lse = q.new_empty(q.shape[:-1], dtype=torch.float32)
        else:
            _tensor("lse", lse, torch.float32, dev, q.shape[:-1], True)
        work = q.new_empty(need.value, dtype=torch.uint8) if need.value else None
    _check("paged_attention", lib.spmm_attn_paged(
        d, _Rows(q.data_ptr(), qs[0], 0, qs[1]), pages, longest, _Rows(out.data_ptr(), os[0], 0, os[1]), lse.data_ptr(),
        work.data_ptr() if work is not None else None, need.value, st))
    return out, lse


def cache_append(k, v, k_pages, v_pages, page_table, lengths, cu=None, stream: int | None = None) -> None:
    """Write the keys and values of new tokens into the cache: those of sequence b go to its last positions before
    ``lengths[b]``.  k and v [batch, key heads, d], one token a sequence (none for a sequence of length 0), or, with
    int32 offsets ``cu`` [batch + 1] on the device, [rows, key heads, d].  Rows whose page is not there are dropped, and
    all rows of a sequence whose length is above what the table can hold.  A page that is written must belong to one
    sequence only."""
    ks = _tensor("k", k)
    dev, dt = k.get_device(), k.dtype
    vs = _tensor("v", v, dt, dev, k.shape)
    if len(ks) != 3:
        raise ValueError(f"k {tuple(k.shape)}: [rows, key heads, d] expected")
    rows, heads, dim = k.shape
    batch, pc = rows, None
    if cu is not None:
        _tensor("cu", cu, torch.int32, dev, None, True)
        if cu.ndim != 1 or cu.shape[0] < 1:
            raise ValueError("cu must be a vector of the number of sequences + 1")
        batch, pc = cu.shape[0] - 1, cu.data_ptr()
    pages = _pages(k_pages, v_pages, page_table, lengths, dim, dt, dev, batch)
    if k_pages.shape[2] != heads:
        raise ValueError(f"{heads} key heads, the pages have {k_pages.shape[2]}")
    if k.requires_grad or v.requires_grad or k_pages.requires_grad or v_pages.requires_grad:
        _lost(k=k, v=v, k_pages=k_pages, v_pages=v_pages)
    _check("cache_append", lib.spmm_attn_append(_desc(k, dev, heads, 0, 0, 1.0, batch, rows, 0), _rows(k, ks, True),
                                                _rows(v, vs, True), pc, pages, _place(dev, stream)[0]))
