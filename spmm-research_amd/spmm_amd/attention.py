"""spmm_amd.attention -- attention under a sliding window with first keys that stay visible, its gradients, the form for
one new token over keys and values in pages, and the write of new rows into the pages (include/spmm_attn.h,
lib/libspmm_attn.so).

Beside ``spmm_amd.pipeline`` (SDDMM -> softmax -> SpMM under any CSR mask) these take the mask that long inputs use, a
band plus the first columns, as two numbers.  A query at position p sees key j if ``j <= p`` and (``window == 0`` or
``p - j < window`` or ``j < sinks``); the queries of a sequence are the last of its keys' positions.

Arguments are torch tensors on one HIP device, float32, float16 or bfloat16 alike, with the head width (1 to 128) as
their innermost, contiguous dimension and any other strides.  Work is ordered on ``stream`` (an integer hipStream_t; by
default the device's current stream), results and workspaces that a call allocates belong to that stream, and calls can
be captured in a graph.  There is no CPU path.
"""
from __future__ import annotations

import contextlib
import ctypes as C

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


def _tensor(name: str, t, like=None, shape=None, dtype=None, contiguous=False):
    """t is a tensor on a HIP device, of like's device and dtype, of the given shape, its rows contiguous."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch tensor")
    if t.device.type != "cuda":
        raise ValueError(f"{name} is on {t.device}: there is no CPU path")
    want = dtype if dtype is not None else like.dtype if like is not None else None
    if want is not None and t.dtype != want:
        raise TypeError(f"{name} is {t.dtype}, expected {want}")
    if like is not None and t.device != like.device:
        raise ValueError(f"{name} is on {t.device}, expected {like.device}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if contiguous and not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if not contiguous and t.ndim and t.shape[-1] > 1 and t.stride(-1) != 1 and t.numel():
        raise ValueError(f"the innermost dimension of {name} must be contiguous")
    return t


def _rows(t, packed: bool = False) -> _Rows:
    """[batch, rows, heads, d], or [rows, heads, d] with offsets."""
    s = t.stride()
    return _Rows(t.data_ptr(), 0, s[0], s[1]) if packed else _Rows(t.data_ptr(), s[0], s[1], s[2])


def _int(name: str, x, lo: int, hi: int = 2 ** 31 - 1) -> int:
    if isinstance(x, bool) or not isinstance(x, int):
        raise TypeError(f"{name} must be an integer")
    if not lo <= x <= hi:
        raise ValueError(f"{name} = {x} is not in {lo} .. {hi}")
    return x


def _place(t, stream):
    """(stream handle, context in which allocations belong to that stream)."""
    if stream is None:
        return torch.cuda.current_stream(t.device).cuda_stream, contextlib.nullcontext()
    if isinstance(stream, bool) or not isinstance(stream, int):
        raise TypeError("stream must be an integer hipStream_t")
    return stream, torch.cuda.stream(torch.cuda.ExternalStream(stream, device=t.device))


def _desc(q, kv_heads: int, window, sinks, scale, batch: int, q_len: int, k_len: int, zero_rest: bool = False) -> _Desc:
    heads, dim = q.shape[-2], q.shape[-1]
    if q.dtype not in _DTYPES:
        raise TypeError(f"element type {q.dtype}: float32, float16 or bfloat16")
    if not 1 <= dim <= MAX_DIM:
        raise ValueError(f"head width {dim} is not in 1 .. {MAX_DIM}")
    if kv_heads < 1 or heads < 1 or heads % kv_heads:
        raise ValueError(f"{heads} heads are not a multiple of {kv_heads} key heads")
    return _Desc(q.device.index, _DTYPES[q.dtype], heads, kv_heads, dim, _int("window", window, 0),
                 _int("sinks", sinks, 0), dim ** -0.5 if scale is None else float(scale), batch, q_len, k_len,
                 int(zero_rest), 0)


def _window_operands(q, k, v, window, sinks, scale, cu_q, cu_k, zero_rest):
    packed = cu_q is not None
    if not packed and cu_k is not None:
        raise ValueError("cu_k without cu_q")
    nd = 3 if packed else 4
    _tensor("q", q)
    _tensor("k", k, q)
    _tensor("v", v, q)
    if q.ndim != nd or k.ndim != nd or v.ndim != nd:
        raise ValueError(f"q, k and v need {nd} dimensions: " + ("[rows, heads, d]" if packed else "[batch, rows, heads, d]"))
    if k.shape != v.shape or k.shape[-1] != q.shape[-1] or (not packed and k.shape[0] != q.shape[0]):
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not fit")
    batch = q.shape[0]
    if packed:
        cu_k = cu_q if cu_k is None else cu_k
        _tensor("cu_q", cu_q, q, dtype=torch.int32, contiguous=True)
        _tensor("cu_k", cu_k, q, dtype=torch.int32, contiguous=True)
        if cu_q.ndim != 1 or cu_q.shape != cu_k.shape or len(cu_q) < 1:
            raise ValueError("cu_q and cu_k must be vectors of the number of sequences + 1")
        batch = len(cu_q) - 1
    d = _desc(q, k.shape[-2], window, sinks, scale, batch, q.shape[-3], k.shape[-3], zero_rest and packed)
    return packed, d, cu_q.data_ptr() if packed else None, cu_k.data_ptr() if packed else None


def window_attention(q, k, v, window: int = 0, sinks: int = 0, scale: float | None = None, cu_q=None, cu_k=None,
                     out=None, lse=None, stream: int | None = None):
    """Causal attention: (out, lse).

    q [batch, rows, heads, d], k and v [batch, key rows, key heads, d]; or, with int32 offsets ``cu_q`` and ``cu_k``
    ([sequences + 1], on the device; cu_k defaults to cu_q), [rows, heads, d] and [key rows, key heads, d].
    ``scale`` defaults to d ** -0.5.  out is like q, lse float32 with q's shape less its last dimension (the log of the sum
    of the exponentials, -inf where a query sees nothing).  With offsets, rows behind the last sequence are set to 0
    (lse -inf) in an out that the call allocates and left as they are, in lse too, if ``out`` is given."""
    packed, d, pq, pk = _window_operands(q, k, v, window, sinks, scale, cu_q, cu_k, out is None)
    st, where = _place(q, stream)
    with where:
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        else:
            _tensor("out", out, q, q.shape)
        if lse is None:
            lse = torch.empty(q.shape[:-1], dtype=torch.float32, device=q.device)
        else:
            _tensor("lse", lse, q, q.shape[:-1], torch.float32, True)
        if packed and d.batch == 0 and d.zero_rest:
            return out.zero_(), lse.fill_(float("-inf"))
    _check("window_attention", lib.spmm_attn_window(d, _rows(q, packed), _rows(k, packed), _rows(v, packed), pq, pk,
                                                    _rows(out, packed), lse.data_ptr(), st))
    return out, lse


def window_attention_backward(dout, q, k, v, out, lse, window: int = 0, sinks: int = 0, scale: float | None = None,
                              cu_q=None, cu_k=None, dq=None, dk=None, dv=None, stream: int | None = None):
    """Gradients (dq, dk, dv) of ``window_attention`` for the gradient ``dout`` of its out; out, lse: what it returned,
    the other arguments as they were.  With offsets, rows behind the last sequence are set to 0 if the call allocates
    all three, and left as they are if any is given."""
    packed, d, pq, pk = _window_operands(q, k, v, window, sinks, scale, cu_q, cu_k, dq is None and dk is None and dv is None)
    _tensor("dout", dout, q, q.shape)
    _tensor("out", out, q, q.shape)
    _tensor("lse", lse, q, q.shape[:-1], torch.float32, True)
    st, where = _place(q, stream)
    need = C.c_size_t()
    _check("window_attention_backward", lib.spmm_attn_window_work(d, int(packed), C.byref(need)))
    with where:
        dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) if g is None else _tensor(n, g, q, t.shape)
                      for n, g, t in (("dq", dq, q), ("dk", dk, k), ("dv", dv, v)))
        work = torch.empty(need.value, dtype=torch.uint8, device=q.device)
        if packed and d.batch == 0 and d.zero_rest:
            return dq.zero_(), dk.zero_(), dv.zero_()
    _check("window_attention_backward", lib.spmm_attn_window_grad(
        d, _rows(dout, packed), _rows(q, packed), _rows(k, packed), _rows(v, packed), _rows(out, packed), lse.data_ptr(),
        pq, pk, _rows(dq, packed), _rows(dk, packed), _rows(dv, packed), work.data_ptr(), need.value, st))
    return dq, dk, dv


def _pages(k_pages, v_pages, page_table, lengths, like, batch: int) -> _Pages:
    _tensor("k_pages", k_pages, like)
    _tensor("v_pages", v_pages, like)
    if k_pages.ndim != 4 or k_pages.shape != v_pages.shape or k_pages.shape[3] != like.shape[-1]:
        raise ValueError(f"pages {tuple(k_pages.shape)} and {tuple(v_pages.shape)}: [pages, rows, key heads, d] expected")
    if k_pages.shape[1] < 1:
        raise ValueError("pages without rows")
    _tensor("page_table", page_table, like, dtype=torch.int32)
    if page_table.ndim != 2 or page_table.shape[0] != batch:
        raise ValueError(f"page_table {tuple(page_table.shape)}: one row for each of {batch} sequences expected")
    _tensor("lengths", lengths, like, (batch,), torch.int32, True)
    ks, vs = k_pages.stride(), v_pages.stride()
    return _Pages(k_pages.data_ptr(), v_pages.data_ptr(), k_pages.shape[0], k_pages.shape[1], ks[0], ks[1], ks[2], vs[0],
                  vs[1], vs[2], page_table.data_ptr(), page_table.shape[1], page_table.stride(0), lengths.data_ptr())


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
    _tensor("q", q)
    if q.ndim != 3:
        raise ValueError(f"q {tuple(q.shape)}: [batch, heads, d] expected")
    pages = _pages(k_pages, v_pages, page_table, lengths, q, q.shape[0])
    d = _desc(q, k_pages.shape[2], window, sinks, scale, q.shape[0], 1, 0)
    room = min(page_table.shape[1] * k_pages.shape[1], 2 ** 30 - 1)
    longest = room if max_length is None else min(_int("max_length", max_length, 0), room)
    st, where = _place(q, stream)
    need = C.c_size_t()
    _check("paged_attention", lib.spmm_attn_paged_work(d, longest, C.byref(need)))
    with where:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device) if out is None else _tensor("out", out, q, q.shape)
        if lse is None:
            lse = torch.empty(q.shape[:-1], dtype=torch.float32, device=q.device)
        else:
            _tensor("lse", lse, q, q.shape[:-1], torch.float32, True)
        work = torch.empty(need.value, dtype=torch.uint8, device=q.device) if need.value else None
    qs, os = q.stride(), out.stride()
    _check("paged_attention", lib.spmm_attn_paged(
        d, _Rows(q.data_ptr(), qs[0], 0, qs[1]), pages, longest, _Rows(out.data_ptr(), os[0], 0, os[1]), lse.data_ptr(),
        work.data_ptr() if work is not None else None, need.value, st))
    return out, lse


def cache_append(k, v, k_pages, v_pages, page_table, lengths, cu=None, stream: int | None = None) -> None:
    """Write the keys and values of new tokens into the cache: those of sequence b go to its last positions before
    ``lengths[b]``.  k and v [batch, key heads, d], one token a sequence (none for a sequence of length 0), or, with
    int32 offsets ``cu`` [batch + 1] on the device, [rows, key heads, d].  Rows whose page is not there are dropped.  A
    page that is written must belong to one sequence only."""
    _tensor("k", k)
    _tensor("v", v, k, k.shape)
    if k.ndim != 3:
        raise ValueError(f"k {tuple(k.shape)}: [rows, key heads, d] expected")
    if cu is not None:
        _tensor("cu", cu, k, dtype=torch.int32, contiguous=True)
        if cu.ndim != 1 or len(cu) < 1:
            raise ValueError("cu must be a vector of the number of sequences + 1")
    batch = k.shape[0] if cu is None else len(cu) - 1
    pages = _pages(k_pages, v_pages, page_table, lengths, k, batch)
    if k_pages.shape[2] != k.shape[1]:
        raise ValueError(f"{k.shape[1]} key heads, the pages have {k_pages.shape[2]}")
    d = _desc(k, k.shape[1], 0, 0, 1.0, batch, k.shape[0], 0)
    st, _ = _place(k, stream)
    _check("cache_append", lib.spmm_attn_append(d, _rows(k, True), _rows(v, True), cu.data_ptr() if cu is not None else None,
                                                pages, st))
