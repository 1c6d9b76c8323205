"""spmm_amd.q4 -- products of a few vectors with 4-bit weights (include/spmm_q4.h, lib/libspmm_q4.so).

Beside ``spmm_amd.pbv`` (K = 1 products with pruned weights): here the weights are all there, 4 bits each with a scale
for every ``group`` columns of a row, ``w = scale * (q - zero)``.  ``Q4Format`` lays the weights out on the device once,
in the order in which the product reads them; ``matvec`` multiplies.  Arguments are torch tensors on one HIP device; work
is ordered on ``stream`` (an integer hipStream_t; by default the device's current stream) and products can be captured
in a graph.  There is no CPU path, and no gradient: outside ``torch.no_grad()`` scales and vectors that require one are
refused.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import SpmmHipError, _open
from .attention import F16, BF16, F32, _HERE, _int, _lost, _place, _stream, _tensor

_DTYPES = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}


class _Desc(C.Structure):
    _fields_ = [("device", C.c_int32), ("dtype", C.c_int32), ("rows", C.c_int64), ("cols", C.c_int64),
                ("group", C.c_int32), ("zeros", C.c_int32)]


def _bind(L: C.CDLL) -> C.CDLL:
    d, vp, i64 = C.POINTER(_Desc), C.c_void_p, C.c_int64
    L.spmm_q4_layout_bytes.argtypes = [d, C.POINTER(C.c_size_t)]
    L.spmm_q4_layout.argtypes = [d, vp, i64, vp, i64, vp, i64, vp, C.c_size_t, vp]
    L.spmm_q4_matvec.argtypes = [d, vp, vp, i64, i64, vp, i64, vp]
    L.spmm_q4_last_error_detail.restype = C.c_char_p
    return L


lib = _bind(_open("libspmm_q4.so"))


def _check(where: str, st: int) -> None:
    if st != 0:
        raise SpmmHipError(where, st, (lib.spmm_q4_last_error_detail() or b"").decode())


class Q4Format:
    """W [rows, cols] in 4 bits, laid out for ``matvec``.

    packed uint8 [rows, (cols + 1) // 2], column 2 i in the low half of byte i; scales [rows, groups], float32, float16 or
    bfloat16 (the type of the vectors too), groups = cols / group rounded up; zeros uint8 [rows, groups], or None for
    8.  group: 32, 64 or a multiple of 128.  The arguments are not kept; what is written to them on ``stream``, or after it, changes
    nothing."""

    format_name = "HIP_Q4_MI355X"

    def __init__(self, packed, scales, zeros=None, cols: int | None = None, group: int = 128, stream: int | None = None):
        ps = _tensor("packed", packed, torch.uint8)
        dev = packed.get_device()
        ss = _tensor("scales", scales, None, dev)
        if scales.dtype not in _DTYPES:
            raise TypeError(f"scales are {scales.dtype}: float32, float16 or bfloat16")
        if len(ps) != 2 or len(ss) != 2:
            raise ValueError("packed and scales must have two dimensions")
        if scales.requires_grad:
            _lost(scales=scales)
        self.rows = packed.shape[0]
        self.cols = 2 * packed.shape[1] if cols is None else _int("cols", cols, 0)
        self.group = _int("group", group, 1)
        if packed.shape[1] != (self.cols + 1) // 2:
            raise ValueError(f"packed has {packed.shape[1]} bytes a row, {self.cols} columns need {(self.cols + 1) // 2}")
        shape = (self.rows, -(-self.cols // self.group))
        _tensor("scales", scales, shape=shape)
        zs = _tensor("zeros", zeros, torch.uint8, dev, shape) if zeros is not None else (0, 0)
        self.dtype, self.device = scales.dtype, packed.device
        self._dev = dev
        self._d = _Desc(dev, _DTYPES[scales.dtype], self.rows, self.cols, self.group, int(zeros is not None))
        need = C.c_size_t()
        _check("Q4Format", lib.spmm_q4_layout_bytes(self._d, need))
        st, where = _place(dev, stream)
        with where or _HERE:
            self._layout = torch.empty(need.value, dtype=torch.uint8, device=packed.device)
        self._stream = st
        if where is not None:                            # the memory of what is read is not handed on before that is done
            for t in (packed, scales) if zeros is None else (packed, scales, zeros):
                t.record_stream(_stream(dev, st))
        self.mem_footprint = float(need.value)
        _check("Q4Format", lib.spmm_q4_layout(self._d, packed.data_ptr(), ps[0], scales.data_ptr(), ss[0],
                                              zeros.data_ptr() if zeros is not None else None, zs[0],
                                              self._layout.data_ptr(), need.value, st))

    def matvec(self, x, out=None, stream: int | None = None):
        """x W^T: x [cols] or [tokens, cols] (rows any distance apart) -> [rows] or [tokens, rows].  Made for a few
        vectors: every 16 of them (5 in float32) read the weights once more.  A call on another stream than the one the
        format was made on has to come after it; the format may be dropped as soon as the call returns."""
        xs = _tensor("x", x, self.dtype, self._dev)
        nd = len(xs)
        if nd not in (1, 2) or x.shape[-1] != self.cols:
            raise ValueError(f"x {tuple(x.shape)}: [{self.cols}] or [tokens, {self.cols}] expected")
        if x.requires_grad:
            _lost(x=x)
        shape = (self.rows,) if nd == 1 else (x.shape[0], self.rows)
        st, where = _place(self._dev, stream)
        with where or _HERE:
            if out is None:
                out = x.new_empty(shape)
                os = out.stride()
            else:
                os = _tensor("out", out, self.dtype, self._dev, shape)
            if self.cols == 0:
                return out.zero_()
        if st != self._stream:                           # the layout, which no caller has, outlives the product there
            self._layout.record_stream(_stream(self._dev, st))
        _check("matvec", lib.spmm_q4_matvec(self._d, self._layout.data_ptr(), x.data_ptr(), xs[0] if nd == 2 else 0,
                                            x.shape[0] if nd == 2 else 1, out.data_ptr(), os[0] if nd == 2 else self.rows, st))
        return out
