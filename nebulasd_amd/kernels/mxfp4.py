"""Microscaled (OCP MX) projections: 4-bit weights, 8-bit activations.

The decode and verify layers are bound by their weights' stream from memory.
``mxfp4_linear`` and ``mxfp4_up_gate_silu_and_mul`` are ``linear`` and
``up_gate_silu_and_mul`` over weights of 4.25 bits a value instead of 16 (the
reference has only fp16 projections: swiftLLM/swiftllm/worker/kernels/linear.py:3-12),
for any number of rows.  A row is cut into blocks of 32 values: one power of
two and 32 codes, E2M1 for the weight (``MXFP4Weight``) and E4M3 for the rows it
is multiplied with (``MXFP8Rows``), which gfx950's scaled matrix instructions
multiply as they are.  Sums are held in fp32, but of the eight products that an
instruction adds at a time bits 13 below the largest one's exponent are cut:
together 2e-5 of the sums' norm, where their rounding to fp16 takes 2.1e-4.
``include/nsd_mx.h`` states the formats, the roundings and the layouts.

A weight comes from ``mxfp4_quantize`` (from fp16, bf16 or fp32) or
``mxfp4_pack`` (from a checkpoint's codes and scales), once.  The products
quantise fp16 rows themselves; rows that several projections read are
quantised once with ``mxfp8_quantize`` and given instead.  The same call gives the
same bits; in a batch of another size, or given in blocks instead of fp16, a row
may be added up in another order and end in another last place.
"""

from __future__ import annotations

import ctypes
import functools

import torch

from .. import _lib
from ._util import require, require_cuda, stream_on

BLOCK = 32
_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}


def _check_blocks(codes, scales, bits: int, rows: int, n_in: int) -> None:
    c, s = _bytes(bits, rows, n_in)
    for t, n in ((codes, c), (scales, s)):
        if t.dtype != torch.uint8 or not t.is_contiguous() or t.numel() != n:
            raise ValueError(f"[{rows}, {n_in}] in MXFP{bits} is {c} bytes of codes and {s} of scales")
    require_cuda(codes, scales)
    _same_device(codes, scales)


def _fixed(self, name, value):
    raise AttributeError(f"{type(self).__name__} is fixed once made: its sizes were checked then")


def _parts(self):
    return type(self), tuple(getattr(self, name) for name in self.__slots__)


class MXFP4Weight:
    """A weight [n_out, n_in] in MXFP4: codes and scales (uint8) in the kernels' layout."""

    __slots__ = ("codes", "scales", "n_out", "n_in")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, n_out: int, n_in: int, _made: bool = False):
        if not _made:
            _check_blocks(codes, scales, 4, n_out, n_in)
        for name, v in zip(self.__slots__, (codes, scales, n_out, n_in)):
            object.__setattr__(self, name, v)

    __setattr__ = _fixed
    __reduce__ = _parts  # copy and pickle


class MXFP8Rows:
    """Rows [rows, n_in] in MXFP8: codes and scales (uint8) in the kernels' layout."""

    __slots__ = ("codes", "scales", "rows", "n_in")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, rows: int, n_in: int, _made: bool = False):
        if not _made:
            _check_blocks(codes, scales, 8, rows, n_in)
        for name, v in zip(self.__slots__, (codes, scales, rows, n_in)):
            object.__setattr__(self, name, v)

    __setattr__ = _fixed
    __reduce__ = _parts  # copy and pickle


@functools.lru_cache(maxsize=4096)
def _bytes(bits: int, rows: int, n_in: int):
    c, s = ctypes.c_int64(), ctypes.c_int64()
    _lib.call("nsd_mx_bytes", bits, rows, n_in, ctypes.byref(c), ctypes.byref(s))
    return c.value, s.value


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(device: int, rows: int, n_out: int, n_in: int, gated: bool, quantised: bool) -> int:
    b = ctypes.c_int64()
    with torch.cuda.device(device):
        _lib.call("nsd_mx_workspace", rows, n_out, n_in, gated, quantised, ctypes.byref(b))
    return b.value


def _call(device: int, name: str, *args) -> None:
    """``name`` on a device and its current stream."""
    if device == torch.cuda.current_device():
        _lib.call(name, *args, stream_on(device))
    else:
        with torch.cuda.device(device):
            _lib.call(name, *args, stream_on(device))


def _same_device(a: torch.Tensor, b: torch.Tensor) -> None:
    if a.get_device() != b.get_device():
        raise ValueError(f"all tensors must be on one device, got {a.device} and {b.device}")


def _matrix(t: torch.Tensor, name: str) -> None:
    if t.dim() != 2 or t.shape[1] < BLOCK or t.shape[1] % BLOCK:
        raise ValueError(f"{name} must be [rows, n_in] with n_in a multiple of {BLOCK}, got {tuple(t.shape)}")


def _empty(bits: int, rows: int, n_in: int, like: torch.Tensor):
    c, s = _bytes(bits, rows, n_in)
    return like.new_empty(c, dtype=torch.uint8), like.new_empty(s, dtype=torch.uint8)


def mxfp4_quantize(w: torch.Tensor) -> MXFP4Weight:
    """w [n_out, n_in] (fp16, bf16 or fp32) in MXFP4.  A block with an infinity or a NaN becomes NaN."""
    require_cuda(w)
    _matrix(w, "w")
    if w.dtype not in _DTYPES:
        raise TypeError(f"w must be fp16, bf16 or fp32, got {w.dtype}")
    require(w, w.dtype, "w")
    n_out, n_in = w.shape
    codes, scales = _empty(4, n_out, n_in, w)
    _call(w.get_device(), "nsd_mxfp4_quantize", w.data_ptr(), _DTYPES[w.dtype], n_out, n_in, codes.data_ptr(), scales.data_ptr())
    return MXFP4Weight(codes, scales, n_out, n_in, _made=True)


def mxfp4_pack(codes: torch.Tensor, scales: torch.Tensor) -> MXFP4Weight:
    """A checkpoint's MXFP4 weight: uint8 codes [n_out, n_in / 2] (the even value in the low half) and uint8
    scales [n_out, n_in / 32]."""
    require_cuda(codes, scales)
    require(codes, torch.uint8, "codes")
    require(scales, torch.uint8, "scales")
    if codes.dim() != 2 or scales.dim() != 2 or scales.shape[1] < 1 or \
            tuple(codes.shape) != (scales.shape[0], scales.shape[1] * BLOCK // 2):
        raise ValueError(f"codes must be [n_out, n_in / 2] and scales [n_out, n_in / {BLOCK}], got "
                         f"{tuple(codes.shape)} and {tuple(scales.shape)}")
    _same_device(codes, scales)
    n_out, n_in = codes.shape[0], 2 * codes.shape[1]
    out = _empty(4, n_out, n_in, codes)
    _call(codes.get_device(), "nsd_mxfp4_pack", codes.data_ptr(), scales.data_ptr(), n_out, n_in, *(t.data_ptr() for t in out))
    return MXFP4Weight(*out, n_out, n_in, _made=True)


def mxfp8_quantize(x: torch.Tensor) -> MXFP8Rows:
    """x [rows, n_in] fp16 in MXFP8.  A block with an infinity or a NaN becomes NaN."""
    require_cuda(x)
    _matrix(x, "x")
    require(x, torch.float16, "x")
    rows, n_in = x.shape
    codes, scales = _empty(8, rows, n_in, x)
    _call(x.get_device(), "nsd_mxfp8_quantize", x.data_ptr(), rows, n_in, codes.data_ptr(), scales.data_ptr())
    return MXFP8Rows(codes, scales, rows, n_in, _made=True)


def _dequantize(b, rows: int, dtype: torch.dtype, name: str) -> torch.Tensor:
    if dtype not in _DTYPES:
        raise TypeError(f"dtype must be fp16, bf16 or fp32, got {dtype}")
    out = b.codes.new_empty((rows, b.n_in), dtype=dtype)
    _call(out.get_device(), name, b.codes.data_ptr(), b.scales.data_ptr(), rows, b.n_in, out.data_ptr(), _DTYPES[dtype])
    return out


def mxfp4_dequantize(w: MXFP4Weight, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values [n_out, n_in] that ``w`` stands for; exact in bf16 and fp32."""
    return _dequantize(w, w.n_out, dtype, "nsd_mxfp4_dequantize")


def mxfp8_dequantize(x: MXFP8Rows, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values [rows, n_in] that ``x`` stands for; exact in bf16 and fp32."""
    return _dequantize(x, x.rows, dtype, "nsd_mxfp8_dequantize")


def _check_x(x: torch.Tensor, w: MXFP4Weight) -> None:
    require_cuda(x)
    require(x, torch.float16, "x")
    if x.dim() != 2:
        raise ValueError(f"x must be [rows, n_in], got {tuple(x.shape)}")
    _same_device(x, w.codes)


def _product(x, w: MXFP4Weight, n: int, out, gated: bool, name: str) -> torch.Tensor:
    # the checks of a decode step's call are kept short: at one row they and
    # the launch are most of its time
    codes = w.codes
    device = codes.get_device()
    quantised = type(x) is MXFP8Rows
    if quantised:
        rows, n_in = x.rows, x.n_in
        _same_device(x.codes, codes)
        given = (None, x.codes.data_ptr(), x.scales.data_ptr())
    else:
        if x.dtype is not torch.float16 or x.dim() != 2 or x.get_device() != device or not x.is_contiguous():
            _check_x(x, w)
        rows, n_in = x.shape
        given = (x.data_ptr(), None, None)
    if n_in != w.n_in:
        raise ValueError(f"x has {n_in} columns, the weight is [{w.n_out}, {w.n_in}]")
    if out is None:
        out = codes.new_empty((rows, n), dtype=torch.float16)
    else:
        require_cuda(out)
        require(out, torch.float16, "out")
        _same_device(out, codes)
        if tuple(out.shape) != (rows, n):
            raise ValueError(f"out must be [{rows}, {n}]")
    if rows == 0:
        return out
    size = _workspace_bytes(device, rows, w.n_out, n_in, gated, quantised)
    # the call's own, so calls on other streams and captured ones share nothing
    ws = codes.new_empty(size) if size else None
    _call(device, name, *given, codes.data_ptr(), w.scales.data_ptr(), out.data_ptr(), rows, n, n_in,
          ws.data_ptr() if size else None, size)
    return out


def mxfp4_linear(x: torch.Tensor | MXFP8Rows, w: MXFP4Weight, out: torch.Tensor | None = None) -> torch.Tensor:
    """``linear`` with an MXFP4 weight: fp16 [rows, n_out] = fp16(X . W^T), X the MXFP8 values of x [rows, n_in]
    (fp16, or quantised already), the sum held in fp32 as the module says."""
    return _product(x, w, w.n_out, out, False, "nsd_mxfp4_linear")


def mxfp4_up_gate_silu_and_mul(x: torch.Tensor | MXFP8Rows, w: MXFP4Weight,
                               out: torch.Tensor | None = None) -> torch.Tensor:
    """``up_gate_silu_and_mul`` with an MXFP4 weight [2 * inter, n_in] (up rows first): fp16 [rows, inter] =
    fp16(up * silu(gate)), the products and the SiLU-and-mul in fp32, rounded once."""
    if w.n_out % 32:
        raise ValueError(f"an up/gate weight has 2 * inter rows, inter a multiple of 16; got {w.n_out}")
    return _product(x, w, w.n_out // 2, out, True, "nsd_mxfp4_up_gate_silu_and_mul")
