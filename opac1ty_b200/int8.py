"""Products in 8-bit integers: tokens and weights as codes with one scale a row (``opc_i8_*``).

    w_qkv = Int8Weight.from_layer(layer)                  # a 2-bit layer, or Int8Weight.quantize(tensor)
    h, x = add_rmsnorm(h, y, norm_weight)                 # the residual stream, and its norm in 8 bits
    qkv = linear(x, w_qkv)
    out = linear(quantize(attention_output), w_o)
    h, x = add_rmsnorm(h, out, norm_weight)
    y = linear(silu_mul(linear(x, w_gate_up)), w_down)

A row stands for ``scale * codes`` with scale = max / 127; the definitions, and what rows of zeros and
rows with infinities or NaN give, are in ``include/opc_b200.h``.  Every computation is a call into
``libopc_b200.so``.  There is no backward pass: results carry no gradient, whatever their inputs ask for.
Tensors given to be written (``out``, ``h_out``) count as changed in place: a backward pass that needs what they
held before is an error, as after torch's own in-place operations.
"""

from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch
from torch.autograd.graph import increment_version

from . import _lib
from . import layer as L
from .kv import _DTYPES, _call, _get_device, _raw_stream

# (sizes, strides, type) -> uninitialized memory on the current device, in half the time of the public calls;
# torch's own name where it has it
_empty_strided = getattr(getattr(getattr(torch._C, "_dynamo", None), "guards", None), "_empty_strided_cuda", None)


def _empty(like: torch.Tensor, index: int, shape: Tuple[int, ...], strides: Tuple[int, ...], dtype: torch.dtype) -> torch.Tensor:
    """Contiguous memory on like's device, whose index is ``index``."""
    if _empty_strided is not None and index == _get_device():
        return _empty_strided(shape, strides, dtype)
    return like.new_empty(shape, dtype=dtype)


MAX_WIDTH = 131071  # longest row: no sum of products of two rows leaves 32 bits
MAX_ROWS = 2**31 - 4096


def _row_bytes(n: int) -> int:
    """Bytes from a row of n codes to the next, as they are laid out here: 128-byte lines for long rows (2000
    tokens, 4112 -> 4096: 32.6 us with rows of 4112 bytes, 25.8 with 4224), sectors for short ones."""
    return -(-n // 128) * 128 if n >= 512 else -(-n // 32) * 32


class Int8Rows:
    """Rows in 8 bits: ``codes`` int8 [rows, n], each row starting on 16 bytes, and ``scales`` fp32
    [rows].  ``values``: what they stand for, where the call that made them was asked for it."""

    __slots__ = ("_codes", "_scales", "_held", "values", "rows", "n", "index", "c", "_ref")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, values: Optional[torch.Tensor] = None):
        if codes.dim() != 2 or codes.dtype != torch.int8 or not codes.is_cuda:
            raise ValueError(f"Int8Rows: codes must be int8 [rows, n] on a CUDA device, got {codes.dtype} "
                             f"{tuple(codes.shape)} on {codes.device}")
        rows, n = codes.shape
        if n < 1 or n > MAX_WIDTH or rows > MAX_ROWS:
            raise ValueError(f"Int8Rows: {rows} rows of {n} values (up to {MAX_ROWS} rows of 1 to {MAX_WIDTH})")
        if scales.dtype != torch.float32 or tuple(scales.shape) != (rows,) or scales.device != codes.device or \
                (rows > 1 and scales.stride(0) != 1):
            raise ValueError(f"Int8Rows: scales must be contiguous float32 [{rows}] on {codes.device}, got {scales.dtype} "
                             f"{tuple(scales.shape)} on {scales.device}")
        ld = codes.stride(0) if rows > 1 else -(-n // 16) * 16
        if (n > 1 and codes.stride(1) != 1) or ld < n or ld % 16 or (rows and codes.data_ptr() % 16):
            raise ValueError(f"Int8Rows: rows of codes must start on 16 bytes and not overlap, got strides {codes.stride()}")
        self._codes, self._scales, self._held, self.values = codes, scales, None, values
        self.rows, self.n, self.index = rows, n, codes.get_device()
        self.c = _lib.I8Rows(rows, n, ld, codes.data_ptr(), scales.data_ptr())
        self._ref = ctypes.addressof(self.c)

    @classmethod
    def _new(cls, like: torch.Tensor, rows: int, n: int, values: Optional[torch.dtype]) -> "Int8Rows":
        """Memory for rows of n values on like's device: codes and then scales in one piece (a tensor costs
        more to make than the quantization of a token)."""
        if n < 1 or n > MAX_WIDTH or rows > MAX_ROWS:  # (the C struct's 32 bits would take more modulo 2^32)
            raise ValueError(f"{rows} rows of {n} values (up to {MAX_ROWS} rows of 1 to {MAX_WIDTH})")
        if values is not None and values not in _DTYPES:
            raise ValueError(f"values must be float16, bfloat16 or float32, got {values}")
        self = cls.__new__(cls)
        index = like.get_device()
        self.values = None if values is None else _empty(like, index, (rows, n), (n, 1), values)
        ld = _row_bytes(n)
        held = _empty(like, index, (rows * (ld // 4 + 1),), (1,), torch.float32)
        self._codes = self._scales = None
        self._held, self.rows, self.n, self.index = held, rows, n, index
        at = held.data_ptr()
        self.c = _lib.I8Rows(rows, n, ld, at, at + rows * ld)
        self._ref = ctypes.addressof(self.c)
        return self

    @property
    def codes(self) -> torch.Tensor:
        if self._codes is None:
            ld = self.c.ld
            codes = self._held[:self.rows * (ld // 4)].view(torch.int8).view(self.rows, ld)
            self._codes = codes if ld == self.n else codes[:, :self.n]
        return self._codes

    @property
    def scales(self) -> torch.Tensor:
        if self._scales is None:
            self._scales = self._held[self.rows * (self.c.ld // 4):]
        return self._scales

    @property
    def device(self) -> torch.device:
        return (self._held if self._codes is None else self._codes).device

    def device_bytes(self) -> int:
        return int(self.rows * (self.c.ld + 4))


class Int8Weight(Int8Rows):
    """A layer's weights [channels, k] in 8 bits, one scale a channel.  ``codes`` in any layout: other
    than rows that start on whole lines of memory are copied into such."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor):
        if codes.dim() == 2 and codes.is_cuda and codes.dtype == torch.int8 and codes.shape[0] and codes.shape[1]:
            m, k = codes.shape
            line = 128 if k >= 512 else 32
            if (m > 1 and (codes.stride(0) % line or codes.stride(0) < k)) or (k > 1 and codes.stride(1) != 1) or codes.data_ptr() % line:
                held = codes.new_zeros((m, _row_bytes(k)))
                held[:, :k] = codes
                codes = held[:, :k]
        super().__init__(codes, scales)
        if self.rows < 1:
            raise ValueError("Int8Weight: no channels")

    @classmethod
    def quantize(cls, weight: torch.Tensor) -> "Int8Weight":
        """From a matrix [channels, k] in float16, bfloat16 or float32."""
        r = quantize(weight)
        return cls(r.codes, r.scales)

    @classmethod
    def from_layer(cls, dl: "L.DeviceLayer") -> "Int8Weight":
        """From a 2-bit layer (outliers included): every row has its few distinct values and its
        outliers, so the 8 bits add at most max |row| / 254 to each weight."""
        return cls.quantize(L.dequantize(dl))


def _matrix(what: str, name: str, t: torch.Tensor, rows: Optional[int] = None, n: int = 0, index: int = 0) -> int:
    """Leading dimension of a matrix t; with ``rows``, it is [rows, n] on device ``index``."""
    shape, strides, at = t.shape, t.stride(), t.get_device()
    if len(shape) != 2 or at < 0 or t.dtype not in _DTYPES or (strides[1] != 1 and shape[1] > 1 and shape[0]):
        raise ValueError(f"{what}: {name} must be float16, bfloat16 or float32 [rows, n] on a CUDA device with unit stride, got "
                         f"{t.dtype} {tuple(shape)} with strides {strides} on {t.device}")
    if rows is not None:
        if shape[0] != rows or shape[1] != n:
            raise ValueError(f"{what}: {name} must be [{rows}, {n}], got {tuple(shape)}")
        if at != index:
            raise ValueError(f"{what}: {name} is on {t.device}, the others on cuda:{index}")
    return strides[0] if shape[0] > 1 else shape[1]


def _vector(what: str, name: str, t: torch.Tensor, n: int, index: int):
    if t.dtype not in _DTYPES or t.shape != (n,) or (n > 1 and t.stride(0) != 1) or t.get_device() != index:
        raise ValueError(f"{what}: {name} must be contiguous float16, bfloat16 or float32 [{n}] on cuda:{index}, got {t.dtype} "
                         f"{tuple(t.shape)} on {t.device}")


def quantize(x: torch.Tensor, values: Optional[torch.dtype] = None) -> Int8Rows:
    """The rows of x [rows, n] in 8 bits.  ``values``: also give what they stand for, in that type."""
    ld = _matrix("quantize", "x", x)
    rows, n = x.shape
    out = Int8Rows._new(x, rows, n, values)
    index, v = out.index, out.values
    _call(_lib.load().opc_i8_quantize, index, x.data_ptr(), ld, _DTYPES[x.dtype], out._ref,
          None if v is None else v.data_ptr(), n, 0 if v is None else _DTYPES[values], _raw_stream(index))
    return out


def silu_mul(gate: torch.Tensor, up: Optional[torch.Tensor] = None, values: Optional[torch.dtype] = None) -> Int8Rows:
    """The rows of silu(gate) * up in 8 bits; without ``up``, gate holds both side by side, gate first."""
    ldg = _matrix("silu_mul", "gate", gate)
    rows, n = gate.shape
    gate_ptr = gate.data_ptr()
    if up is None:
        if n % 2:
            raise ValueError(f"silu_mul: gate and up side by side need an even width, got {n}")
        n //= 2
        up_ptr, ldu = gate_ptr + n * gate.element_size(), ldg
    else:
        ldu = _matrix("silu_mul", "up", up, rows, n, gate.get_device())
        if up.dtype != gate.dtype:
            raise ValueError(f"silu_mul: gate is {gate.dtype}, up {up.dtype}")
        up_ptr = up.data_ptr()
    out = Int8Rows._new(gate, rows, n, values)
    index, v = out.index, out.values
    _call(_lib.load().opc_i8_silu_mul, index, gate_ptr, ldg, up_ptr, ldu, _DTYPES[gate.dtype], out._ref,
          None if v is None else v.data_ptr(), n, 0 if v is None else _DTYPES[values], _raw_stream(index))
    return out


def add_rmsnorm(h: torch.Tensor, y: Optional[torch.Tensor] = None, weight: Optional[torch.Tensor] = None, eps: float = 1e-5,
                h_out: Optional[torch.Tensor] = None, values: Optional[torch.dtype] = None) -> Tuple[torch.Tensor, Int8Rows]:
    """(h + y, the rows of its root-mean-square norm times ``weight`` in 8 bits).  y has h's type, or
    any beside an h of float32.  The sum goes to ``h_out`` (which may be h, or a y of its type; no other
    overlap) or a new tensor; without y the first result is h itself (or h copied into ``h_out``)."""
    ldh = _matrix("add_rmsnorm", "h", h)
    rows, n = h.shape
    index, h_type = h.get_device(), _DTYPES[h.dtype]
    y_ptr = w_ptr = o_ptr = None
    ldy = y_type = w_type = ldo = 0
    given = h_out is not None
    if y is not None:
        ldy = _matrix("add_rmsnorm", "y", y, rows, n, index)
        y_ptr, y_type = y.data_ptr(), _DTYPES[y.dtype]
        if y_type != h_type and h_type != _lib.OPC_F32:
            raise ValueError(f"add_rmsnorm: y is {y.dtype} beside an h of {h.dtype}")
        if h_out is None:
            h_out = _empty(h, index, (rows, n), (n, 1), h.dtype)
            o_ptr, ldo = h_out.data_ptr(), n
    if given:
        ldo = _matrix("add_rmsnorm", "h_out", h_out, rows, n, index)
        if h_out.dtype != h.dtype:
            raise ValueError(f"add_rmsnorm: h_out is {h_out.dtype}, h {h.dtype}")
        if rows > 1 and ldo < n:
            raise ValueError(f"add_rmsnorm: the rows of h_out overlap (strides {h_out.stride()})")
        o_ptr = h_out.data_ptr()
    if weight is not None:
        _vector("add_rmsnorm", "weight", weight, n, index)
        w_ptr, w_type = weight.data_ptr(), _DTYPES[weight.dtype]
    out = Int8Rows._new(h, rows, n, values)
    v = out.values
    _call(_lib.load().opc_i8_add_rmsnorm, index, h.data_ptr(), ldh, h_type, y_ptr, ldy, y_type, w_ptr, w_type, eps, o_ptr, ldo,
          out._ref, None if v is None else v.data_ptr(), n, 0 if v is None else _DTYPES[values], _raw_stream(index))
    if h_out is None:
        return h, out
    if given:
        increment_version(h_out)
    return h_out, out


def linear(x: Int8Rows, weight: Int8Weight, bias: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.float16,
           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x times weight transposed, with both scales (and a bias [channels]): [rows, channels] in
    ``dtype``, or in ``out`` and its type."""
    index, rows, m = x.index, x.rows, weight.rows
    if weight.n != x.n or weight.index != index:
        raise ValueError(f"linear: x has rows of {x.n} on cuda:{index}, the weight of {weight.n} on cuda:{weight.index}")
    if out is None:
        if dtype not in _DTYPES:
            raise ValueError(f"linear: results are float16, bfloat16 or float32, not {dtype}")
        result = _empty(weight.scales, index, (rows, m), (m, 1), dtype)
        ldy = m
    else:
        result = out
        ldy = _matrix("linear", "out", out, rows, m, index)
        if rows > 1 and ldy < m:
            raise ValueError(f"linear: the rows of out overlap (strides {out.stride()})")
        dtype = out.dtype
    b_ptr, b_type = None, 0
    if bias is not None:
        _vector("linear", "bias", bias, m, index)
        b_ptr, b_type = bias.data_ptr(), _DTYPES[bias.dtype]
    _call(_lib.load().opc_i8_gemm, index, x._ref, weight._ref, b_ptr, b_type, result.data_ptr(), ldy, _DTYPES[dtype],
          _raw_stream(index))
    if out is not None:
        increment_version(out)
    return result
