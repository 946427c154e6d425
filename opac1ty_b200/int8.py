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
"""

from __future__ import annotations

import ctypes
import functools
from typing import Optional, Tuple

import torch

from . import _lib
from . import layer as L
from .kv import _DTYPES, _call, _check_workspace, _raw_stream, _workspace

MAX_WIDTH = 131071  # longest row: no sum of products of two rows leaves 32 bits


class Int8Rows:
    """Rows in 8 bits: ``codes`` int8 [rows, n], each row starting on 16 bytes, and ``scales`` fp32
    [rows].  ``values``: what they stand for, where the call that made them was asked for it."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, values: Optional[torch.Tensor] = None):
        if codes.dim() != 2 or codes.dtype != torch.int8 or not codes.is_cuda:
            raise ValueError(f"Int8Rows: codes must be int8 [rows, n] on a CUDA device, got {codes.dtype} "
                             f"{tuple(codes.shape)} on {codes.device}")
        rows, n = codes.shape
        if n < 1 or n > MAX_WIDTH:
            raise ValueError(f"Int8Rows: rows of {n} values (1 to {MAX_WIDTH})")
        if scales.dtype != torch.float32 or tuple(scales.shape) != (rows,) or scales.device != codes.device or \
                (rows > 1 and scales.stride(0) != 1):
            raise ValueError(f"Int8Rows: scales must be contiguous float32 [{rows}] on {codes.device}, got {scales.dtype} "
                             f"{tuple(scales.shape)} on {scales.device}")
        ld = codes.stride(0) if rows > 1 else -(-n // 16) * 16
        if (n > 1 and codes.stride(1) != 1) or ld < n or ld % 16 or (rows and codes.data_ptr() % 16):
            raise ValueError(f"Int8Rows: rows of codes must start on 16 bytes and not overlap, got strides {codes.stride()}")
        self._set(codes, scales, values, rows, n, ld)

    def _set(self, codes, scales, values, rows, n, ld):
        self.codes, self.scales, self.values = codes, scales, values
        self.rows, self.n, self.device = rows, n, codes.device
        self.c = _lib.I8Rows(rows, n, ld, codes.data_ptr(), scales.data_ptr())
        self._ref = ctypes.addressof(self.c)

    @classmethod
    def _new(cls, like: torch.Tensor, rows: int, n: int, values: Optional[torch.dtype]) -> "Int8Rows":
        """Memory for rows of n values on like's device."""
        if n < 1 or n > MAX_WIDTH:
            raise ValueError(f"rows of {n} values (1 to {MAX_WIDTH})")
        if values is not None and values not in _DTYPES:
            raise ValueError(f"values must be float16, bfloat16 or float32, got {values}")
        ld = -(-n // 16) * 16
        codes = like.new_empty((rows, ld), dtype=torch.int8)
        self = cls.__new__(cls)
        self._set(codes if ld == n else codes[:, :n], like.new_empty(rows, dtype=torch.float32),
                  None if values is None else like.new_empty((rows, n), dtype=values), rows, n, ld)
        return self

    def _values_args(self) -> Tuple[Optional[int], int, int]:
        v = self.values
        return (None, 0, 0) if v is None else (v.data_ptr(), self.n, _DTYPES[v.dtype])

    def device_bytes(self) -> int:
        return int(self.rows * (self.c.ld + 4))


class Int8Weight(Int8Rows):
    """A layer's weights [channels, k] in 8 bits, one scale a channel.  ``codes`` in any layout: other
    than rows that start on 16 bytes are copied into such."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor):
        if codes.dim() == 2 and codes.is_cuda and codes.dtype == torch.int8 and codes.shape[0] and codes.shape[1]:
            m, k = codes.shape
            if (m > 1 and (codes.stride(0) % 16 or codes.stride(0) < k)) or (k > 1 and codes.stride(1) != 1) or codes.data_ptr() % 16:
                held = codes.new_zeros((m, -(-k // 16) * 16))
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


def _matrix(what: str, name: str, t: torch.Tensor, rows: Optional[int] = None, n: Optional[int] = None) -> int:
    """Leading dimension of a matrix t, checked."""
    if t.dim() != 2 or not t.is_cuda or t.dtype not in _DTYPES or (t.shape[1] > 1 and t.numel() and t.stride(1) != 1):
        raise ValueError(f"{what}: {name} must be float16, bfloat16 or float32 [rows, n] on a CUDA device with unit stride, got "
                         f"{t.dtype} {tuple(t.shape)} with strides {t.stride()} on {t.device}")
    if (rows is not None and t.shape[0] != rows) or (n is not None and t.shape[1] != n):
        raise ValueError(f"{what}: {name} must be [{rows}, {n}], got {tuple(t.shape)}")
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _like(what: str, name: str, t: torch.Tensor, other: torch.Tensor):
    if t.device != other.device:
        raise ValueError(f"{what}: {name} is on {t.device}, the others on {other.device}")


def quantize(x: torch.Tensor, values: Optional[torch.dtype] = None) -> Int8Rows:
    """The rows of x [rows, n] in 8 bits.  ``values``: also give what they stand for, in that type."""
    ld = _matrix("quantize", "x", x)
    out = Int8Rows._new(x, x.shape[0], x.shape[1], values)
    _call(_lib.load().opc_i8_quantize, x.device.index, x.data_ptr(), ld, _DTYPES[x.dtype], out._ref, *out._values_args(),
          _raw_stream(x.device.index))
    return out


def silu_mul(gate: torch.Tensor, up: Optional[torch.Tensor] = None, values: Optional[torch.dtype] = None) -> Int8Rows:
    """The rows of silu(gate) * up in 8 bits; without ``up``, gate holds both side by side, gate first."""
    ldg = _matrix("silu_mul", "gate", gate)
    rows, n = gate.shape
    size = gate.element_size()
    if up is None:
        if n % 2:
            raise ValueError(f"silu_mul: gate and up side by side need an even width, got {n}")
        n //= 2
        up_ptr, ldu = gate.data_ptr() + n * size, ldg
    else:
        ldu = _matrix("silu_mul", "up", up, rows, n)
        _like("silu_mul", "up", up, gate)
        if up.dtype != gate.dtype:
            raise ValueError(f"silu_mul: gate is {gate.dtype}, up {up.dtype}")
        up_ptr = up.data_ptr()
    out = Int8Rows._new(gate, rows, n, values)
    _call(_lib.load().opc_i8_silu_mul, gate.device.index, gate.data_ptr(), ldg, up_ptr, ldu, _DTYPES[gate.dtype], out._ref,
          *out._values_args(), _raw_stream(gate.device.index))
    return out


def add_rmsnorm(h: torch.Tensor, y: Optional[torch.Tensor] = None, weight: Optional[torch.Tensor] = None, eps: float = 1e-5,
                h_out: Optional[torch.Tensor] = None, values: Optional[torch.dtype] = None) -> Tuple[torch.Tensor, Int8Rows]:
    """(h + y, the rows of its root-mean-square norm times ``weight`` in 8 bits).  y has h's type, or
    any beside an h of float32.  The sum goes to ``h_out`` (which may be h) or a new tensor; without y
    the first result is h itself (or h copied into ``h_out``)."""
    rows, n = h.shape if h.dim() == 2 else (0, 0)
    ldh = _matrix("add_rmsnorm", "h", h)
    ldy = 0
    if y is not None:
        ldy = _matrix("add_rmsnorm", "y", y, rows, n)
        _like("add_rmsnorm", "y", y, h)
        if y.dtype != h.dtype and h.dtype != torch.float32:
            raise ValueError(f"add_rmsnorm: y is {y.dtype} beside an h of {h.dtype}")
        if h_out is None:
            h_out = torch.empty_like(h, memory_format=torch.contiguous_format)
    ldo = 0
    if h_out is not None:
        ldo = _matrix("add_rmsnorm", "h_out", h_out, rows, n)
        _like("add_rmsnorm", "h_out", h_out, h)
        if h_out.dtype != h.dtype:
            raise ValueError(f"add_rmsnorm: h_out is {h_out.dtype}, h {h.dtype}")
        if rows > 1 and ldo < n:
            raise ValueError(f"add_rmsnorm: the rows of h_out overlap (strides {h_out.stride()})")
    if weight is not None:
        if weight.dtype not in _DTYPES or tuple(weight.shape) != (n,) or (n > 1 and weight.stride(0) != 1):
            raise ValueError(f"add_rmsnorm: weight must be contiguous float16, bfloat16 or float32 [{n}], got {weight.dtype} "
                             f"{tuple(weight.shape)}")
        _like("add_rmsnorm", "weight", weight, h)
    out = Int8Rows._new(h, rows, n, values)
    _call(_lib.load().opc_i8_add_rmsnorm, h.device.index, h.data_ptr(), ldh, _DTYPES[h.dtype],
          y.data_ptr() if y is not None else None, ldy, _DTYPES[y.dtype] if y is not None else 0,
          weight.data_ptr() if weight is not None else None, _DTYPES[weight.dtype] if weight is not None else 0, float(eps),
          h_out.data_ptr() if h_out is not None else None, ldo, out._ref, *out._values_args(), _raw_stream(h.device.index))
    return (h if h_out is None else h_out), out


@functools.lru_cache(maxsize=1024)
def linear_workspace_bytes(rows: int, channels: int, k: int, device: int) -> int:
    return int(_lib.load().opc_i8_gemm_workspace_bytes(rows, channels, k, device))


def linear(x: Int8Rows, weight: Int8Weight, bias: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.float16,
           out: Optional[torch.Tensor] = None, workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x times weight transposed, with both scales (and a bias [channels]): [rows, channels] in
    ``dtype``, or in ``out`` and its type.  ``workspace``: zeroed uint8 memory of
    ``linear_workspace_bytes`` that no other call in flight uses (one per stream by default)."""
    dev, rows, m = x.device, x.rows, weight.rows
    if weight.n != x.n or weight.device != dev:
        raise ValueError(f"linear: x has rows of {x.n} on {dev}, the weight of {weight.n} on {weight.device}")
    if out is None:
        if dtype not in _DTYPES:
            raise ValueError(f"linear: results are float16, bfloat16 or float32, not {dtype}")
        out = x.scales.new_empty((rows, m), dtype=dtype)
        ldy = m
    else:
        ldy = _matrix("linear", "out", out, rows, m)
        if out.device != dev or (rows > 1 and ldy < m):
            raise ValueError(f"linear: out must be on {dev} in rows that do not overlap, got strides {out.stride()} on {out.device}")
    if bias is not None and (bias.dtype not in _DTYPES or tuple(bias.shape) != (m,) or (m > 1 and bias.stride(0) != 1) or bias.device != dev):
        raise ValueError(f"linear: bias must be contiguous float16, bfloat16 or float32 [{m}] on {dev}, got {bias.dtype} "
                         f"{tuple(bias.shape)} on {bias.device}")
    stream = _raw_stream(dev.index)
    if workspace is None:
        workspace = _workspace(dev, stream, linear_workspace_bytes(rows, m, x.n, dev.index), "i8")
    else:
        _check_workspace("linear", workspace, dev)
    _call(_lib.load().opc_i8_gemm, dev.index, x._ref, weight._ref, bias.data_ptr() if bias is not None else None,
          _DTYPES[bias.dtype] if bias is not None else 0, out.data_ptr(), ldy, _DTYPES[out.dtype], workspace.data_ptr(),
          workspace.numel(), stream)
    return out
