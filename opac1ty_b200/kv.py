"""The paged key/value cache held in 4 bits: append, read back, attention (``opc_kv_*``).

    cache = KVCache(kv_heads=8, head_dim=128, n_pages=1024, page_size=64)
    batch = KVBatch(q_start, kv_len, page_table)          # int32 tensors on the cache's device
    rope = Rope(128, theta=500000.0)
    q = append(cache, batch, k, v, q=q, rope=rope)        # stores k and v, returns the turned q
    out = attention(cache, batch, q)

Rows are packed: rows ``q_start[s] .. q_start[s+1]`` of q, k and v are the last rows of sequence s,
which holds ``kv_len[s]`` tokens once they are in.  The layout of a page, the quantization and the
treatment of rows that belong nowhere are in ``include/opc_b200.h``.  The lengths and the page table
are read on the device: a captured graph replays with what they hold then.  Every computation is a
call into ``libopc_b200.so``.  There is no backward pass: results carry no gradient, whatever their
inputs ask for.
"""

from __future__ import annotations

import ctypes
import threading
from typing import Dict, Optional, Tuple

import numpy as np
import torch

from . import _lib
from .layer import _as_cuda_device

_HALVES = {torch.float16: _lib.OPC_F16, torch.bfloat16: _lib.OPC_BF16}
_DTYPES = {torch.float16: _lib.OPC_F16, torch.bfloat16: _lib.OPC_BF16, torch.float32: _lib.OPC_F32}


def _public_stream(index: int) -> int:
    return torch.cuda.current_stream(index).cuda_stream


# the current device, and the handle of a device's current stream: torch's own names where it has them
# (the public calls, which take their place elsewhere, wrap them in checks and objects)
_get_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _public_stream)


def _call(fn, index: int, *args):
    """fn(*args) with `index` the current device, which the library launches on."""
    prev = _get_device()
    if prev == index:
        rc = fn(*args)
    else:
        torch.cuda.set_device(index)
        try:
            rc = fn(*args)
        finally:
            torch.cuda.set_device(prev)
    if rc < 0:
        raise _lib.OpcError(rc, _lib.last_error())


_ws_lock = threading.Lock()
_workspaces: Dict[Tuple[int, int, str], torch.Tensor] = {}


def _workspace(device: torch.device, stream: int, nbytes: int, kind: str) -> torch.Tensor:
    """A zeroed workspace for one device and stream.  Calls under graph capture get one of their
    own from the graph's memory, so graphs captured on one stream may be replayed side by side; every
    replay clears it (0.8 us for a token of one sequence, 6 to 7 us for chunks and prompts: a workspace
    given by the caller saves that)."""
    if torch.cuda.is_current_stream_capturing():
        return torch.zeros(nbytes, dtype=torch.uint8, device=device)
    key = (device.index, stream, kind)
    ws = _workspaces.get(key)
    if ws is None or ws.numel() < nbytes:
        with _ws_lock:
            ws = _workspaces.get(key)
            if ws is None or ws.numel() < nbytes:
                ws = _workspaces[key] = torch.zeros(max(nbytes, 1 << 20), dtype=torch.uint8, device=device)
    return ws


def _check_workspace(what: str, ws: torch.Tensor, device: torch.device):
    if ws.device != device or ws.dtype != torch.uint8 or not ws.is_contiguous():
        raise ValueError(f"{what}: the workspace must be contiguous uint8 values on {device}, got {ws.dtype} "
                         f"{tuple(ws.shape)} on {ws.device}")


class KVCache:
    """n_pages pages of page_size tokens for kv_heads heads of head_dim, 4 bits a value
    (``opc_kv_plan``).  ``pages``: an existing uint8 tensor of ``total_bytes`` bytes to use."""

    def __init__(self, kv_heads: int, head_dim: int, n_pages: int, page_size: int = 64, device=None,
                 pages: Optional[torch.Tensor] = None):
        self.c = _lib.KvCache()
        _lib.check(_lib.load().opc_kv_plan(int(kv_heads), int(head_dim), int(page_size), int(n_pages),
                                           ctypes.byref(self.c)))
        if pages is None:
            pages = torch.zeros(n_pages, kv_heads, self.c.head_bytes, dtype=torch.uint8, device=_as_cuda_device(device))
        if not pages.is_cuda or pages.dtype != torch.uint8 or not pages.is_contiguous() or \
                pages.numel() != self.c.total_bytes:
            raise ValueError(f"KVCache: pages must be {self.c.total_bytes} contiguous uint8 values on a CUDA device, "
                             f"got {pages.dtype} {tuple(pages.shape)} on {pages.device}")
        if device is not None and pages.device != _as_cuda_device(device):
            raise ValueError(f"KVCache: pages are on {pages.device}, not {device}")
        self.pages = pages
        self.device = pages.device
        self.c.pages = pages.data_ptr()
        self.kv_heads, self.head_dim = int(kv_heads), int(head_dim)
        self.page_size, self.n_pages = int(page_size), int(n_pages)
        self._ref = ctypes.addressof(self.c)

    def device_bytes(self) -> int:
        return int(self.c.total_bytes)


class KVBatch:
    """The rows of a call (``opc_kv_batch``): int32 tensors ``q_start`` [n + 1], ``kv_len`` [n] and
    ``page_table`` [n, pages] on one CUDA device.  ``n_tokens`` (rows in q, k, v), ``max_q`` and
    ``max_kv`` bound the sequences on the host; those not given are read from the tensors, which
    waits for the device."""

    def __init__(self, q_start: torch.Tensor, kv_len: torch.Tensor, page_table: torch.Tensor,
                 n_tokens: Optional[int] = None, max_q: Optional[int] = None, max_kv: Optional[int] = None):
        for name, t, dim in (("q_start", q_start, 1), ("kv_len", kv_len, 1), ("page_table", page_table, 2)):
            if not t.is_cuda or t.dtype != torch.int32 or t.dim() != dim or t.device != q_start.device:
                raise ValueError(f"KVBatch: {name} must be a {dim}-d int32 tensor on one CUDA device, got {t.dtype} "
                                 f"{tuple(t.shape)} on {t.device}")
            if t.numel() and t.stride(-1) != 1:
                raise ValueError(f"KVBatch: {name} needs unit stride")
        n = kv_len.numel()
        if q_start.numel() != n + 1 or page_table.shape[0] != n:
            raise ValueError(f"KVBatch: {q_start.numel()} starts and {page_table.shape[0]} table rows for {n} sequences")
        if n > 1 and page_table.numel() and page_table.stride(0) < page_table.shape[1]:
            raise ValueError(f"KVBatch: the rows of page_table overlap (strides {page_table.stride()}); give each sequence its own")
        if n_tokens is None:
            n_tokens = int(q_start[-1])
        if max_q is None:
            max_q = int((q_start[1:] - q_start[:-1]).max()) if n else 0
        if max_kv is None:
            max_kv = int(kv_len.max()) if n else 0
        self.q_start, self.kv_len, self.page_table = q_start, kv_len, page_table
        self.device = q_start.device
        self.n_seqs, self.n_tokens = n, int(n_tokens)
        self.c = _lib.KvBatch(n_seqs=n, n_tokens=int(n_tokens), max_q=int(max_q), max_kv=int(max_kv),
                              q_start=q_start.data_ptr(), kv_len=kv_len.data_ptr(), page_table=page_table.data_ptr(),
                              table_stride=max(page_table.stride(0), page_table.shape[1]) if n > 1
                              else page_table.shape[1], max_pages=page_table.shape[1])
        self._ref = ctypes.addressof(self.c)
        self._need: Dict[Tuple[int, int, int, int], int] = {}  # workspace bytes by (device, heads, kv heads, head_dim)


class Rope:
    """Rotary embedding of the first ``rot_dim`` dimensions (``opc_rope``): pair i turns by
    position * theta^(-2i/rot_dim), or by position * inv_freq[i] (radians, float64) when given.
    Pairs are (i, i + rot_dim/2), or (2i, 2i + 1) with ``interleaved``."""

    def __init__(self, rot_dim: int, theta: float = 10000.0, inv_freq=None, interleaved: bool = False, device=None):
        if rot_dim < 16 or rot_dim % 16:
            raise ValueError(f"Rope: rot_dim must be a positive multiple of 16, got {rot_dim}")
        if inv_freq is None:
            f = float(theta) ** (-np.arange(0, rot_dim, 2, dtype=np.float64) / rot_dim)
        else:
            f = np.ascontiguousarray(np.asarray(inv_freq, dtype=np.float64).reshape(-1))
        if f.size != rot_dim // 2:
            raise ValueError(f"Rope: {f.size} frequencies for rot_dim {rot_dim}")
        turns = np.zeros(f.size, dtype=np.uint64)
        _lib.check(_lib.load().opc_rope_turns(f.ctypes.data, f.size, turns.ctypes.data))
        self.device = _as_cuda_device(device)
        self.turns = torch.from_numpy(turns.view(np.int64)).to(self.device)
        self.rot_dim, self.interleaved = int(rot_dim), bool(interleaved)
        self.c = _lib.Rope(rot_dim=self.rot_dim, interleaved=int(self.interleaved), turns=self.turns.data_ptr())
        self._ref = ctypes.addressof(self.c)


def _rows(what: str, name: str, t: torch.Tensor, n: int, heads: Optional[int], hd: int, dtype, device) -> Tuple[int, int]:
    """(leading dimension, heads) of rows t [n, heads, head_dim] or [n, heads * head_dim]."""
    shape, stride = t.shape, t.stride()
    if len(shape) == 3:
        h = shape[1]
        ok = shape[2] == hd and stride[2] == 1 and (h == 1 or stride[1] == hd)
    else:
        h = shape[1] // hd if len(shape) == 2 else 0
        ok = len(shape) == 2 and shape[1] == h * hd and stride[1] == 1
    if not ok or h < 1 or shape[0] != n or (heads is not None and h != heads):
        raise ValueError(f"{what}: {name} must be [{n}, {heads if heads is not None else 'heads'}, {hd}] with "
                         f"contiguous heads, got {tuple(shape)} with strides {stride}")
    if t.device != device or t.dtype != dtype or dtype not in _HALVES:
        raise ValueError(f"{what}: {name} must be float16 or bfloat16 like the others on {device}, got {t.dtype} on {t.device}")
    return (stride[0] if n > 1 else h * hd), h


def _same_device(what: str, cache: KVCache, batch: KVBatch):
    if batch.device != cache.device:
        raise ValueError(f"{what}: the batch is on {batch.device}, the cache on {cache.device}")


def append(cache: KVCache, batch: KVBatch, k: torch.Tensor, v: torch.Tensor, q: Optional[torch.Tensor] = None,
           rope: Optional[Rope] = None, q_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Store the batch's rows of k (turned by ``rope``) and v; with q, return q turned (in ``q_out``,
    which may be q, or a new tensor)."""
    hd, dev = cache.head_dim, cache.device
    _same_device("append", cache, batch)
    ldk, _ = _rows("append", "k", k, batch.n_tokens, cache.kv_heads, hd, k.dtype, dev)
    ldv, _ = _rows("append", "v", v, batch.n_tokens, cache.kv_heads, hd, k.dtype, dev)
    ldq = ldo = heads = 0
    qp = op = None
    if q is not None:
        ldq, heads = _rows("append", "q", q, batch.n_tokens, None, hd, k.dtype, dev)
        if q_out is None:
            q_out = torch.empty_like(q, memory_format=torch.contiguous_format)  # (half of torch.empty's time)
        ldo, _ = _rows("append", "q_out", q_out, batch.n_tokens, heads, hd, k.dtype, dev)
        qp, op = q.data_ptr(), q_out.data_ptr()
    elif q_out is not None:
        raise ValueError("append: q_out given without q")
    if rope is not None and rope.device != dev:
        raise ValueError(f"append: the rope is on {rope.device}, the cache on {dev}")
    _call(_lib.load().opc_kv_append, dev.index, cache._ref, batch._ref, heads, _DTYPES[k.dtype],
          rope._ref if rope is not None else None, k.data_ptr(), ldk, v.data_ptr(), ldv, qp, ldq, op, ldo,
          _raw_stream(dev.index))
    return q_out


def read(cache: KVCache, batch: KVBatch, dtype: torch.dtype = torch.float16, k: Optional[torch.Tensor] = None,
         v: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """(k, v) [n_tokens, kv_heads, head_dim] as the cache holds them at the batch's rows, in the given
    tensors or new ones.  Rows without a place in the cache are not written."""
    dev = cache.device
    _same_device("read", cache, batch)
    shape = (batch.n_tokens, cache.kv_heads, cache.head_dim)
    if k is None and v is None:
        k = cache.pages.new_empty(shape, dtype=dtype)
        v = torch.empty_like(k)
    elif k is None or v is None:
        raise ValueError("read: k and v go together")
    ldk, _ = _rows("read", "k", k, batch.n_tokens, cache.kv_heads, cache.head_dim, k.dtype, dev)
    ldv, _ = _rows("read", "v", v, batch.n_tokens, cache.kv_heads, cache.head_dim, k.dtype, dev)
    _call(_lib.load().opc_kv_read, dev.index, cache._ref, batch._ref, _DTYPES[k.dtype], k.data_ptr(), ldk, v.data_ptr(), ldv,
          _raw_stream(dev.index))
    return k, v


def attention_workspace_bytes(cache: KVCache, batch: KVBatch, heads: int) -> int:
    key = (cache.device.index, heads, cache.kv_heads, cache.head_dim)
    need = batch._need.get(key)
    if need is None:
        need = batch._need[key] = int(_lib.load().opc_kv_attention_workspace_bytes(cache._ref, batch._ref, int(heads),
                                                                                  cache.device.index))
    return need


def attention(cache: KVCache, batch: KVBatch, q: torch.Tensor, scale: Optional[float] = None,
              out: Optional[torch.Tensor] = None, return_lse: bool = False,
              workspace: Optional[torch.Tensor] = None):
    """Causal attention of the rows q [n_tokens, heads, head_dim] over the cache: out, or (out, lse)
    with lse [n_tokens, heads] fp32.  ``scale``: 1/sqrt(head_dim) by default.  ``workspace``: zeroed
    uint8 memory of ``attention_workspace_bytes`` that no other call in flight uses (one per stream
    by default).  Rows that belong to no sequence are not written."""
    hd, dev = cache.head_dim, cache.device
    _same_device("attention", cache, batch)
    ldq, heads = _rows("attention", "q", q, batch.n_tokens, None, hd, q.dtype, dev)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    ldo, _ = _rows("attention", "out", out, batch.n_tokens, heads, hd, q.dtype, dev)
    lse = q.new_empty((batch.n_tokens, heads), dtype=torch.float32) if return_lse else None
    stream = _raw_stream(dev.index)
    if workspace is None:
        workspace = _workspace(dev, stream, attention_workspace_bytes(cache, batch, heads), "kv")
    else:
        _check_workspace("attention", workspace, dev)
    _call(_lib.load().opc_kv_attention, dev.index, cache._ref, batch._ref, heads, _DTYPES[q.dtype],
          hd ** -0.5 if scale is None else float(scale), q.data_ptr(), ldq, out.data_ptr(), ldo,
          lse.data_ptr() if return_lse else None, workspace.data_ptr(), workspace.numel(), stream)
    return (out, lse) if return_lse else out
