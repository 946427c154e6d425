"""Log probabilities of given tokens, entropy and top alternatives (``opc_token_logprobs``)."""

from __future__ import annotations

import functools
from typing import NamedTuple, Optional

import torch

from . import _lib
from .kv import _DTYPES, _call, _check_workspace, _raw_stream, _workspace


class TokenLogprobs(NamedTuple):
    """What ``token_logprobs`` returns; parts that were not asked for are None."""

    logprob: Optional[torch.Tensor]       # [rows] fp32
    entropy: Optional[torch.Tensor]       # [rows] fp32
    top_ids: Optional[torch.Tensor]       # [rows, top_k] int32
    top_logprobs: Optional[torch.Tensor]  # [rows, top_k] fp32


@functools.lru_cache(maxsize=256)
def _need(rows: int, vocab: int, top_k: int, device: int) -> int:
    return int(_lib.load().opc_token_logprobs_workspace_bytes(rows, vocab, top_k, device))


def token_logprobs(logits: torch.Tensor, targets: Optional[torch.Tensor] = None, top_k: int = 0,
                   entropy: bool = True, workspace: Optional[torch.Tensor] = None) -> TokenLogprobs:
    """For every row of logits [rows, vocab] (float16, bfloat16 or float32, any row stride from vocab on): the log
    probability of its target (int32 or int64 [rows]; negative: none, 0), the entropy, and the top_k
    (at most 32) most probable tokens with their log probabilities, equal logits by the lower id.
    There is no backward pass: the results carry no gradient."""
    if logits.dim() != 2 or not logits.is_cuda or logits.dtype not in _DTYPES or (logits.numel() and logits.stride(1) != 1):
        raise ValueError(f"token_logprobs: logits must be float16, bfloat16 or float32 [rows, vocab] on a CUDA device with "
                         f"unit stride, got {logits.dtype} {tuple(logits.shape)} on {logits.device}")
    rows, vocab = logits.shape
    dev = logits.device
    if targets is not None:
        if targets.dtype not in (torch.int32, torch.int64) or tuple(targets.shape) != (rows,) or targets.device != dev:
            raise ValueError(f"token_logprobs: targets must be int32 or int64 [{rows}] on {dev}, got {targets.dtype} "
                             f"{tuple(targets.shape)} on {targets.device}")
        if targets.dtype == torch.int64:  # ids beyond int32 stay outside the vocabulary
            targets = targets.clamp(-1, 2**31 - 1).to(torch.int32)
        targets = targets.contiguous()
    logprob = torch.empty(rows, dtype=torch.float32, device=dev) if targets is not None else None
    ent = None
    if entropy:
        ent = torch.empty_like(logprob) if logprob is not None else torch.empty(rows, dtype=torch.float32, device=dev)
    ids = torch.empty(rows, top_k, dtype=torch.int32, device=dev) if top_k >= 0 else None
    top = torch.empty(rows, top_k, dtype=torch.float32, device=dev) if top_k >= 0 else None
    lib = _lib.load()
    stream = _raw_stream(dev.index)
    if workspace is None:
        workspace = _workspace(dev, stream, _need(rows, vocab, top_k, dev.index), "score")
    else:
        _check_workspace("token_logprobs", workspace, dev)
    _call(lib.opc_token_logprobs, dev.index, logits.data_ptr(), logits.stride(0) if rows > 1 else vocab,
          _DTYPES[logits.dtype], rows, vocab, targets.data_ptr() if targets is not None else None,
          logprob.data_ptr() if logprob is not None else None, ent.data_ptr() if ent is not None else None, top_k,
          ids.data_ptr() if ids is not None else None, top.data_ptr() if top is not None else None,
          workspace.data_ptr(), workspace.numel(), stream)
    return TokenLogprobs(logprob, ent, ids, top)
