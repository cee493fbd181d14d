"""Log probabilities of tokens from logits: what a served request that asks for them is answered with, and how texts are scored."""
from __future__ import annotations

import struct
from typing import NamedTuple, Optional

import torch

from .. import _native
from .kernels import OperandError, _DT, _check

MAX_TOP = 32
_CALL = struct.Struct("=7Q3q4i")            # the launcher's call record (token_logprobs.cu)


class TokenLogprobs(NamedTuple):
    """Per row: log probability and rank (1: the most likely) of the given token, entropy of the row in nats, and the ``top``
    most likely tokens with their log probabilities."""
    logprob: torch.Tensor          # fp32 [rows]
    rank: torch.Tensor             # int32 [rows]
    entropy: torch.Tensor          # fp32 [rows]
    top_ids: torch.Tensor          # int32 [rows, top]
    top_logprobs: torch.Tensor     # fp32 [rows, top]


def token_logprobs(logits: torch.Tensor, tokens: Optional[torch.Tensor] = None, top: int = 0) -> TokenLogprobs:
    """``logits``: fp32, bf16 or fp16 [rows, vocab], row stride free.  ``tokens``: int32 or int64 [rows]; a token outside
    [0, vocab), -1 for instance, is none: its log probability and rank are 0 (all are without ``tokens``).  ``top``: up to 32
    alternatives.  Equal logits rank by index, the lower first.  A row whose logits are all -inf gives every token -inf and
    an entropy of 0; NaN or +inf among the logits makes the row's figures NaN (ranks count NaN as largest)."""
    if logits.dim() != 2 or logits.dtype not in _DT or logits.device.type != "cuda":
        raise OperandError(f"token_logprobs needs a matrix of fp32, bf16 or fp16 logits on a CUDA device, got {logits.dtype} "
                           f"{tuple(logits.shape)} on {logits.device}")
    rows, vocab = logits.shape
    if vocab < 1 or vocab > 2 ** 30 or (logits.stride(1) != 1 and vocab > 1):
        raise OperandError(f"logits must have a vocabulary and unit column stride, got {tuple(logits.shape)}, strides {logits.stride()}")
    if not 0 <= int(top) <= min(MAX_TOP, vocab):
        raise OperandError(f"top is {top}; up to {min(MAX_TOP, vocab)} alternatives of {vocab} tokens")
    index = logits.get_device()
    if tokens is not None:
        if tokens.dtype not in (torch.int32, torch.int64) or tokens.dim() != 1 or tokens.numel() != rows or tokens.get_device() != index:
            raise OperandError(f"tokens must be {rows} int32 or int64 values on {logits.device}, got {tokens.dtype} {tuple(tokens.shape)} on "
                               f"{tokens.device}")
    if index != torch._C._cuda_getDevice():
        with torch.cuda.device(index):
            return token_logprobs(logits, tokens, top)
    top = int(top)
    f, i = logits.new_empty(((2 + top) * rows,), dtype=torch.float32), logits.new_empty(((1 + top) * rows,), dtype=torch.int32)
    logprob, entropy, tops = f.split((rows, rows, top * rows))
    rank, ids = i.split((rows, top * rows))
    at, ints = f.data_ptr(), i.data_ptr()
    token_ptr, stride, wide = 0, 0, 0
    if tokens is not None:
        token_ptr, stride, wide = tokens.data_ptr(), tokens.stride(0) if rows > 1 else 1, int(tokens.dtype is torch.int64)
    rc = _native.cuda().ronn_token_logprobs(_CALL.pack(logits.data_ptr(), token_ptr, at, at + 4 * rows, at + 8 * rows, ints, ints + 4 * rows,
                                                       logits.stride(0) if rows > 1 else vocab, rows, stride, vocab, wide, top,
                                                       _DT[logits.dtype]), torch._C._cuda_getCurrentRawStream(index))
    _check(rc, "token_logprobs")
    return TokenLogprobs(logprob, rank, entropy, ids.view(rows, top), tops.view(rows, top))
