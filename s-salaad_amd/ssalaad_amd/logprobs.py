"""Log probabilities of given tokens, with the entropy and the top alternatives.

The reference's generation returns tokens only
(ssalaad/inference/generate.py:12-26); a server that scores prompts or reports
alternatives reads them off the logits `DecodeEngine.step` or a model returns.
"""

from __future__ import annotations

import struct
from typing import NamedTuple

import torch

from . import _lib
from .paged import _call

_ARGS = struct.Struct("=12q")  # ssl_token_logprobs_args


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor      # [rows] fp32: log p(token)
    entropy: torch.Tensor       # [rows] fp32: −Σ p log p
    top_ids: torch.Tensor       # [rows, top] int64, most likely first, ties by lower index
    top_logprobs: torch.Tensor  # [rows, top] fp32


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, top: int = 0) -> TokenLogprobs:
    """Scores of `tokens` [rows] (int64) under `logits` [rows, vocab] (float32,
    bfloat16 or float16): log probabilities, entropies and the `top` (up to 64)
    most likely tokens. Logits of -inf have probability 0. A token outside
    [0, vocab) scores NaN, as does every value of a row that holds a NaN, a +inf
    or nothing above -inf. There is no gradient: logits that require one give plain
    values. The four outputs share one allocation, which any of them keeps. Runs
    on torch's current stream; nothing synchronises.
    """
    out = _lib.tensorcall().logprobs(logits, tokens, top)
    if out is not None:
        return TokenLogprobs(*_lib.completed(out, "ssl_token_logprobs"))
    if not logits.is_cuda:
        raise ValueError("token_logprobs runs on a ROCm GPU device; move the logits there first")
    if logits.dim() != 2 or logits.shape[1] == 0:
        raise ValueError(f"logits must be [rows, vocab], got {tuple(logits.shape)}")
    dev = logits.device
    rows, vocab = logits.shape
    dt = _lib.dtype_code(logits.dtype)
    if tokens.dtype is not torch.int64:
        raise TypeError(f"tokens must be int64, got {tokens.dtype}")
    if tokens.shape != (rows,) or tokens.device != dev:
        raise ValueError(f"tokens must be [{rows}] on {dev}")
    if not 0 <= top <= min(vocab, 64):
        raise ValueError(f"top must lie in [0, {min(vocab, 64)}], got {top}")
    if logits.stride(1) != 1 or (rows > 1 and logits.stride(0) < vocab):
        logits = logits.contiguous()
    if not tokens.is_contiguous():
        tokens = tokens.contiguous()
    logprob, entropy = torch.empty((2, rows), dtype=torch.float32, device=dev).unbind()
    ids = torch.empty((rows, top), dtype=torch.int64, device=dev)
    top_logprobs = torch.empty((rows, top), dtype=torch.float32, device=dev)
    if rows:
        ld = logits.stride(0) if rows > 1 else vocab
        _call("ssl_token_logprobs", _ARGS.pack(
            _ARGS.size, logits.data_ptr(), ld, rows, vocab, tokens.data_ptr(), top,
            logprob.data_ptr(), entropy.data_ptr(), ids.data_ptr(), top_logprobs.data_ptr(), dt),
            dev)
    return TokenLogprobs(logprob, entropy, ids, top_logprobs)
