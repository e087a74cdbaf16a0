"""Log probabilities of given tokens, with entropy, rank and the best
alternatives, on the B200 kernel: what a server answers beside a token, and
what scoring a text with a quantised pack sums up."""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _native as _n

MAX_TOP = 32
_IDS = {torch.int32: _n.DT_I32, torch.int64: _n.DT_I64}


class TokenLogprobs(NamedTuple):
    logprob: torch.Tensor       # fp32 [rows]
    entropy: torch.Tensor       # fp32 [rows], nats
    rank: torch.Tensor          # int32 [rows], 1: the most likely; 0: no such token
    top_logprobs: torch.Tensor  # fp32 [rows, top], descending
    top_ids: torch.Tensor       # int32 [rows, top]


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, top: int = 0) -> TokenLogprobs:
    """log softmax of ``logits`` (fp32, fp16 or bf16 [rows, vocab]) at
    ``tokens`` (int32 or int64 [rows]) in one pass over the logits, computed in
    fp32.  Equal logits rank lowest index first.  Tokens outside the vocabulary
    (padding) get logprob -inf and rank 0.  ``top``: 0 to 32 alternatives."""
    who = "token_logprobs"
    _n.require_cuda(logits, tokens, who=who)
    if logits.dim() != 2 or not logits.is_floating_point():
        raise ValueError(f"{who}: logits must be fp32, fp16 or bf16 [rows, vocab]")
    x = _n.dtype_code(logits)
    rows, vocab = logits.shape
    ids = _IDS.get(tokens.dtype)
    if ids is None or tokens.shape != (rows,):
        raise ValueError(f"{who}: tokens must be int32 or int64 [{rows}]")
    if not 0 <= top <= min(MAX_TOP, vocab):
        raise ValueError(f"{who}: top must be in 0..{min(MAX_TOP, vocab)}")
    if logits.stride(1) != 1 or (rows > 1 and logits.stride(0) < vocab):
        logits = logits.contiguous()
    tokens = tokens.contiguous()
    dev = logits.device
    # one buffer: logprob, entropy, rank, alternatives
    buf = torch.empty(rows * (3 + 2 * top), dtype=torch.float32, device=dev)
    if rows:
        with _n.on_device(dev):
            lib = _n.load()
            stream = _n.raw_stream(dev)
            ws = _n.zeroed_workspace(dev, lib.exl3_token_logprobs_workspace_size(rows, vocab, top, x), stream)
            at, n = buf.data_ptr(), 4 * rows
            _n.check(lib.exl3_token_logprobs(
                logits.data_ptr(), x, rows, logits.stride(0), vocab, tokens.data_ptr(), ids, top, at, at + n,
                at + 2 * n, at + 3 * n, at + (3 + top) * n, ws.data_ptr(), ws.numel(), stream), who)
    lp, ent, rank, tlp, tid = buf.split((rows, rows, rows, rows * top, rows * top))
    return TokenLogprobs(lp, ent, rank.view(torch.int32), tlp.view(rows, top), tid.view(torch.int32).view(rows, top))


__all__ = ["MAX_TOP", "TokenLogprobs", "token_logprobs"]
