"""Log probabilities of given tokens, with entropy, rank and the best
alternatives, on the B200 kernel: what a server answers beside a token, and
what scoring a text with a quantised pack sums up."""

from __future__ import annotations

import functools
from typing import NamedTuple

import torch

from . import _native as _n

MAX_TOP = 32
_LOGITS = {torch.float32: _n.DT_F32, torch.float16: _n.DT_F16, torch.bfloat16: _n.DT_BF16}
_IDS = {torch.int32: _n.DT_I32, torch.int64: _n.DT_I64}


class TokenLogprobs(NamedTuple):
    logprob: torch.Tensor       # fp32 [rows]
    entropy: torch.Tensor       # fp32 [rows], nats
    rank: torch.Tensor          # int32 [rows], 1: the most likely; 0: no such token
    top_logprobs: torch.Tensor  # fp32 [rows, top], descending
    top_ids: torch.Tensor       # int32 [rows, top]


@functools.lru_cache(maxsize=256)
def _workspace_bytes(device: int, rows: int, vocab: int, top: int, x: int) -> int:
    return _n.load().exl3_token_logprobs_workspace_size(rows, vocab, top, x)


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, top: int = 0) -> TokenLogprobs:
    """log softmax of ``logits`` (fp32, fp16 or bf16 [rows, vocab]) at
    ``tokens`` (int32 or int64 [rows]) in one pass over the logits, computed in
    fp32.  Equal logits rank lowest index first.  Tokens outside the vocabulary
    (padding) get logprob -inf and rank 0.  ``top``: 0 to 32 alternatives.  For
    inference: a backward pass through the result raises."""
    short = _n.binding().token_logprobs(logits, tokens, top)
    if short is not None:
        return TokenLogprobs(*short)
    x, ids = _LOGITS.get(logits.dtype), _IDS.get(tokens.dtype)
    who = "token_logprobs"
    _n.require_one_device(logits, tokens, who=who)
    if not (x is not None and ids is not None and logits.dim() == 2 and tokens.shape == logits.shape[:1]
            and 0 <= top <= MAX_TOP and top <= logits.size(1)):
        if x is None or logits.dim() != 2:
            raise ValueError(f"{who}: logits must be fp32, fp16 or bf16 [rows, vocab]")
        if ids is None or tokens.shape != logits.shape[:1]:
            raise ValueError(f"{who}: tokens must be int32 or int64 [{logits.size(0)}]")
        raise ValueError(f"{who}: top must be in 0..{min(MAX_TOP, logits.size(1))}")
    dev = logits.device.index
    if dev != _n.current_device():
        with torch.cuda.device(dev):
            return token_logprobs(logits, tokens, top=top)
    rows, vocab = logits.shape
    row_stride, step = logits.stride()
    if step != 1 or (rows > 1 and row_stride < vocab):
        logits = logits.clone(memory_format=torch.contiguous_format)
        row_stride = vocab
    if not tokens.is_contiguous():
        tokens = tokens.contiguous()

    def result(t):
        return _n.inference_only("token_logprobs", t, logits)

    # one buffer: logprob and entropy, the alternatives' values; rank, their ids
    buf = logits.new_empty(rows * (2 + top), dtype=torch.float32)
    whole = logits.new_empty(rows * (1 + top), dtype=torch.int32)
    if rows:
        stream = _n.raw_stream(dev)
        ws, ws_bytes = _n.serve_workspace(dev, stream, _workspace_bytes(dev, rows, vocab, top, x))
        at, to, n = buf.data_ptr(), whole.data_ptr(), 4 * rows
        rc = _n.load().exl3_token_logprobs(_n.PACK_TOKEN_LOGPROBS(
            logits.data_ptr(), x, rows, row_stride, vocab, tokens.data_ptr(), ids, top, at, at + n, to, at + 2 * n,
            to + n, ws, ws_bytes), stream)
        if rc:
            _n.check(rc, "token_logprobs")
    if top == 0:
        lp, ent = torch.unsafe_split_with_sizes(buf, (rows, rows))
        return TokenLogprobs(result(lp), result(ent), whole, buf.new_empty((rows, 0)), whole.new_empty((rows, 0)))
    lp, ent, vals = torch.unsafe_split_with_sizes(buf, (rows, rows, rows * top))
    rank, best = torch.unsafe_split_with_sizes(whole, (rows, rows * top))
    return TokenLogprobs(result(lp), result(ent), rank, result(vals.view(rows, top)), best.view(rows, top))


__all__ = ["MAX_TOP", "TokenLogprobs", "token_logprobs"]
