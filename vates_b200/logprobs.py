"""Log probabilities of given tokens, with rank, entropy and the best
alternatives, in one pass over the logits (``vb_token_logprobs``)."""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple

import torch

from ._lib import VB_TOKEN_LOGPROBS_WORKSPACE_HEAD, VbTokenLogprobsArgs, check, lib
from .pool import current_device, current_stream, on_device, status_ptr
from .scratch import Scratch

MAX_TOP = 32
_DTYPES = {torch.bfloat16: 0, torch.float32: 1}
_scratch = Scratch(VB_TOKEN_LOGPROBS_WORKSPACE_HEAD)  # rows split over several CTAs
_needs: dict = {}  # its bytes by (rows, vocab, top)


class TokenLogprobs(NamedTuple):
    logprob: torch.Tensor       # float32 [rows]: log p of the row's token
    rank: torch.Tensor          # int32 [rows]: tokens ahead of it (0: the most likely)
    entropy: torch.Tensor       # float32 [rows], nats
    top_ids: torch.Tensor       # int32 [rows, top], best first, ties to the lowest id
    top_logprobs: torch.Tensor  # float32 [rows, top]


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0,
                   temperature: float = 1.0, status=None, stream=None) -> TokenLogprobs:
    """``log_softmax(logits / temperature)`` of row ``r`` at ``tokens[r]`` and
    what a server reports beside it.

    ``logits`` bf16 or float32 ``[rows, vocab]`` (any row stride), ``tokens``
    int32 ``[rows]``, ``top`` alternatives (0 to 32). Logits of -inf are tokens
    that cannot follow. A NaN or +inf in a row makes its floating results NaN;
    a token outside the vocabulary gives NaN and rank -1 and sets
    VB_STATUS_BOUNDS in ``status``."""
    dev = logits.get_device()
    # with it as the current stream, results belong to it
    if dev >= 0 and (stream is not None or current_device() != dev):
        with on_device(logits.device, stream):
            return token_logprobs(logits, tokens, top, temperature, status)
    if logits.dim() != 2 or logits.dtype not in _DTYPES or dev < 0:
        raise ValueError("logits: bfloat16 or float32 CUDA [rows, vocab] are needed, got "
                         f"{logits.dtype} {tuple(logits.shape)} on {logits.device}")
    rows, vocab = logits.shape
    if tokens.dtype != torch.int32 or tuple(tokens.shape) != (rows,) \
            or tokens.get_device() != dev or not tokens.is_contiguous():
        raise ValueError(f"tokens: contiguous int32 [{rows}] on {logits.device} is needed, got "
                         f"{tokens.dtype} {tuple(tokens.shape)} on {tokens.device}")
    if not 0 <= top <= min(MAX_TOP, vocab):
        raise ValueError(f"top={top}: 0 to {MAX_TOP} and at most the vocabulary ({vocab})")
    if logits.stride(1) != 1 and vocab > 1:
        logits = logits.contiguous()
    lp = logits.new_empty(rows, dtype=torch.float32)
    ent = torch.empty_like(lp)
    rank = torch.empty_like(tokens)
    tlp = lp.new_empty((rows, top))
    ids = rank.new_empty((rows, top))
    st = current_stream(dev)
    need = _needs.get((rows, vocab, top))
    if need is None:
        if len(_needs) > 4096:
            _needs.clear()
        need = _needs[rows, vocab, top] = max(
            1 << 16, lib.vb_token_logprobs_workspace_size(rows, vocab, top))
    ws = _scratch.get(need, logits.device, st)
    a = VbTokenLogprobsArgs(logits.data_ptr(), tokens.data_ptr(), lp.data_ptr(), ent.data_ptr(),
                            rank.data_ptr(), ids.data_ptr(), tlp.data_ptr(),
                            None if status is None else status_ptr(status, dev),
                            ws.data_ptr(), ws.numel(), logits.stride(0), temperature, rows, vocab,
                            top, _DTYPES[logits.dtype])
    check(lib.vb_token_logprobs(C.byref(a), st), "vb_token_logprobs")
    return TokenLogprobs(lp, rank, ent, ids, tlp)


__all__ = ["TokenLogprobs", "token_logprobs"]
