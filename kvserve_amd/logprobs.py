"""Log probabilities of given tokens, with entropy and the likeliest alternatives, in one pass over the logits
(kvh_token_logprobs): what a serving engine answers `logprobs` requests and scores prompts with."""

from __future__ import annotations

from typing import NamedTuple

import torch

from kvserve_amd import _lib
from kvserve_amd.attention import _calls, _check_index, _current, _require, _stream_handle

MAX_TOP = 64  # alternatives of a row at most


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor  # fp32 [T]: log softmax(logits)[token]
    entropy: torch.Tensor  # fp32 [T]: -sum p log p
    top_logprobs: torch.Tensor  # fp32 [T, top], descending
    top_ids: torch.Tensor  # int64 [T, top]; equal logits by ascending id


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0) -> TokenLogprobs:
    """logits: [T, vocab] on a HIP device (fp32, fp16 or bf16, any row stride, contiguous last dim); tokens: int64 [T];
    top: alternatives per row, 0 .. MAX_TOP.

    Statistics in fp32 whatever the logits' type. A logit of -inf is a token that cannot be; a row with a NaN or a +inf,
    or of -inf alone, gives NaN, as does a token outside the vocabulary (its row's other outputs are unaffected). NaN counts
    as -inf in the order of the alternatives. Forward only: the outputs carry no gradient, whatever the logits require."""
    calls = _calls()
    if calls is not None:
        r = calls.token_logprobs(logits, tokens, top)
        if r is not None:
            return TokenLogprobs(*r)
    _require(logits.dim() == 2 and logits.stride(-1) == 1, "logits must be [T, vocab] with a contiguous last dim")
    _require(logits.is_cuda, "logits must be on a HIP device")
    _require(logits.dtype in _lib.KVH_DTYPE, f"unsupported dtype {logits.dtype} (float32, float16, bfloat16)")
    if tokens.get_device() != logits.get_device():
        raise ValueError(f"tokens must be on the logits' device {logits.device} (got {tokens.device})")
    _check_index(tokens, "tokens", 1)
    rows, vocab = logits.shape
    _require(tokens.shape[0] == rows, "one token per row of logits")
    _require(0 <= top <= min(MAX_TOP, vocab), f"top must be 0 .. {min(MAX_TOP, vocab)} (got {top})")
    dev, dtype = logits.device, _lib.KVH_DTYPE[logits.dtype]
    stats = torch.empty((2, rows), dtype=torch.float32, device=dev)
    top_logprobs = torch.empty((rows, top), dtype=torch.float32, device=dev)
    top_ids = torch.empty((rows, top), dtype=torch.int64, device=dev)
    got = TokenLogprobs(stats[0], stats[1], top_logprobs, top_ids)
    if rows == 0:
        return got
    lib = _lib.load()
    need = lib.kvh_token_logprobs_workspace_size(rows, vocab, top, dtype)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    with _current(logits.get_device()):
        st = lib.kvh_token_logprobs(
            logits.data_ptr(), logits.stride(0), tokens.data_ptr(), stats.data_ptr(), stats.data_ptr() + 4 * rows,
            top_logprobs.data_ptr() if top else None, top_ids.data_ptr() if top else None, rows, vocab, top, dtype,
            ws.data_ptr() if ws is not None else None, need, _stream_handle(dev),
        )  # fmt: skip
    _lib.check(st, "kvh_token_logprobs")
    return got
