"""Log probabilities of given tokens with the entropy and the top alternatives of each row: what a server returns
beside the tokens it picks, or scores a prompt by. One kernel, one pass over the logits. The reference returns logits only
(kernels/e2e/model.py:248-253)."""

from __future__ import annotations

import torch

from kernels import _lib

MAX_TOP = 32
_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}


def token_logprobs(logits, targets, top=0):
    """logits [M, V] (fp16, bf16 or fp32, unit column stride, any row stride), targets int64 [M]. Returns (logprob fp32
    [M] of the targets, entropy fp32 [M] in nats, top_logprobs fp32 [M, top], top_ids int64 [M, top]: the `top` <= 32
    largest logits of each row, best first, ties to the lowest index). A negative target stands for no token: its log
    probability is 0. A target >= V gives NaN and sets the device error DK_DEVERR_BAD_TOKEN. Logits of -inf are tokens
    that cannot occur; a row with a NaN or +inf, or nothing but -inf, has NaN log probabilities."""
    what = "token_logprobs"
    _lib.require_extent(logits.dim() == 2 and logits.shape[1] > 0 and logits.stride(1) == 1,
                        f"{what}: logits must be [rows, vocab] with unit column stride")
    M, V = logits.shape
    _lib.require_extent(logits.stride(0) >= V or M <= 1, f"{what}: rows of logits overlap")
    _lib.require_extent(targets.dim() == 1 and targets.shape[0] == M and targets.is_contiguous(),
                        f"{what}: targets must hold one token per row")
    _lib.require_extent(0 <= top <= min(MAX_TOP, V), f"{what}: top must be 0..{MAX_TOP}, at most the vocabulary")
    if logits.dtype not in _DTYPES:
        raise RuntimeError(f"{what}: logits must be fp16, bf16 or fp32, got {logits.dtype}")
    if targets.dtype != torch.int64:
        raise RuntimeError(f"{what}: targets must be int64")
    _lib.require_cuda(what, logits, targets)
    dev = logits.device
    if targets.device != dev:
        raise RuntimeError(f"{what}: tensors on {dev} and {targets.device}")
    stats = torch.empty((2, M), dtype=torch.float32, device=dev)
    values = torch.empty((M, top), dtype=torch.float32, device=dev)
    ids = torch.empty((M, top), dtype=torch.int64, device=dev)
    lp, entropy = stats[0], stats[1]
    _lib.call("dk_token_logprobs", logits.data_ptr(), max(logits.stride(0), V), _DTYPES[logits.dtype], targets.data_ptr(),
              M, V, top, lp.data_ptr(), entropy.data_ptr(), values.data_ptr(), ids.data_ptr(),
              torch.cuda.current_stream(dev).cuda_stream)
    return lp, entropy, values, ids
