"""Tokens drawn for many requests at once, each with settings and a random number of its own.

The engines' ``umb_sample_rows`` has one setting for all rows of a call; a batch of requests has as many as it has rows.
"""
from __future__ import annotations

import torch

from .. import _lib

MAX_VOCAB = 1 << 19


def _per_row(what: str, v, rows: int, dtype, device):
    if v is None:
        return None
    if not isinstance(v, torch.Tensor):
        return torch.full((rows,), v, dtype=dtype, device=device)
    if v.shape != (rows,) or v.dtype != dtype or v.device != device or not v.is_contiguous():
        raise ValueError(f"{what}: a contiguous {dtype} tensor of {rows} values on {device} is wanted, got {v.dtype} {tuple(v.shape)} on {v.device}")
    return v


def sample_rows(logits, uniforms, temperature=None, top_k=None, top_p=None, min_p=None):
    """Draws one token per row of ``logits`` (fp32 ``[rows, V]``, rows any distance apart) from ``uniforms`` (fp32 ``[rows]`` in [0, 1)).

    ``temperature``, ``top_p``, ``min_p`` (fp32) and ``top_k`` (int32) are tensors of one value per row, or one number for all; None: 1, 1, 0
    and all.  A temperature of 0 takes the largest logit.  What each filter keeps: include/umbrella_seq.h, ``umb_sample_requests``.

    Returns (tokens int32 ``[rows]``, their shares of the kept mass fp32 ``[rows]``); -1 and 0 for a row that rules every token out.
    """
    if logits.dim() != 2 or logits.dtype != torch.float32 or logits.device.type != "cuda":
        raise ValueError(f"logits: an fp32 [rows, V] tensor on a GPU is wanted, got {logits.dtype} {tuple(logits.shape)} on {logits.device}")
    (rows, V), dev = logits.shape, logits.device
    if not 1 <= V <= MAX_VOCAB:
        raise ValueError(f"logits: 1 to {MAX_VOCAB} columns are wanted, got {V}")
    if rows > 0 and ((V > 1 and logits.stride(1) != 1) or (rows > 1 and logits.stride(0) < V)):
        raise ValueError(f"logits: rows of neighbouring values are wanted, got strides {logits.stride()}")
    if uniforms is None or not isinstance(uniforms, torch.Tensor):
        raise ValueError("uniforms: a random number per row is wanted")
    uniforms = _per_row("uniforms", uniforms, rows, torch.float32, dev)
    temperature, top_p, min_p = (_per_row(n, v, rows, torch.float32, dev) for n, v in (("temperature", temperature), ("top_p", top_p), ("min_p", min_p)))
    top_k = _per_row("top_k", top_k, rows, torch.int32, dev)
    tokens, probs = torch.empty(rows, dtype=torch.int32, device=dev), torch.empty(rows, dtype=torch.float32, device=dev)
    if rows:
        n = _lib.load_seq().umb_sample_requests_bytes(rows, V)
        scratch = torch.empty(n, dtype=torch.uint8, device=dev)
        _lib.seq_call_on(dev, "umb_sample_requests", tokens, probs, logits, logits.stride(0) if rows > 1 else V, rows, V, uniforms, temperature, top_k, top_p, min_p,
                         scratch, n)
    return tokens, probs
