"""Low-rank adapters of many requests beside a projection that all of them share."""
from __future__ import annotations

import torch

from .. import _lib

MAX_RANK, MAX_ROWS, MAX_WIDTH = 128, 1 << 20, 1 << 24


def stack_adapters(adapters, device=None, dtype=None):
    """[(A [r, K], B [N, r], scale)] of any ranks -> the stacked (a [S, R, K], b [S, N, R], scale fp32 [S], rank int32 [S]) of ``add_adapters``,
    R the largest rank rounded up to 8 (rows of whole 16-byte pieces)."""
    if not adapters:
        raise ValueError("at least one adapter is wanted")
    first = adapters[0][0]
    device, dtype = device or first.device, dtype or first.dtype
    K, N = first.shape[1], adapters[0][1].shape[0]
    for i, (a, b, _) in enumerate(adapters):
        if a.dim() != 2 or b.dim() != 2 or a.shape[1] != K or b.shape[0] != N or a.shape[0] != b.shape[1] or not 1 <= a.shape[0] <= MAX_RANK:
            raise ValueError(f"adapter {i}: A [r, {K}] and B [{N}, r] of a rank r of 1 to {MAX_RANK} are wanted, got {tuple(a.shape)} and {tuple(b.shape)}")
    R = (max(a.shape[0] for a, _, _ in adapters) + 7) // 8 * 8
    sa, sb = torch.zeros(len(adapters), R, K, dtype=dtype, device=device), torch.zeros(len(adapters), N, R, dtype=dtype, device=device)
    for i, (a, b, _) in enumerate(adapters):
        sa[i, :a.shape[0]] = a.to(device=device, dtype=dtype)
        sb[i, :, :a.shape[0]] = b.to(device=device, dtype=dtype)
    return (sa, sb, torch.tensor([float(s) for _, _, s in adapters], dtype=torch.float32, device=device),
            torch.tensor([a.shape[0] for a, _, _ in adapters], dtype=torch.int32, device=device))


def add_adapters(base, x, a, b, adapter, scale=None, rank=None, out=None):
    """``out[t] = base[t] + scale[i] b[i] (a[i] x[t])`` with ``i = adapter[t]``; rows whose number is none of the adapters' (-1) are their base.

    base, out: fp32 ``[T, N]`` (out may be base, and shares no memory with the others; None: a new tensor); x ``[T, K]``, a ``[S, R, K]``, b ``[S, N, R]`` of one type (bf16, fp16, fp32);
    adapter int32 ``[T]``; scale fp32 ``[S]``; rank int32 ``[S]``: how many of an adapter's R rows count (None: all).  All contiguous, on one GPU.
    """
    if x.dim() != 2 or a.dim() != 3 or b.dim() != 3:
        raise ValueError(f"x [T, K], a [S, R, K] and b [S, N, R] are wanted, got {[tuple(t.shape) for t in (x, a, b)]}")
    (T, K), (S, R, _), N, dev, dt = x.shape, a.shape, b.shape[1], x.device, x.dtype
    code = _lib.seq_dtype_code(dt)
    if dev.type != "cuda":
        raise ValueError(f"tensors on a GPU are wanted, got {dev}")
    if T > MAX_ROWS or max(N, K) > MAX_WIDTH:
        raise ValueError(f"up to {MAX_ROWS} rows of {MAX_WIDTH} values are possible, got x {tuple(x.shape)} and {N} columns")
    if S < 1 or not 1 <= R <= MAX_RANK or K < 1 or N < 1:
        raise ValueError(f"at least one adapter of a rank of 1 to {MAX_RANK} is wanted, got a of {tuple(a.shape)}")
    if out is None:
        out = torch.empty((T, N), dtype=torch.float32, device=dev)
    for what, t, shape, kind in (("a", a, (S, R, K), dt), ("b", b, (S, N, R), dt), ("base", base, (T, N), torch.float32), ("out", out, (T, N), torch.float32),
                                 ("adapter", adapter, (T,), torch.int32), ("scale", scale, (S,), torch.float32), ("rank", rank, (S,), torch.int32), ("x", x, (T, K), dt)):
        if t is not None and (t.shape != shape or t.dtype != kind or t.device != dev or not t.is_contiguous()):
            raise ValueError(f"{what}: a contiguous {kind} tensor {shape} on {dev} is wanted, got {t.dtype} {tuple(t.shape)} of strides {t.stride()} on {t.device}")
    if T:
        n = _lib.load_seq().umb_seq_adapters_floats(T, K, R)
        scratch = torch.empty(n, dtype=torch.float32, device=dev) if n else None
        _lib.seq_call_on(dev, "umb_seq_adapters", out, base, x, a, b, adapter, scale, rank, T, N, K, S, R, scratch, n, code)
    return out
