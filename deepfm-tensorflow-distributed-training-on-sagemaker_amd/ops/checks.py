"""Argument checks and launch context of the operators that allocate their own results
(``ops.experts``, ``ops.act8``).

Shapes, types and strides are checked before the device, so a wrong call is refused the same way
with or without a GPU.  Launches go to the current stream of the operands' device, whichever device
is current; nothing synchronizes, so calls can be captured into a HIP graph.  A small call's time is
the host's: the checks of a good call build no text.
"""
from __future__ import annotations

from typing import Optional, Sequence, Tuple

import torch

LIMIT = 1 << 31          # rows, columns: int32 in the kernels


def rows2d(t: torch.Tensor, what: str, dtypes: Sequence[torch.dtype], M: Optional[int] = None,
           N: Optional[int] = None) -> int:
    """``t`` is [M, N] of one of ``dtypes`` with unit column stride and rows that do not overlap.  Elements from a
    row to the next (of a single row: any that hold it)."""
    if isinstance(t, torch.Tensor) and t.dim() == 2 and t.dtype in dtypes:
        m, n = t.shape
        s0, s1 = t.stride()
        if ((M is None or m == M) and (N is None or n == N) and m < LIMIT and n < LIMIT
                and (((s1 == 1 or n == 1) and (s0 >= n or m == 1)) or m == 0 or n == 0)):
            return s0 if m > 1 or s0 > n else n
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{what} must be a tensor")
    if t.dim() != 2:
        raise ValueError(f"{what} must be 2-D, got {tuple(t.shape)}")
    if t.dtype not in dtypes:
        raise ValueError(f"{what} must be one of {[str(d) for d in dtypes]}, got {t.dtype}")
    if (M is not None and t.shape[0] != M) or (N is not None and t.shape[1] != N):
        raise ValueError(f"{what} must be [{'any' if M is None else M}, {'any' if N is None else N}], "
                         f"got {tuple(t.shape)}")
    if max(t.shape) >= LIMIT:
        raise ValueError(f"{what} is too large: {tuple(t.shape)}")
    raise ValueError(f"{what} must have adjacent columns and rows that do not overlap, got strides {t.stride()}")


def flat(t: torch.Tensor, what: str, dtype: torch.dtype, shape: tuple) -> None:
    """``t`` is a contiguous tensor of exactly this type and shape."""
    if not (isinstance(t, torch.Tensor) and t.dtype == dtype and t.shape == shape and t.is_contiguous()):
        got = f", got {t.dtype} {tuple(t.shape)}" if isinstance(t, torch.Tensor) else ""
        raise ValueError(f"{what} must be a contiguous {dtype} {tuple(shape)}{got}")


def out_or_new(out: Optional[torch.Tensor], M: int, N: int, dtype, device, what: str = "out") -> Tuple[torch.Tensor, int]:
    """``out`` or a new tensor, and its row stride."""
    if out is None:
        return torch.empty(M, N, dtype=dtype, device=device), N
    return out, rows2d(out, what, (dtype,), M, N)


def call(what: str, tensors, fn, *args) -> int:
    """``fn(*args, stream)`` on the current stream of the operands' device; refuses operands (None: not
    given) that are not on one GPU.  The result of ``fn``."""
    first = tensors[0]
    at = first.get_device()               # (-1: the host)
    for t in tensors:
        if t is not None and t.get_device() != at:
            raise ValueError(f"{what}: operands on {first.device} and {t.device}")
    if at < 0:
        raise ValueError(f"{what} runs on the GPU: operands are on {first.device}")
    if at == torch._C._cuda_getDevice():
        # (the handle itself: torch.cuda.current_stream() takes 5 us to wrap it)
        return fn(*args, torch._C._cuda_getCurrentRawStream(at))
    with torch.cuda.device(at):
        return fn(*args, torch._C._cuda_getCurrentRawStream(at))
