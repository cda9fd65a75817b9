"""Argument checks and launch context of the operators that allocate their own results
(``ops.experts``, ``ops.act8``).

Shapes, types and strides are checked before the device, so a wrong call is refused the same way
with or without a GPU.  Launches go to the current stream of the operands' device, whichever device
is current; nothing synchronizes, so calls can be captured into a HIP graph.
"""
from __future__ import annotations

import contextlib
from typing import Optional, Sequence

import torch

LIMIT = 1 << 31          # rows, columns: int32 in the kernels


def need(ok: bool, msg: str) -> None:
    if not ok:
        raise ValueError(msg)


def contiguous(t: torch.Tensor) -> bool:
    return t.is_contiguous()


def row_stride(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[1])


def rows2d(t: torch.Tensor, what: str, dtypes: Sequence[torch.dtype], M: Optional[int] = None,
           N: Optional[int] = None) -> None:
    """``t`` is [M, N] of one of ``dtypes`` with unit column stride and rows that do not overlap."""
    need(isinstance(t, torch.Tensor), f"{what} must be a tensor")
    need(t.dim() == 2, f"{what} must be 2-D, got {tuple(t.shape)}")
    need(t.dtype in dtypes, f"{what} must be one of {[str(d) for d in dtypes]}, got {t.dtype}")
    need((M is None or t.shape[0] == M) and (N is None or t.shape[1] == N),
         f"{what} must be [{'any' if M is None else M}, {'any' if N is None else N}], got {tuple(t.shape)}")
    need(t.shape[0] < LIMIT and t.shape[1] < LIMIT, f"{what} is too large: {tuple(t.shape)}")
    if t.numel():
        need(t.shape[1] == 1 or t.stride(1) == 1, f"{what}'s columns must be adjacent")
        need(t.shape[0] == 1 or t.stride(0) >= t.shape[1], f"{what}'s rows must not overlap")


def flat(t: torch.Tensor, what: str, dtype: torch.dtype, shape) -> None:
    """``t`` is a contiguous tensor of exactly this type and shape."""
    need(isinstance(t, torch.Tensor) and t.dtype == dtype and tuple(t.shape) == tuple(shape) and contiguous(t),
         f"{what} must be a contiguous {dtype} {tuple(shape)}"
         + (f", got {t.dtype} {tuple(t.shape)}" if isinstance(t, torch.Tensor) else ""))


def out_or_new(out: Optional[torch.Tensor], shape, dtype, device, what: str = "out") -> torch.Tensor:
    if out is None:
        return torch.empty(shape, dtype=dtype, device=device)
    rows2d(out, what, (dtype,), *shape)
    return out


@contextlib.contextmanager
def _on(dev):
    with torch.cuda.device(dev):
        yield torch.cuda.current_stream(dev).cuda_stream


class _Here:
    """The current device's stream, without switching (the usual case)."""
    __slots__ = ("st",)

    def __init__(self, st):
        self.st = st

    def __enter__(self):
        return self.st

    def __exit__(self, *exc):
        return False


def launch(what: str, *tensors):
    """Context with the stream to launch on; refuses operands that are not on one GPU."""
    dev = tensors[0].device
    for t in tensors:
        if t is not None and t.device != dev:
            raise ValueError(f"{what}: operands on {dev} and {t.device}")
    if dev.type != "cuda":
        raise ValueError(f"{what} runs on the GPU: operands are on {dev}")
    if dev.index == torch.cuda.current_device():
        return _Here(torch.cuda.current_stream().cuda_stream)
    return _on(dev)
