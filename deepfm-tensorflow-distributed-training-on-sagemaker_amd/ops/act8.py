"""Activations kept in 8 bits for the backward pass (csrc/kernels/act8.hip).

``pack`` turns [M, N] activations into OCP e4m3 codes and one power-of-two scale per row and 32
columns: 1.03 bytes a value instead of 2 or 4.  A block's scale is the smallest 2^e (e in [-110,
120]) that keeps its largest finite magnitude within 448; a code is the e4m3 value nearest to
x / 2^e (ties to even).  Two rules serve the backward pass: a value that is not zero never becomes
a zero (it takes the smallest code of its sign instead), so a relu or dropout mask read from the
codes is the mask of the finite activations themselves; and infinities and NaN become NaN, in their own
place only (a mask is zero there).  A finite value stays finite: the code of 256 at the scale 2^120, of magnitudes from 248 *
2^120 on, stands for 240 * 2^120, because 2^128 is past fp32 and bf16.

The codes go into the gradient products as they are: ``experts.group_wgrad`` takes an ``Act8`` for
its input, ``experts.group_dgrad`` for its mask.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional

import torch

from . import _lib
from ._lib import Act8Args, check, ptr
from .checks import call, flat, out_or_new, rows2d

BLOCK = 32            # columns per scale


class Act8(NamedTuple):
    """8-bit activations: ``codes`` uint8 [M, N] (e4m3; rows may be strided), ``scales`` uint8
    [M, ceil(N / 32)], a scale's exponent + 127."""
    codes: torch.Tensor
    scales: torch.Tensor


def scale_cols(N: int) -> int:
    return -(-N // BLOCK)


def empty(M: int, N: int, device) -> Act8:
    """Uninitialised storage for [M, N] activations."""
    return Act8(torch.empty(M, N, dtype=torch.uint8, device=device),
                torch.empty(M, scale_cols(N), dtype=torch.uint8, device=device))


_U8 = (torch.uint8,)


def check_act8(a: Act8, M: int, N: int, what: str) -> int:
    """``a`` is an [M, N] Act8.  The row stride of its codes."""
    if not isinstance(a, Act8):
        raise ValueError(f"{what} must be an Act8")
    ld = rows2d(a.codes, what + ".codes", _U8, M, N)
    flat(a.scales, what + ".scales", torch.uint8, (M, scale_cols(N)))
    return ld


def check_own_act8(a: Act8, what: str) -> int:
    """``a`` is an Act8 whose parts fit one another.  The row stride of its codes."""
    if not isinstance(a, Act8):
        raise ValueError(f"{what} must be an Act8")
    ld = rows2d(a.codes, what + ".codes", _U8)
    flat(a.scales, what + ".scales", torch.uint8, (a.codes.shape[0], scale_cols(a.codes.shape[1])))
    return ld


_VALUES = (torch.float32, torch.bfloat16)


def pack(x: torch.Tensor, out: Optional[Act8] = None) -> Act8:
    """x [M, N] (fp32 or bf16, rows may be strided) -> ``Act8``."""
    ld = rows2d(x, "x", _VALUES)
    M, N = x.shape
    if out is None:
        out, ldc = empty(M, N, x.device), N
    else:
        ldc = check_act8(out, M, N, "out")
    a = Act8Args(ptr(x), ptr(out.codes), ptr(out.scales), 0, ld, ldc, M, N,
                 1 if x.dtype == torch.bfloat16 else 0)
    check(call("act8.pack", (x, *out), _lib.get_lib().hfm_act8_pack, C.byref(a)), "act8_pack")
    return out


def unpack(a: Act8, dtype: torch.dtype = torch.bfloat16, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The values that ``a`` stands for, in fp32 or bf16 (exact in both: four significant bits, and magnitudes from
    2^-119 to 240 * 2^120)."""
    ldc = check_own_act8(a, "a")
    M, N = a.codes.shape
    if dtype not in _VALUES:
        raise ValueError(f"unpack to fp32 or bf16, not {dtype}")
    out, ld = out_or_new(out, M, N, dtype, a.codes.device)
    args = Act8Args(0, ptr(a.codes), ptr(a.scales), ptr(out), ld, ldc, M, N,
                    1 if dtype == torch.bfloat16 else 0)
    check(call("act8.unpack", (*a, out), _lib.get_lib().hfm_act8_unpack, C.byref(args)), "act8_unpack")
    return out
