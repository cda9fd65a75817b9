"""Mixture-of-experts operators (csrc/kernels/experts.hip, group.hip): routing, the exchange of rows
between token order and expert order, and the experts' products, each with its gradient.

One training step of a layer of E experts, of which every token takes ``top_k``::

    r  = route(logits, top_k)                       # choices, weights, expert order
    h  = group_linear(x, w1, b1, r.offs, relu=True, src=r.src, top_k=top_k)
    ys = group_linear(h, w2, b2, r.offs)
    y  = combine(ys, r)
    ...
    dys, dweight = combine_bwd(dy, ys, r)
    dw2, db2 = group_wgrad(dys, h, r.offs)
    dh  = group_dgrad(dys, w2t, r.offs, mask=h)
    dw1, db1 = group_wgrad(dh, x, r.offs, src=r.src, top_k=top_k)
    dx  = dispatch_bwd(group_dgrad(dh, w1t, r.offs), r)
    dlogits = route_bwd(logits, r, dweight)

``x`` goes into the first product through ``src`` (no copy in expert order); ``dispatch`` makes that
copy where one is wanted.  ``h`` (or ``x``) can be kept in 8 bits between the passes: ``act8.pack``
after the forward, and the ``Act8`` in place of ``h`` in ``group_wgrad`` and ``group_dgrad``.

Expert order.  Slot s = t * top_k + j is choice j of token t.  ``src`` lists the live slots by expert,
in slot order within an expert; ``offs[e]`` is the first place of expert e and ``offs[E]`` the number
of live slots; ``pos`` is the place of each slot.  Group sizes stay on the GPU: a call takes ``S``
rows at most and no result depends on rows from ``offs[E]`` on, which keep what they held (a result
that the call allocated holds nothing there).

Results are allocated by the call unless ``out`` is given; workspaces come from torch's allocator on
the current stream, so calls on several streams and in several graphs share nothing.

``out`` shares no memory with the operands, but ``combine_bwd`` may write over ``ys`` and ``group_dgrad`` over a
bf16 ``mask``.

Any widths and strides are taken, sizes up to 2^31 - 1024.  Large products are fastest where rows start on 16 bytes and widths are
multiples of 8 (16 for 8-bit ``x``): operands that are otherwise are copied in the call.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional, Tuple, Union

import torch

from . import _lib
from ._lib import ExchArgs, GroupNtArgs, GroupWgArgs, RouteArgs, RouteBwdArgs, check, ptr
from .act8 import Act8, check_act8, check_own_act8
from .checks import call, flat, out_or_new, rows2d

MAX_EXPERTS = 1024
MAX_TOP_K = 16
_MAX_SLOTS = 1 << 30
_MAX_SIZE = (1 << 31) - 1024          # grouped products: int32 that counts on to the next whole tiles
_VALUES = (torch.float32, torch.bfloat16)
_BF = (torch.bfloat16,)
_EX_DISPATCH, _EX_DISPATCH_BWD, _EX_COMBINE, _EX_COMBINE_BWD = 0, 1, 2, 3


class Routes(NamedTuple):
    """Choices and expert order of T tokens (see the module's text): ``expert`` int32 [T, top_k]
    (-1: none), ``weight`` fp32 [T, top_k], ``pos`` int32 [T, top_k] (-1: none), ``src`` int32
    [T * top_k] (-1 behind the last live slot), ``offs`` int32 [E + 1]."""
    expert: torch.Tensor
    weight: torch.Tensor
    pos: torch.Tensor
    src: torch.Tensor
    offs: torch.Tensor


def _bf(t) -> int:
    return 1 if t.dtype == torch.bfloat16 else 0


def _check_gate(logits, top_k):
    ld = rows2d(logits, "logits", _VALUES)
    T, E = logits.shape
    if not 1 <= E <= MAX_EXPERTS:
        raise ValueError(f"1 to {MAX_EXPERTS} experts, got {E}")
    if not (isinstance(top_k, int) and 1 <= top_k <= min(E, MAX_TOP_K)):
        raise ValueError(f"top_k must be 1 to {min(E, MAX_TOP_K)}, got {top_k}")
    if T * top_k > _MAX_SLOTS:
        raise ValueError(f"{T} x {top_k} slots are more than {_MAX_SLOTS}")
    return T, E, ld


def _check_routes(r: Routes, T: Optional[int] = None) -> Tuple[int, int]:
    if not isinstance(r, Routes):
        raise ValueError("routes must be a Routes")
    expert, weight, pos, src, _ = r
    if expert.dim() != 2 or not 1 <= expert.shape[1] <= MAX_TOP_K:
        raise ValueError(f"routes.expert must be [T, 1 to {MAX_TOP_K}]")
    n, k = shape = expert.shape
    if T is not None and n != T:
        raise ValueError(f"routes are of {n} tokens, the rows of {T}")
    if n * k > _MAX_SLOTS:
        raise ValueError(f"{n} x {k} slots are more than {_MAX_SLOTS}")
    flat(expert, "routes.expert", torch.int32, shape)
    flat(weight, "routes.weight", torch.float32, shape)
    flat(pos, "routes.pos", torch.int32, shape)
    flat(src, "routes.src", torch.int32, (n * k,))
    return n, k


def route(logits: torch.Tensor, top_k: int, renormalize: bool = True, valid: Optional[torch.Tensor] = None,
          out: Optional[Routes] = None) -> Routes:
    """The ``top_k`` experts of every row of ``logits`` [T, E] (fp32 or bf16), the largest first and the
    lowest index first among equals; weights are the softmax over the chosen (``renormalize``) or
    over all experts.  A logit of -inf or NaN closes its expert, +inf counts as the largest finite
    number; rows where ``valid`` (bool [T]) is False choose nothing."""
    T, E, ld = _check_gate(logits, top_k)
    if valid is not None:
        flat(valid, "valid", torch.bool, (T,))
    dev = logits.device
    if out is None:
        i32 = dict(dtype=torch.int32, device=dev)
        out = Routes(torch.empty(T, top_k, **i32), torch.empty(T, top_k, dtype=torch.float32, device=dev),
                     torch.empty(T, top_k, **i32), torch.empty(T * top_k, **i32), torch.empty(E + 1, **i32))
    else:
        if _check_routes(out, T)[1] != top_k:
            raise ValueError("out has another top_k")
        flat(out.offs, "out.offs", torch.int32, (E + 1,))
    lib = _lib.get_lib()
    n = lib.hfm_route_ws_ints(T, E)
    ws = torch.empty(n, dtype=torch.int32, device=dev) if n else None
    a = RouteArgs(ptr(logits), ptr(valid), *(ptr(t) for t in out), ptr(ws), 0, ld, T, E, top_k,
                  1 if renormalize else 0, _bf(logits), 0, 0)
    check(call("route", (logits, valid, *out), lib.hfm_route, C.byref(a)), "route")
    return out


def route_bwd(logits: torch.Tensor, routes: Routes, dweight: torch.Tensor, renormalize: bool = True,
              out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """dL/dlogits (the logits' type) from dL/dweight (fp32 [T, top_k]); ``logits``, ``routes`` and
    ``renormalize`` as in ``route``.  Closed experts, empty slots and rows that are not valid get zeros."""
    rows2d(logits, "logits", _VALUES)
    T, k = _check_routes(routes, logits.shape[0])
    _, E, ld = _check_gate(logits, k)
    flat(dweight, "dweight", torch.float32, (T, k))
    out, ldo = out_or_new(out, T, E, logits.dtype, logits.device)
    a = RouteBwdArgs(ptr(logits), ptr(routes.expert), ptr(routes.weight), ptr(dweight), ptr(out),
                     ld, ldo, T, E, k, 1 if renormalize else 0, _bf(logits))
    check(call("route_bwd", (logits, *routes, dweight, out), _lib.get_lib().hfm_route_bwd, C.byref(a)), "route_bwd")
    return out


def _exchange(mode, what, a, b, out, pos, weight, dweight, lda, ldb, ldo, T, k, D):
    args = ExchArgs(a.data_ptr(), ptr(b), out.data_ptr(), pos.data_ptr(), ptr(weight), ptr(dweight), lda, ldb, ldo, T, k, D,
                    T * k, _bf(a))
    check(call(what, (a, b, out, pos, weight, dweight), _lib.get_lib().hfm_exchange, mode, C.byref(args)), what)


def dispatch(x: torch.Tensor, routes: Routes, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x [T, D] (fp32 or bf16) -> its rows in expert order, [T * top_k, D]."""
    ld = rows2d(x, "x", _VALUES)
    T, D = x.shape
    _, k = _check_routes(routes, T)
    out, ldo = out_or_new(out, T * k, D, x.dtype, x.device)
    _exchange(_EX_DISPATCH, "dispatch", x, None, out, routes.pos, None, None, ld, 0, ldo, T, k, D)
    return out


def dispatch_bwd(dxs: torch.Tensor, routes: Routes, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Gradient of ``dispatch``: dx[t] = the sum of token t's rows of dxs (fp32 sum, in slot order)."""
    ld = rows2d(dxs, "dxs", _VALUES)
    T, k = _check_routes(routes)
    n, D = dxs.shape
    if n != T * k:
        raise ValueError(f"dxs must have {T * k} rows, got {n}")
    out, ldo = out_or_new(out, T, D, dxs.dtype, dxs.device)
    _exchange(_EX_DISPATCH_BWD, "dispatch_bwd", dxs, None, out, routes.pos, None, None, ld, 0, ldo, T, k, D)
    return out


def combine(ys: torch.Tensor, routes: Routes, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """ys [T * top_k, D] in expert order -> y[t] = sum_j weight[t, j] ys[pos[t, j]] (fp32 sum, in slot
    order); a token without live slots gets zeros."""
    ld = rows2d(ys, "ys", _VALUES)
    T, k = _check_routes(routes)
    n, D = ys.shape
    if n != T * k:
        raise ValueError(f"ys must have {T * k} rows, got {n}")
    out, ldo = out_or_new(out, T, D, ys.dtype, ys.device)
    _exchange(_EX_COMBINE, "combine", ys, None, out, routes.pos, routes.weight, None, ld, 0, ldo, T, k, D)
    return out


def combine_bwd(dy: torch.Tensor, ys: torch.Tensor, routes: Routes,
                out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Gradients of ``combine``: (dys [T * top_k, D], dweight fp32 [T, top_k]) from dy [T, D]."""
    ld = rows2d(dy, "dy", _VALUES)
    T, D = dy.shape
    _, k = _check_routes(routes, T)
    ldb = rows2d(ys, "ys", (dy.dtype,), T * k, D)
    out, ldo = out_or_new(out, T * k, D, dy.dtype, dy.device)
    dweight = torch.empty(T, k, dtype=torch.float32, device=dy.device)
    _exchange(_EX_COMBINE_BWD, "combine_bwd", dy, ys, out, routes.pos, routes.weight, dweight, ld, ldb, ldo, T, k, D)
    return out, dweight


# ------------------------------------------------------------------ grouped products
def _check_groups(offs, E):
    flat(offs, "offs", torch.int32, (E + 1,))


def _check_sizes(*sizes):
    if max(sizes) > _MAX_SIZE:
        raise ValueError(f"rows, widths and experts up to {_MAX_SIZE}, got {sizes}")


def _check_gather(src, top_k, S):
    if not (isinstance(top_k, int) and 1 <= top_k <= _MAX_SIZE):
        raise ValueError(f"top_k must be an int from 1 to {_MAX_SIZE}, got {top_k}")
    if src is not None:
        flat(src, "src", torch.int32, (S,))
    elif top_k != 1:
        raise ValueError("top_k without src")


def _check_weight(w, what, K):
    if not (isinstance(w, torch.Tensor) and w.dim() == 3 and w.dtype == torch.bfloat16):
        raise ValueError(f"{what} must be a 3-D bf16 tensor")
    e, n, k = w.shape
    if k != K or e < 1:
        raise ValueError(f"{what} must be [1 or more, any, {K}], got {tuple(w.shape)}")
    if w.numel() and ((k != 1 and w.stride(2) != 1) or w.stride(1) < 0 or w.stride(0) < 0):
        raise ValueError(f"{what}'s last axis must be adjacent, got strides {w.stride()}")


def _check_out_type(dtype):
    if dtype not in _VALUES:
        raise ValueError(f"out must be bf16 or fp32, not {dtype}")


_NEEDS_WS = -1


def _nt(what, a: GroupNtArgs, tensors):
    lib, r = _lib.get_lib(), C.byref(a)
    rc = call(what, tensors, lib.hfm_group_nt, r)
    if rc == _NEEDS_WS:                    # copies of operands of odd widths
        ws = torch.empty(lib.hfm_group_nt_ws_bytes(r), dtype=torch.uint8, device=tensors[0].device)
        a.ws = ptr(ws)
        rc = call(what, tensors, lib.hfm_group_nt, r)
    check(rc, what)


def group_linear(x: torch.Tensor, w: torch.Tensor, bias: Optional[torch.Tensor], offs: torch.Tensor,
                 relu: bool = False, src: Optional[torch.Tensor] = None, top_k: int = 1,
                 out: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """out[p] = [relu](x[row(p)] w[e(p)]^T + bias[e(p)]) for every place p below offs[E]; x bf16 [rows, K],
    w bf16 [E, N, K], bias fp32 [E, N] or None, out bf16 or fp32 [S, N].  row(p) = p, or with ``src`` (int32
    [S]) row(p) = src[p] // top_k, the token of the slot; an entry of ``src`` that is no slot of a row
    of x reads as a row of zeros.  Without ``src``, S is x's rows."""
    ld = rows2d(x, "x", _BF)
    _check_weight(w, "w", x.shape[1])
    E, N, K = w.shape
    _check_groups(offs, E)
    S = x.shape[0] if src is None else src.shape[0]
    _check_gather(src, top_k, S)
    _check_sizes(S, x.shape[0], E, N, K)
    if bias is not None:
        flat(bias, "bias", torch.float32, (E, N))
    if out is not None:
        out_dtype = out.dtype
    _check_out_type(out_dtype)
    out, ldo = out_or_new(out, S, N, out_dtype, x.device)
    a = GroupNtArgs(ptr(x), ptr(w), ptr(bias), 0, ptr(out), ptr(offs), ptr(src), ld, w.stride(1),
                    w.stride(0), 0, ldo, S, x.shape[0], K, N, E, top_k, 1 if relu else 0, 0,
                    0 if _bf(out) else 1, 1.0)
    _nt("group_linear", a, (x, w, bias, offs, src, out))
    return out


def group_dgrad(dz: torch.Tensor, wt: torch.Tensor, offs: torch.Tensor,
                mask: Union[None, torch.Tensor, Act8] = None, scale: float = 1.0,
                out: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """Gradient towards the layer's input in expert order: out[p] = scale * dz[p] w[e(p)], zero where
    ``mask`` [S, K] (the input itself, bf16 or ``Act8``: what its relu and dropout left) is not above
    zero.  dz bf16 [S, N]; ``wt`` bf16 [E, K, N] is the transposed copy of w."""
    ld = rows2d(dz, "dz", _BF)
    S = dz.shape[0]
    _check_weight(wt, "wt", dz.shape[1])
    E, K, N = wt.shape
    _check_groups(offs, E)
    _check_sizes(S, E, N, K)
    m, ldm, m8 = None, 0, 0
    if isinstance(mask, Act8):
        m, ldm, m8 = mask.codes, check_act8(mask, S, K, "mask"), 1
    elif mask is not None:
        m, ldm = mask, rows2d(mask, "mask", _BF, S, K)
    if out is not None:
        out_dtype = out.dtype
    _check_out_type(out_dtype)
    out, ldo = out_or_new(out, S, K, out_dtype, dz.device)
    a = GroupNtArgs(ptr(dz), ptr(wt), 0, ptr(m), ptr(out), ptr(offs), 0, ld, wt.stride(1), wt.stride(0),
                    ldm, ldo, S, S, N, K, E, 1, 0, m8, 0 if _bf(out) else 1, float(scale))
    _nt("group_dgrad", a, (dz, wt, offs, m, out))
    return out


def group_wgrad(dz: torch.Tensor, x: Union[torch.Tensor, Act8], offs: torch.Tensor,
                src: Optional[torch.Tensor] = None, top_k: int = 1, bias: bool = True,
                out: Optional[Tuple[torch.Tensor, Optional[torch.Tensor]]] = None
                ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Gradients of w and bias, fp32: dw[e] = sum over the rows p of expert e of dz[p]^T x[row(p)]
    ([E, N, K]) and db[e] = sum dz[p] ([E, N], None without ``bias``); an expert without rows gets zeros.
    dz bf16 [S, N]; x bf16 [rows, K] or ``Act8``; ``src`` and ``top_k`` as in ``group_linear``.
    ``out``: the pair to write into, contiguous."""
    ld = rows2d(dz, "dz", _BF)
    S, N = dz.shape
    x8 = isinstance(x, Act8)
    if x8:
        ldx = check_own_act8(x, "x")
    else:
        ldx = rows2d(x, "x", _BF)
    xv = x.codes if x8 else x
    K = xv.shape[1]
    if not (isinstance(offs, torch.Tensor) and offs.dim() == 1 and offs.shape[0] >= 2):
        raise ValueError("offs must be int32 [E + 1]")
    E = offs.shape[0] - 1
    _check_groups(offs, E)
    _check_gather(src, top_k, S)
    _check_sizes(S, xv.shape[0], E, N, K)
    if src is None and xv.shape[0] != S:
        raise ValueError(f"x must have {S} rows, got {xv.shape[0]}")
    if out is None:
        dw = torch.empty(E, N, K, dtype=torch.float32, device=dz.device)
        db = torch.empty(E, N, dtype=torch.float32, device=dz.device) if bias else None
    else:
        dw, db = out
        flat(dw, "dw", torch.float32, (E, N, K))
        if db is not None:
            flat(db, "db", torch.float32, (E, N))
    lib = _lib.get_lib()
    a = GroupWgArgs(ptr(dz), ptr(xv), ptr(x.scales) if x8 else 0, ptr(offs), ptr(src), ptr(dw), ptr(db), 0,
                    ld, ldx, S, xv.shape[0], K, N, E, top_k, 1)
    r = C.byref(a)
    n = lib.hfm_group_wgrad_ws_floats(r)      # split products, column sums, copies of operands of odd widths
    ws = torch.empty(n, dtype=torch.float32, device=dz.device) if n else None
    a.ws = ptr(ws)
    check(call("group_wgrad", (dz, xv, x.scales if x8 else None, offs, src, dw, db), lib.hfm_group_wgrad, r), "group_wgrad")
    return dw, db
