"""Refusals of the expert and 8-bit operators: the same with and without a GPU, before anything is
launched."""
import ctypes as C

import pytest
import torch

from hipfm.ops import _lib
from hipfm.ops import act8 as A8
from hipfm.ops import experts as EX

BF, F32, I32, U8 = torch.bfloat16, torch.float32, torch.int32, torch.uint8


def z(*s, dtype=BF):
    return torch.zeros(*s, dtype=dtype)


def routes(T=4, k=2, E=3, **kw):
    d = dict(expert=z(T, k, dtype=I32), weight=z(T, k, dtype=F32), pos=z(T, k, dtype=I32), src=z(T * k, dtype=I32),
             offs=z(E + 1, dtype=I32))
    d.update(kw)
    return EX.Routes(**d)


OFFS = z(4, dtype=I32)
W = z(3, 16, 8)
ACT = A8.Act8(z(6, 8, dtype=U8), z(6, 1, dtype=U8))

CALLS = {
    "gate type": lambda: EX.route(z(4, 3, dtype=torch.float16), 1),
    "gate shape": lambda: EX.route(z(4, 3, 2, dtype=F32), 1),
    "gate experts": lambda: EX.route(z(2, 1025, dtype=F32), 1),
    "gate no experts": lambda: EX.route(z(2, 0, dtype=F32), 1),
    "gate columns": lambda: EX.route(z(3, 4, dtype=F32).t(), 1),
    "gate rows": lambda: EX.route(z(1, 4, dtype=F32).expand(3, 4), 1),
    "top_k 0": lambda: EX.route(z(4, 3, dtype=F32), 0),
    "top_k over E": lambda: EX.route(z(4, 3, dtype=F32), 4),
    "top_k over 16": lambda: EX.route(z(4, 30, dtype=F32), 17),
    "valid type": lambda: EX.route(z(4, 3, dtype=F32), 1, valid=z(4, dtype=U8)),
    "valid rows": lambda: EX.route(z(4, 3, dtype=F32), 1, valid=z(5, dtype=torch.bool)),
    "route out": lambda: EX.route(z(4, 3, dtype=F32), 1, out=routes()),
    "route out offs": lambda: EX.route(z(4, 5, dtype=F32), 2, out=routes()),
    "bwd rows": lambda: EX.route_bwd(z(5, 3, dtype=F32), routes(), z(4, 2, dtype=F32)),
    "bwd dweight": lambda: EX.route_bwd(z(4, 3, dtype=F32), routes(), z(4, 2)),
    "bwd out": lambda: EX.route_bwd(z(4, 3, dtype=F32), routes(), z(4, 2, dtype=F32), out=z(4, 3)),
    "dispatch type": lambda: EX.dispatch(z(4, 8, dtype=torch.float64), routes()),
    "dispatch rows": lambda: EX.dispatch(z(5, 8), routes()),
    "dispatch out": lambda: EX.dispatch(z(4, 8), routes(), out=z(7, 8)),
    "dispatch pos": lambda: EX.dispatch(z(4, 8), routes(pos=z(4, 2, dtype=torch.int64))),
    "routes not Routes": lambda: EX.dispatch(z(4, 8), tuple(routes())),
    "combine rows": lambda: EX.combine(z(7, 8), routes()),
    "combine weight": lambda: EX.combine(z(8, 8), routes(weight=z(4, 2))),
    "dispatch_bwd rows": lambda: EX.dispatch_bwd(z(7, 8), routes()),
    "combine_bwd types": lambda: EX.combine_bwd(z(4, 8), z(8, 8, dtype=F32), routes()),
    "combine_bwd width": lambda: EX.combine_bwd(z(4, 8), z(8, 9), routes()),
    "linear x type": lambda: EX.group_linear(z(6, 8, dtype=F32), W, None, OFFS),
    "linear w shape": lambda: EX.group_linear(z(6, 9), W, None, OFFS),
    "linear w 2-D": lambda: EX.group_linear(z(6, 8), W[0], None, OFFS),
    "linear offs": lambda: EX.group_linear(z(6, 8), W, None, z(3, dtype=I32)),
    "linear offs type": lambda: EX.group_linear(z(6, 8), W, None, z(4, dtype=torch.int64)),
    "linear bias": lambda: EX.group_linear(z(6, 8), W, z(3, 16), OFFS),
    "linear out rows": lambda: EX.group_linear(z(6, 8), W, None, OFFS, out=z(5, 16)),
    "linear out type": lambda: EX.group_linear(z(6, 8), W, None, OFFS, out_dtype=torch.float16),
    "linear top_k": lambda: EX.group_linear(z(6, 8), W, None, OFFS, top_k=2),
    "linear src": lambda: EX.group_linear(z(6, 8), W, None, OFFS, src=z(6, dtype=torch.int64)),
    "linear src top_k": lambda: EX.group_linear(z(6, 8), W, None, OFFS, src=z(6, dtype=I32), top_k=0),
    "linear w axis": lambda: EX.group_linear(z(6, 16), W.transpose(1, 2), None, OFFS),
    "dgrad wt": lambda: EX.group_dgrad(z(6, 16), W, OFFS),
    "dgrad mask": lambda: EX.group_dgrad(z(6, 8), W, OFFS, mask=z(6, 8)),
    "dgrad mask type": lambda: EX.group_dgrad(z(6, 8), W, OFFS, mask=z(6, 16, dtype=F32)),
    "dgrad mask act8": lambda: EX.group_dgrad(z(6, 8), W, OFFS, mask=ACT),
    "wgrad rows": lambda: EX.group_wgrad(z(6, 16), z(7, 8), OFFS),
    "wgrad offs": lambda: EX.group_wgrad(z(6, 16), z(6, 8), z(1, dtype=I32)),
    "wgrad scales": lambda: EX.group_wgrad(z(6, 16), A8.Act8(z(6, 40, dtype=U8), z(6, 1, dtype=U8)), OFFS),
    "wgrad out": lambda: EX.group_wgrad(z(6, 16), z(6, 8), OFFS, out=(z(3, 16, 8), None)),
    "wgrad src": lambda: EX.group_wgrad(z(6, 16), z(9, 8), OFFS, src=z(5, dtype=I32), top_k=2),
    "pack type": lambda: A8.pack(z(3, 3, dtype=torch.float16)),
    "pack 1-D": lambda: A8.pack(z(3)),
    "pack out": lambda: A8.pack(z(3, 33), out=A8.Act8(z(3, 33, dtype=U8), z(3, 1, dtype=U8))),
    "pack out type": lambda: A8.pack(z(3, 3), out=A8.Act8(z(3, 3, dtype=torch.int8), z(3, 1, dtype=U8))),
    "unpack type": lambda: A8.unpack(ACT, torch.float16),
    "unpack not Act8": lambda: A8.unpack(z(3, 3)),
    "unpack out": lambda: A8.unpack(ACT, BF, out=z(6, 9)),
}


@pytest.mark.parametrize("name", sorted(CALLS))
def test_refused(name):
    with pytest.raises(ValueError) as e:
        CALLS[name]()
    assert "runs on the GPU" not in str(e.value), "refused for its device only"


GOOD = {
    "route": lambda: EX.route(z(4, 3, dtype=F32), 2),
    "route_bwd": lambda: EX.route_bwd(z(4, 3, dtype=F32), routes(), z(4, 2, dtype=F32)),
    "dispatch": lambda: EX.dispatch(z(4, 8), routes()),
    "dispatch_bwd": lambda: EX.dispatch_bwd(z(8, 8), routes()),
    "combine": lambda: EX.combine(z(8, 8), routes()),
    "combine_bwd": lambda: EX.combine_bwd(z(4, 8), z(8, 8), routes()),
    "group_linear": lambda: EX.group_linear(z(6, 8), W, z(3, 16, dtype=F32), OFFS),
    "group_dgrad": lambda: EX.group_dgrad(z(6, 8), W, OFFS, mask=z(6, 16)),
    "group_wgrad": lambda: EX.group_wgrad(z(6, 16), ACT, OFFS),
    "act8.pack": lambda: A8.pack(z(6, 8)),
    "act8.unpack": lambda: A8.unpack(ACT),
}


@pytest.mark.parametrize("name", sorted(GOOD))
def test_host_tensors_refused(name):
    with pytest.raises(ValueError, match=f"{name} runs on the GPU"):
        GOOD[name]()


def meta(*s, dtype=BF):
    return torch.empty(*s, dtype=dtype, device="meta")


PAST = 2 ** 32 + 4             # (4 in 32 bits)
WIDE = {
    "linear slots": lambda: EX.group_linear(meta(4, 8), meta(1, 8, 8), None, meta(2, dtype=I32), src=meta(PAST, dtype=I32)),
    "linear columns": lambda: EX.group_linear(meta(4, 8), meta(1, 1, 8).expand(1, PAST, 8), None, meta(2, dtype=I32)),
    "linear experts": lambda: EX.group_linear(meta(4, 8), meta(1, 8, 8).expand(PAST, 8, 8), None, meta(PAST + 1, dtype=I32)),
    "linear rows of the last tile": lambda: EX.group_linear(meta(2 ** 31 - 1, 1), meta(1, 8, 1), None, meta(2, dtype=I32)),
    "linear top_k": lambda: EX.group_linear(meta(4, 8), meta(1, 8, 8), None, meta(2, dtype=I32), src=meta(5, dtype=I32), top_k=PAST),
    "dgrad rows of the last tile": lambda: EX.group_dgrad(meta(2 ** 31 - 1, 1), meta(1, 8, 1), meta(2, dtype=I32)),
    "dgrad columns": lambda: EX.group_dgrad(meta(4, 8), meta(1, 1, 8).expand(1, PAST, 8), meta(2, dtype=I32)),
    "wgrad experts": lambda: EX.group_wgrad(meta(4, 8), meta(4, 8), meta(PAST + 1, dtype=I32)),
    "wgrad rows of the last tile": lambda: EX.group_wgrad(meta(2 ** 31 - 1, 1), meta(2 ** 31 - 1, 1), meta(2, dtype=I32)),
    "wgrad top_k": lambda: EX.group_wgrad(meta(4, 8), meta(4, 8), meta(2, dtype=I32), src=meta(4, dtype=I32), top_k=PAST),
}


@pytest.mark.parametrize("name", sorted(WIDE))
def test_sizes_past_32_bits_refused(name):
    with pytest.raises(ValueError) as e:
        WIDE[name]()
    assert "runs on the GPU" not in str(e.value), "its size would reach the kernel in 32 bits"


def nt_args(**kw):
    d = dict(lda=kw["K"], ldb=kw["K"], es=0, ldo=kw["N"], rows=kw["S"], top_k=1, scale=1.0)
    return _lib.GroupNtArgs(**{**d, **kw})


def test_lines_of_rows_are_counted_in_32_bits():
    """Where offsets that are not in order could make the count of all groups' rows overflow, the kernels that count them
    are not taken (seen by their workspace: copies of the odd rows, slabs for the bias)."""
    lib = _lib.get_lib()
    for E, large in ((1, True), (1024, True), (1 << 14, False), (1 << 16, False), (1 << 17, False)):
        a = nt_args(S=1 << 24, E=E, K=1024, N=256, lda=1025)
        assert (lib.hfm_group_nt_ws_bytes(C.byref(a)) > 0) == large, E
    for E, S, large in ((1, 1 << 24, True), (1024, 1 << 24, True), (65535, 1 << 22, False), (65535, 1 << 21, True)):
        b = _lib.GroupWgArgs(S=S, rows=S, E=E, K=8, N=8, ldz=8, ldx=8, top_k=1, ns=1, db=16)
        assert (lib.hfm_group_wgrad_ws_floats(C.byref(b)) > 0) == large, E


def test_launches_past_the_grid_refused():
    """Before anything is launched (1: an invalid value; a launch without a GPU gives another error)."""
    lib = _lib.get_lib()
    a = nt_args(S=1 << 25, E=1 << 25, K=4, N=128)
    b = _lib.GroupWgArgs(S=8, rows=8, E=1 << 25, K=1, N=1, ldz=1, ldx=1, top_k=1, ns=1)
    assert lib.hfm_group_nt(C.byref(a), None) == 1 and lib.hfm_group_wgrad(C.byref(b), None) == 1
