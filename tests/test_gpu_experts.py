"""Expert routing, exchange, grouped products and 8-bit activations against 64-bit definitions.

Tolerances: a result rounded to a type is off by half a step, finfo.eps / 2 of the value; a sum of n
products accumulated in fp32 by n * 2^-23 of the sum of their magnitudes (each addition rounds by at
most 2^-23 of a partial sum that is at most that large, whatever the order)."""
import math

import pytest
import torch

import experts_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
NEG = float(torch.finfo(torch.float32).min)


def ops():
    from hipfm.ops import act8, experts
    return experts, act8


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g).to(dtype)


def close(got, want, bound, what=""):
    got = got.double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    bad = ~((got - want).abs() <= bound) & ~torch.isnan(want) & (got != want)
    assert not bad.any(), (what, int(bad.sum()), got[bad][:4], want[bad][:4])


# ------------------------------------------------------------------ route
def check_route(logits, k, renorm, valid=None):
    EX, _ = ops()
    r = EX.route(logits.to(DEV), k, renormalize=renorm, valid=None if valid is None else valid.to(DEV))
    expert, w, pos, src, offs = R.route(logits, k, renorm, valid)
    for name, a, b in (("expert", r.expert, expert), ("pos", r.pos, pos), ("src", r.src, src), ("offs", r.offs, offs)):
        assert torch.equal(a.cpu(), b), name
    # exp's argument is off by half a step of itself, exp and the division by a few, the sum by its terms
    l = logits.double().clamp(min=-1e4, max=1e4).nan_to_num(nan=0.0)
    span = (l.amax(1) - l.amin(1)).clamp(max=200)[:, None]
    close(r.weight, w, w * (span + logits.shape[1] + 8) * 2.0 ** -23, "weight")
    return r, w


@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 8, 2), (7, 3, 3), (48, 8, 2), (513, 64, 2), (1000, 65, 4), (3000, 5, 1),
                                   (2049, 256, 8), (300, 1000, 16), (20000, 16, 2), (70001, 4, 4)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_route(T, E, k, dtype):
    g = gen(T + E)
    lg = (randn(g, T, E) * 2).to(dtype)
    valid = torch.rand(T, generator=g) > 0.2
    check_route(lg, k, True)
    check_route(lg, k, False, valid)


@pytest.mark.parametrize("renorm", [True, False])
def test_route_ties_closed_and_extreme(renorm):
    inf, nan = math.inf, math.nan
    rows = [[0.0] * 6, [-inf] * 6, [nan] * 6, [1.0, nan, 1.0, -inf, 1.0, 1.0], [-inf, -inf, 3.0, -inf, -inf, -inf],
            [inf, 1.0, inf, 0.0, -inf, nan], [NEG] * 6, [NEG, 0.0, NEG, NEG, 0.0, NEG], [-0.0, 0.0, -0.0, 0.0, -1.0, 2.0],
            [3e38, -3e38, 0.0, 1.0, 2.0, 3e38], [1e-40, 0.0, 2e-40, -1e-40, 0.0, 0.0]]
    lg = torch.tensor(rows)
    r, w = check_route(lg, 3, renorm)
    EX, _ = ops()
    d = EX.route_bwd(lg.to(DEV), r, torch.ones(len(rows), 3, device=DEV) * torch.tensor([1.0, 2.0, 3.0], device=DEV), renormalize=renorm)
    assert torch.isfinite(d).all() and (d.cpu()[(torch.isnan(lg)) | (lg == -inf)] == 0).all()


@pytest.mark.parametrize("T,E,k", [(40, 100, 5), (900, 128, 8), (30, 256, 16), (900, 300, 8), (4097, 512, 3), (700, 1024, 4)])
def test_route_equal_values(T, E, k):
    """Few different values, so that every choice has equals, in one lane's list and in many; whole rows closed."""
    g = gen(T + E)
    lg = torch.randint(-1, 2, (T, E), generator=g).float()
    lg[lg == 0] = -0.0
    lg[torch.rand(T, E, generator=g) < 0.3] = 0.0
    lg[torch.rand(T, E, generator=g) < 0.2] = -math.inf
    lg[::7] = -math.inf
    lg[1::7, : E - 2] = -math.inf
    check_route(lg, k, True)
    check_route(lg.bfloat16(), k, False, torch.rand(T, generator=g) > 0.1)


@pytest.mark.parametrize("E", [5, 37, 130, 515])
def test_route_gradient_rows_at_any_alignment(E):
    EX, _ = ops()
    g = gen(E)
    big = randn(g, 61, E + 9).to(DEV)
    dw = randn(g, 61, 3).to(DEV)
    for dt in (torch.float32, torch.bfloat16):
        lg, out = big.to(dt)[:, 3:3 + E], torch.full((61, E + 5), 7.0, dtype=dt, device=DEV)
        for renorm in (True, False):
            r = EX.route(lg, 3, renormalize=renorm)
            want = EX.route_bwd(lg.contiguous(), r, dw, renormalize=renorm)
            EX.route_bwd(lg, r, dw, renormalize=renorm, out=out[:, 1:1 + E])
            assert torch.equal(out[:, 1:1 + E], want) and (out[:, 0] == 7).all() and (out[:, 1 + E:] == 7).all()


def test_route_no_rows_and_strides():
    EX, _ = ops()
    r = EX.route(torch.empty(0, 5, device=DEV), 2)
    assert r.offs.tolist() == [0] * 6 and r.expert.shape == (0, 2)
    big = randn(gen(5), 90, 40).to(DEV)
    r1, r2 = EX.route(big[::3, 7:20], 2), EX.route(big[::3, 7:20].contiguous(), 2)
    assert all(torch.equal(a, b) for a, b in zip(r1, r2))


@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (33, 8, 2), (777, 100, 4), (64, 1024, 16)])
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_route_gradient(T, E, k, renorm, dtype):
    EX, _ = ops()
    g = gen(E)
    lg = randn(g, T, E).to(dtype)
    lg[torch.rand(T, E, generator=g) < 0.1] = -math.inf
    valid = torch.rand(T, generator=g) > 0.2
    dw = randn(g, T, k)
    r = EX.route(lg.to(DEV), k, renormalize=renorm, valid=valid.to(DEV))
    d = EX.route_bwd(lg.to(DEV), r, dw.to(DEV), renormalize=renorm)
    expert, w, *_ = R.route(lg, k, renorm, valid)
    on = expert >= 0

    def weights(l):                        # the chosen experts' weights of fp64 logits
        m = torch.where(torch.isfinite(l), l, -1e300)
        ll = m.gather(1, expert.clamp(min=0).long())
        base = m.detach().amax(1, keepdim=True)
        num = torch.where(on, torch.exp(torch.where(on, ll - base, 0.0)), 0.0)
        den = num.sum(1, keepdim=True) if renorm else torch.where(on[:, :1], torch.exp(m - base), 0.0).sum(1, keepdim=True)
        return torch.where(on, num / den.clamp(min=1e-300), 0.0)

    l64 = lg.double()
    fin = torch.where(torch.isfinite(l64), l64, -1e300).requires_grad_()
    (weights(fin) * dw.double()).sum().backward()
    want = torch.where(torch.isfinite(l64), fin.grad, 0.0)
    scale = (w * dw.double().abs()).sum(1, keepdim=True) + dw.abs().amax(1, keepdim=True).double()
    close(d, want, HALF[dtype] * want.abs() + (E + 40) * 2.0 ** -23 * scale, "dlogits")
    # along a direction, against differences of the definition
    u = randn(g, T, E).double()
    h = 1e-6
    num = ((weights(fin.detach() + h * u) - weights(fin.detach() - h * u)) / (2 * h) * dw.double()).sum()
    ana = (d.double().cpu() * u).sum()
    # (the fp64 difference: h^2 |w'''| <= 1e-12, rounding 1e-16 / h = 1e-10 a slot)
    slack = ((HALF[dtype] * want.abs() + (E + 40) * 2.0 ** -23 * scale) * u.abs()).sum() + 1e-8 * T * k * dw.abs().max()
    assert abs(float(num - ana)) <= float(slack)


# ------------------------------------------------------------------ exchange
def some_routes(g, T, E, k, dead=0.15):
    EX, _ = ops()
    expert = torch.rand(T, E, generator=g).argsort(1)[:, :k].int()
    expert = torch.where(torch.rand(T, k, generator=g) < dead, -1, expert)
    w = torch.where(expert < 0, 0.0, torch.rand(T, k, generator=g))
    pos, src, offs = R.order(expert, E)
    return EX.Routes(*(t.to(DEV) for t in (expert, w, pos, src, offs))), (expert, w.double(), pos, src, offs)


@pytest.mark.parametrize("T,D,E,k", [(1, 1, 1, 1), (1, 4096, 4, 2), (37, 8, 5, 1), (100, 313, 6, 3), (64, 1248, 8, 2),
                                     (501, 72, 32, 8), (20, 40, 16, 16), (9, 1000, 7, 5)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_exchange(T, D, E, k, dtype):
    EX, _ = ops()
    g = gen(T * D + k)
    r, (expert, w, pos, src, offs) = some_routes(g, T, E, k)
    live = int(offs[-1])
    x, ys, dy, dxs = randn(g, T, D, dtype=dtype), randn(g, T * k, D, dtype=dtype), randn(g, T, D, dtype=dtype), randn(g, T * k, D, dtype=dtype)
    for t in (ys, dxs):                        # rows behind the last live slot are never read
        t[live:] = math.nan
    tok = src[:live].long() // k
    out = torch.full((T * k, D), 7.0, dtype=dtype, device=DEV)
    xs = EX.dispatch(x.to(DEV), r, out=out)
    assert torch.equal(xs[:live].cpu(), x[tok]) and bool((xs[live:] == 7).all())
    on = pos >= 0
    rows = torch.where(on[:, :, None], ys.double()[pos.clamp(min=0).long()], 0.0)
    y = EX.combine(ys.to(DEV), r)
    want = (rows * w[:, :, None]).sum(1)
    close(y, want, HALF[dtype] * want.abs() + k * 2.0 ** -23 * (rows.abs() * w[:, :, None]).sum(1), "y")
    gr = torch.where(on[:, :, None], dxs.double()[pos.clamp(min=0).long()], 0.0)
    dx = EX.dispatch_bwd(dxs.to(DEV), r)
    close(dx, gr.sum(1), HALF[dtype] * gr.sum(1).abs() + k * 2.0 ** -23 * gr.abs().sum(1), "dx")
    out = torch.full((T * k, D), 7.0, dtype=dtype, device=DEV)
    dys, dweight = EX.combine_bwd(dy.to(DEV), ys.to(DEV), r, out=out)
    want = dy.double()[tok] * w.view(-1)[src[:live].long()][:, None]
    close(dys[:live], want, HALF[dtype] * want.abs() + 2.0 ** -24 * want.abs(), "dys")
    assert bool((dys[live:] == 7).all())
    dot = (rows * dy.double()[:, None, :]).sum(2)
    close(dweight, dot, (D + 8) * 2.0 ** -23 * (rows * dy.double()[:, None, :]).abs().sum(2), "dweight")


def test_exchange_strides_and_alignment():
    EX, _ = ops()
    g = gen(3)
    r, _ = some_routes(g, 50, 4, 2)
    for dt in (torch.float32, torch.bfloat16):
        for off, D, pad in ((0, 64, 8), (1, 64, 7), (3, 24, 5), (8, 24, 8)):
            xb, yb = randn(g, 50, off + D + pad, dtype=dt).to(DEV), randn(g, 100, off + D + pad, dtype=dt).to(DEV)
            x, ys = xb[:, off: off + D], yb[:, off: off + D]
            ob = torch.zeros_like(yb)
            xs = EX.dispatch(x, r, out=ob[:, off: off + D])
            live = int(r.offs[-1])
            assert torch.equal(xs[:live], EX.dispatch(x.contiguous(), r)[:live])
            assert not ob[:, :off].any() and not ob[:, off + D:].any()
            assert torch.equal(EX.combine(ys, r), EX.combine(ys.contiguous(), r))
            a, b = EX.combine_bwd(x, ys, r), EX.combine_bwd(x.contiguous(), ys.contiguous(), r)
            assert torch.equal(a[0][:live], b[0][:live])
            # (16-byte accesses sum the D products in another order: each within its bound)
            rows = torch.where(r.pos[:, :, None] >= 0, ys.double()[r.pos.clamp(min=0).long()], 0.0)
            mag = (rows * x.double()[:, None, :]).abs().sum(2).cpu()
            close(a[1], b[1].double().cpu(), 2 * (D + 8) * 2.0 ** -23 * mag, "dweight")


# ------------------------------------------------------------------ 8-bit activations
@pytest.mark.parametrize("M,N", [(1, 1), (3, 31), (5, 32), (17, 33), (64, 400), (33, 401), (7, 4096), (130, 1248)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_pack(M, N, dtype):
    _, A8 = ops()
    g = gen(M * N)
    x = (randn(g, M, N) * torch.exp(4 * randn(g, M, N))).to(dtype)
    x[torch.rand(M, N, generator=g) < 0.3] = 0
    codes, scales, vals = R.pack(x)
    a = A8.pack(x.to(DEV))
    assert torch.equal(a.scales.cpu(), scales) and torch.equal(a.codes.cpu(), codes)
    assert torch.equal((a.codes.cpu() & 127) == 0, x == 0)
    for dt in (torch.float32, torch.bfloat16):     # four significant bits: exact in both
        assert torch.equal(A8.unpack(a, dt).double().cpu(), vals)


def test_pack_extremes():
    _, A8 = ops()
    fmax, inf, nan = float(torch.finfo(torch.float32).max), math.inf, math.nan
    rows = [[0.0, -0.0, 1e-45, -1e-45], [fmax, -fmax, 1e-38, -1e-45], [inf, 1.0, -inf, nan], [nan, nan, -0.0, 0.0],
            [448.0, 447.9, 464.0, 1e-4], [449.0, 1.0, -2.0 ** -11, 2.0 ** -9], [2.0 ** -120, 2.0 ** -126, 3e-39, 0.0],
            [240.0, 248.0, 232.0, 17.0], [1.0, 1.0625, 1.1875, 1.3125]]
    x = torch.tensor(rows).repeat(1, 9)            # 36 columns: a whole block and a part of one
    x[:, 33] *= 0.0
    for dt in (torch.float32, torch.bfloat16):
        codes, scales, _ = R.pack(x.to(dt))
        a = A8.pack(x.to(dt).to(DEV))
        assert torch.equal(a.scales.cpu(), scales)
        got, want = a.codes.cpu(), codes
        same = (got == want) | ((got & 127 == 127) & (want & 127 == 127))      # (a NaN's sign says nothing)
        assert same.all(), (x[~same][:4], got[~same][:4], want[~same][:4])


def test_pack_strides_and_empty():
    _, A8 = ops()
    g = gen(2)
    for dt in (torch.float32, torch.bfloat16):
        for off, N, pad in ((0, 64, 16), (1, 64, 15), (8, 40, 16), (3, 33, 4)):
            b = randn(g, 40, off + N + pad, dtype=dt).to(DEV)
            x = b[::2, off: off + N]
            cb = torch.zeros(20, off + N + pad, dtype=torch.uint8, device=DEV)
            a = A8.pack(x, out=A8.Act8(cb[:, off: off + N], torch.zeros(20, A8.scale_cols(N), dtype=torch.uint8, device=DEV)))
            c = A8.pack(x.contiguous())
            assert torch.equal(a.codes, c.codes) and torch.equal(a.scales, c.scales)
            assert not cb[:, :off].any() and not cb[:, off + N:].any()
            assert torch.equal(A8.unpack(a, dt), A8.unpack(c, dt))
    for M, N in ((0, 5), (5, 0)):
        a = A8.pack(torch.empty(M, N, device=DEV))
        assert A8.unpack(a).shape == (M, N)


# ------------------------------------------------------------------ grouped products
def groups(sizes, tail=0):
    offs = torch.tensor([0] + sizes).cumsum(0).int()
    return offs, int(offs[-1]) + tail


SIZES = [[1], [5], [0, 3, 0], [64, 1, 0, 200], [127, 128, 129], [300], [0, 0], [1] * 70, [513, 0, 31, 256]]


def product_ref(x, w, e, rows):
    """(product, bound of its fp32 sum) of rows x[p] w[e(p)]^T in fp64, zeros where e is -1."""
    out = torch.zeros(rows, w.shape[1], dtype=torch.float64)
    mag = torch.zeros_like(out)
    for i in range(w.shape[0]):
        at = e == i
        out[at] = x[at].double() @ w[i].double().T
        mag[at] = x[at].double().abs() @ w[i].double().abs().T
    return out, (x.shape[1] + 4) * 2.0 ** -23 * mag


@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("K,N", [(1, 1), (64, 64), (40, 130), (320, 256), (33, 17), (128, 1)])
def test_group_linear(sizes, K, N):
    EX, _ = ops()
    E = len(sizes)
    g = gen(K * N + E)
    offs, S = groups(sizes, tail=3)
    e = R.group_ids(offs, S)
    x, w, b = randn(g, S, K, dtype=torch.bfloat16), randn(g, E, N, K, dtype=torch.bfloat16), randn(g, E, N)
    x[e < 0] = math.nan
    want, bound = product_ref(x, w, e, S)
    live = e >= 0
    want = want + torch.where(live[:, None], b.double()[e.clamp(min=0)], 0.0)
    bound = bound + 2.0 ** -23 * want.abs()
    for dt in (torch.bfloat16, torch.float32):
        out = torch.full((S, N), 7.0, dtype=dt, device=DEV)
        y = EX.group_linear(x.to(DEV), w.to(DEV), b.to(DEV), offs.to(DEV), out=out)
        close(y[live], want[live], (HALF[dt] * want.abs() + bound * 1.01)[live], "y")
        assert bool((y[~live] == 7).all())
    y = EX.group_linear(x.to(DEV), w.to(DEV), b.to(DEV), offs.to(DEV), relu=True)
    close(y[live], want[live].clamp(min=0), (HALF[torch.bfloat16] * want.abs() + bound * 1.01)[live], "relu")
    # through src: the same rows, shuffled, as choice j of their token
    perm = torch.randperm(S, generator=g)
    back = torch.empty_like(perm)
    back[perm] = torch.arange(S)
    src = (back * 3 + torch.randint(0, 3, (S,), generator=g)).int()
    z = EX.group_linear(x[perm].to(DEV), w.to(DEV), b.to(DEV), offs.to(DEV), relu=True, src=src.to(DEV), top_k=3)
    assert torch.equal(z[live], y[live])


@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("K,N", [(1, 1), (64, 64), (130, 40), (256, 320), (33, 17)])
@pytest.mark.parametrize("kind", ["none", "bf16", "act8"])
def test_group_dgrad(sizes, K, N, kind):
    EX, A8 = ops()
    E = len(sizes)
    g = gen(K * N + E)
    offs, S = groups(sizes, tail=2)
    e = R.group_ids(offs, S)
    live = e >= 0
    dz, w = randn(g, S, N, dtype=torch.bfloat16), randn(g, E, N, K, dtype=torch.bfloat16)
    dz[~live] = math.nan
    h = torch.relu(randn(g, S, K)).to(torch.bfloat16)
    if S > 1:
        h[0, 0], h[1, 0] = math.nan, 1e-30
    want, bound = product_ref(dz, w.transpose(1, 2), e, S)
    want, bound = want * 0.75, bound * 0.75 + 2.0 ** -23 * want.abs()
    if kind != "none":
        want = torch.where(h.double() > 0, want, 0.0)
    mask = {"none": None, "bf16": h.to(DEV), "act8": A8.pack(h.to(DEV))}[kind]
    for dt in (torch.bfloat16, torch.float32):
        out = torch.full((S, K), 7.0, dtype=dt, device=DEV)
        dx = EX.group_dgrad(dz.to(DEV), w.transpose(1, 2).contiguous().to(DEV), offs.to(DEV), mask=mask, scale=0.75, out=out)
        close(dx[live], want[live], (HALF[dt] * want.abs() + bound * 1.01)[live], "dx")
        assert bool((dx[~live] == 7).all())


@pytest.mark.parametrize("sizes", SIZES + [[3000], [2500, 700]])
@pytest.mark.parametrize("K,N", [(1, 1), (64, 64), (130, 40), (320, 256), (33, 17)])
@pytest.mark.parametrize("x8", [False, True])
def test_group_wgrad(sizes, K, N, x8):
    EX, A8 = ops()
    E = len(sizes)
    g = gen(K * N + E)
    offs, S = groups(sizes, tail=2)
    e = R.group_ids(offs, S)
    dz, x = randn(g, S, N, dtype=torch.bfloat16), randn(g, S, K, dtype=torch.bfloat16)
    dz[e < 0] = math.nan
    x[e < 0] = math.nan
    xv = x.double()
    xd = x.to(DEV)
    if x8:
        xv = R.pack(x)[2]
        xd = A8.pack(xd)
    dw, db = EX.group_wgrad(dz.to(DEV), xd, offs.to(DEV))
    perm = torch.randperm(S, generator=g)
    back = torch.empty_like(perm)
    back[perm] = torch.arange(S)
    src = (back * 2 + 1).int().to(DEV)
    xp = A8.Act8(xd.codes[perm.to(DEV)], xd.scales[perm.to(DEV)]) if x8 else xd[perm.to(DEV)]
    dw2, db2 = EX.group_wgrad(dz.to(DEV), xp, offs.to(DEV), src=src, top_k=2)
    assert torch.equal(dw, dw2) and torch.equal(db, db2)
    assert EX.group_wgrad(dz.to(DEV), xd, offs.to(DEV), bias=False)[1] is None
    for i in range(E):
        at = e == i
        n = int(at.sum())
        a, b = dz[at].double(), xv[at]
        close(dw[i], a.T @ b, (n + 4) * 2.0 ** -23 * (a.abs().T @ b.abs()), "dw")
        close(db[i], a.sum(0), (n + 4) * 2.0 ** -23 * a.abs().sum(0), "db")


LARGE = [([9000, 0, 257, 1, 5000, 256], 200, 1032), ([20000], 64, 777), ([3] * 150, 72, 40), ([700, 4000, 1300], 1248, 2048),
         ([1, 0, 30000], 136, 264), ([5000, 6000], 512, 1000), ([6000, 0, 7000], 517, 1003), ([3000, 2500, 1], 1032, 1000),
         ([9000], 1001, 390), ([9000, 0, 700], 40, 1000), ([9000, 700], 1000, 40), ([5000, 4000], 33, 1001),
         ([5000, 4000], 1001, 33), ([700, 300], 512, 512), ([1500, 0, 500], 1024, 328), ([2100], 8, 2048), ([2100], 2048, 16)]


@pytest.mark.parametrize("S,K,N", [(300, 40, 72), (9000, 320, 512)])
def test_results_over_operands_they_may_replace(S, K, N):
    """combine_bwd over ys, group_dgrad over its bf16 mask."""
    EX, _ = ops()
    g = torch.Generator(device=DEV).manual_seed(S)
    r = EX.route(torch.randn(S, 6, device=DEV, generator=g), 3)
    dy, ys = torch.randn(S, N, device=DEV, generator=g), torch.randn(3 * S, N, device=DEV, generator=g)
    dys, dw = EX.combine_bwd(dy, ys, r)
    dys2, dw2 = EX.combine_bwd(dy, ys, r, out=ys)
    assert dys2.data_ptr() == ys.data_ptr() and torch.equal(dys2, dys) and torch.equal(dw2, dw)
    offs = torch.tensor([0, S // 3, S], dtype=torch.int32, device=DEV)
    dz, wt = torch.randn(S, K, device=DEV, generator=g).bfloat16(), torch.randn(2, N, K, device=DEV, generator=g).bfloat16()
    mask = torch.randn(S, N, device=DEV, generator=g).bfloat16()
    dx = EX.group_dgrad(dz, wt, offs, mask=mask)
    assert torch.equal(EX.group_dgrad(dz, wt, offs, mask=mask, out=mask), dx)


def test_large_products_of_rows_at_any_alignment():
    """Operands, masks and results that start at odd places in wider rows give what aligned ones give.  The kernel
    may be another one, whose fp32 sums run in another order: each result is within (terms + 4) 2^-23 of the
    products' magnitudes of the exact one, and a bf16 result within half a step more."""
    EX, A8 = ops()
    g = torch.Generator(device=DEV).manual_seed(9)
    S, K, N, E = 9000, 320, 600, 3
    offs, _ = groups([4000, 0, 4900], tail=0)
    o, live = offs.int().to(DEV), int(offs[-1])

    def shifted(t):
        wide = torch.full((*t.shape[:-1], t.shape[-1] + 11), math.nan, dtype=t.dtype, device=DEV)
        wide[..., 3:3 + t.shape[-1]] = t
        return wide[..., 3:3 + t.shape[-1]]

    def same(a, b, terms, mag, scale=1.0):
        a, b = a.double(), b.double()
        half = HALF[torch.bfloat16] if terms < 2000 else 0.0
        return bool(((a - b).abs() <= 2 * (terms + 4) * 2.0 ** -23 * scale * mag + half * (a.abs() + b.abs())).all())

    def mags(p, q):                                 # rows of an expert times its weights
        return torch.cat([p[lo:hi].double().abs() @ q[e].double().abs().T for e, (lo, hi) in enumerate(zip(offs, offs[1:]))])

    x, w, dz = (torch.randn(*s, device=DEV, generator=g).bfloat16() for s in ((S, K), (E, N, K), (S, N)))
    wt = w.transpose(1, 2).contiguous()
    out = torch.full((S, N + 7), 5.0, dtype=torch.bfloat16, device=DEV)
    y = EX.group_linear(x, w, None, o)
    EX.group_linear(shifted(x), shifted(w), None, o, out=out[:, 3:3 + N])
    assert same(out[:live, 3:3 + N], y[:live], K, mags(x, w)) and bool((out[:, :3] == 5).all()) and bool((out[:, 3 + N:] == 5).all())
    assert bool((out[live:] == 5).all())
    mask = torch.randn(S, K, device=DEV, generator=g).bfloat16()
    dx = EX.group_dgrad(dz, wt, o, mask=mask, scale=2.0)
    dx2 = EX.group_dgrad(shifted(dz), shifted(wt), o, mask=shifted(mask), scale=2.0)
    assert same(dx2[:live], dx[:live], N, mags(dz, wt), 2.0) and torch.equal(dx2[:live] == 0, dx[:live] == 0)
    dw, db = EX.group_wgrad(dz, x, o)
    dw2, db2 = EX.group_wgrad(shifted(dz), shifted(x), o)
    for e, (lo, hi) in enumerate(zip(offs, offs[1:])):
        z, v = dz[lo:hi].double().abs(), x[lo:hi].double().abs()
        assert same(dw2[e], dw[e], 4900, z.T @ v) and same(db2[e], db[e], 4900, z.sum(0))
    src = torch.randperm(S, device=DEV, generator=g).int()
    ys, yg = EX.group_linear(shifted(x), w, None, o, src=src), EX.group_linear(x, w, None, o, src=src)
    assert same(ys[:live], yg[:live], K, mags(x[src.long()], w))
    a = A8.pack(x)
    # no row of x at all: every place reads zeros
    none = torch.full((S,), -1, dtype=torch.int32, device=DEV)
    assert bool((EX.group_linear(x[:0], w, None, o, src=none)[:live] == 0).all())
    for e in (x[:0], A8.Act8(a.codes[:0], a.scales[:0])):
        dw0, db0 = EX.group_wgrad(dz, e, o, src=none)
        assert bool((dw0 == 0).all()) and bool(((db0 - db).abs() <= 2 * (4900 + 4) * 2.0 ** -23 * dz.float().abs().sum(0)).all())


def test_odd_large_products_in_a_graph():
    """The copies of odd operands are made in the call, in every replay."""
    EX, A8 = ops()
    g = torch.Generator(device=DEV).manual_seed(11)
    S, K, N = 9000, 333, 601
    o = torch.tensor([0, 3000, 8990], dtype=torch.int32, device=DEV)
    x, w, dz = (torch.randn(*s, device=DEV, generator=g).bfloat16() for s in ((S, K), (2, N, K), (S, N)))
    wt = w.transpose(1, 2).contiguous()

    def run():
        return (EX.group_linear(x, w, None, o)[:8990], EX.group_dgrad(dz, wt, o, mask=x)[:8990], *EX.group_wgrad(dz, x, o))

    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run()
    for i in range(3):
        x.copy_(torch.randn(S, K, device=DEV, generator=g))
        dz.copy_(torch.randn(S, N, device=DEV, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, run())), i


@pytest.mark.parametrize("sizes", [[10], [300], [40, 700], [0, 130, 1], [64 * 9 + 1, 64 * 5], [1] * 6, [0, 0]])
@pytest.mark.parametrize("x8", [False, True])
def test_weight_gradient_of_few_rows_in_a_large_order(sizes, x8):
    """Room for many rows, few of them live: the split over rows is planned on the room."""
    EX, A8 = ops()
    g = torch.Generator(device=DEV).manual_seed(len(sizes))
    S, N, K = 16384, 512, 768
    offs = torch.tensor([0] + sizes).cumsum(0)
    dz = torch.randn(S, N, device=DEV, generator=g).bfloat16()
    x = torch.randn(S, K, device=DEV, generator=g).bfloat16()
    live = int(offs[-1])
    dz[live:], x[live:] = math.nan, math.nan
    a = A8.pack(x) if x8 else x
    xv = (A8.unpack(a, torch.float32) if x8 else x).double()
    nan = torch.full((1 << 28,), math.nan, device=DEV)         # what the workspace may hold
    del nan
    dw, db = EX.group_wgrad(dz, a, offs.int().to(DEV))
    for e in range(len(sizes)):
        lo, hi = int(offs[e]), int(offs[e + 1])
        z, v = dz[lo:hi].double(), xv[lo:hi]
        c = (hi - lo + 4) * 2.0 ** -23
        assert bool(((dw[e].double() - z.T @ v).abs() <= c * (z.abs().T @ v.abs())).all()), e
        assert bool(((db[e].double() - z.sum(0)).abs() <= c * z.abs().sum(0)).all()), e


@pytest.mark.parametrize("sizes,K,N", LARGE)
def test_group_products_many_tiles(sizes, K, N):
    """The same three products where the output has many tiles (the large-tile kernels)."""
    EX, A8 = ops()
    E = len(sizes)
    g = torch.Generator(device=DEV).manual_seed(K + N)
    offs, S = groups(sizes, tail=5)
    e = R.group_ids(offs, S)
    o = offs.to(DEV)

    def rn(*shape, dtype=torch.bfloat16):
        return torch.randn(*shape, device=DEV, generator=g).to(dtype)

    x, w, b, dz = rn(S, K), rn(E, N, K), rn(E, N, dtype=torch.float32), rn(S, N)
    x[S - 5:], dz[S - 5:] = math.nan, math.nan
    live = S - 5

    def spans():
        return [(i, int(offs[i]), int(offs[i + 1])) for i in range(E) if offs[i + 1] > offs[i]]

    def check(got, want, bound, what):
        d = (got.double() - want).abs()
        assert bool((d <= bound).all()), (what, float((d - bound).max()))

    half = HALF[torch.bfloat16]
    out = torch.full((S, N), 7.0, dtype=torch.bfloat16, device=DEV)
    y = EX.group_linear(x, w, b, o, relu=True, out=out)
    assert bool((y[live:] == 7).all())
    k3 = torch.randint(0, 3, (S,), device=DEV, generator=g)
    perm = torch.randperm(S, device=DEV, generator=g)
    src = (torch.argsort(perm) * 3 + k3).int()
    assert torch.equal(EX.group_linear(x[perm], w, b, o, relu=True, src=src, top_k=3)[:live], y[:live])
    gone = src.clone()
    gone[::7] = -1
    z = EX.group_linear(x[perm], w, b, o, src=gone, top_k=3, out_dtype=torch.float32)
    zero = torch.arange(S, device=DEV) % 7 == 0
    h = torch.relu(rn(S, K, dtype=torch.float32)).to(torch.bfloat16)
    a8 = A8.pack(h)
    wt = w.transpose(1, 2).contiguous()
    dx = EX.group_dgrad(dz, wt, o, mask=h, scale=0.5)
    assert torch.equal(dx[:live], EX.group_dgrad(dz, wt, o, mask=a8, scale=0.5)[:live])
    dw, db = EX.group_wgrad(dz, x, o)
    dwp, dbp = EX.group_wgrad(dz, x[perm], o, src=src, top_k=3)
    assert torch.equal(dw, dwp) and torch.equal(db, dbp)
    dw8, db8 = EX.group_wgrad(dz, a8, o)
    ap = A8.Act8(a8.codes[perm], a8.scales[perm])
    dw8p, db8p = EX.group_wgrad(dz, ap, o, src=src, top_k=3)
    assert torch.equal(dw8, dw8p) and torch.equal(db8, db8p)
    h8 = A8.unpack(a8, torch.float32).double()
    for i, lo, hi in spans():
        xd, wd, zd = x[lo:hi].double(), w[i].double(), dz[lo:hi].double()
        c = 2.0 ** -23 * 1.01
        p, mag = xd @ wd.T, xd.abs() @ wd.abs().T
        want = p + b[i].double()
        check(y[lo:hi], want.clamp(min=0), half * want.abs() + c * ((K + 4) * mag + want.abs()), "y")
        want = torch.where(zero[lo:hi, None], 0.0, p) + b[i].double()
        check(z[lo:hi], want, 2.0 ** -24 * want.abs() + c * ((K + 4) * mag + want.abs()), "z")
        want = 0.5 * (zd @ wd) * (h[lo:hi] > 0)
        check(dx[lo:hi], want, half * want.abs() + c * ((N + 4) * 0.5 * (zd.abs() @ wd.abs()) + want.abs()), "dx")
        check(dw[i], zd.T @ xd, c * (hi - lo + 4) * (zd.abs().T @ xd.abs()), "dw")
        check(dw8[i], zd.T @ h8[lo:hi], c * (hi - lo + 4) * (zd.abs().T @ h8[lo:hi]), "dw8")
        for d in (db, db8):                    # (of two kernels where the width suits one of the types only)
            check(d[i], zd.sum(0), c * (hi - lo + 4) * zd.abs().sum(0), "db")
    for i in range(E):
        if sizes[i] == 0:
            assert not dw[i].any() and not db[i].any() and not dw8[i].any()


def test_group_bad_device_data_stays_in_bounds():
    """Offsets that are not in order and sources that are no slots: rows read as documented, no more."""
    EX, _ = ops()
    g = gen(1)
    x, w = randn(g, 100, 64, dtype=torch.bfloat16).to(DEV), randn(g, 3, 64, 64, dtype=torch.bfloat16).to(DEV)
    for o in ([0, 50, 20, 100], [-5, 10, 400, 100], [90, 80, 70, 60], [2 ** 30, 0, -2 ** 31, 2 ** 31 - 1]):
        offs = torch.tensor(o, dtype=torch.int32, device=DEV)
        out = torch.zeros(100, 64, dtype=torch.bfloat16, device=DEV)
        EX.group_linear(x, w, None, offs, out=out)
        dw, _ = EX.group_wgrad(x, x, offs)
        assert torch.isfinite(out).all() and torch.isfinite(dw).all()
    offs = torch.tensor([0, 3, 6, 6], dtype=torch.int32, device=DEV)
    src = torch.tensor([0, -1, 199, 200, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device=DEV)
    y = EX.group_linear(x, w, None, offs, src=src, top_k=2)
    ok = EX.group_linear(torch.stack([x[0], x[0] * 0, x[99], x[0] * 0, x[0] * 0, x[0] * 0]), w, None, offs)
    assert torch.equal(y, ok)


def test_group_strides():
    EX, A8 = ops()
    g = gen(8)
    offs, S = groups([70, 0, 61])
    for off, K, N, pad in ((0, 64, 128, 8), (1, 64, 64, 3), (8, 72, 40, 16), (3, 33, 50, 2)):
        xb = randn(g, S, off + K + pad, dtype=torch.bfloat16).to(DEV)
        wb = randn(g, 3, N + 2, off + K + pad, dtype=torch.bfloat16).to(DEV)
        x, w = xb[:, off: off + K], wb[:, 1: N + 1, off: off + K]
        o = offs.to(DEV)
        assert torch.equal(EX.group_linear(x, w, None, o), EX.group_linear(x.contiguous(), w.contiguous(), None, o))
        ob = torch.zeros(S, off + N + pad, dtype=torch.bfloat16, device=DEV)
        y = EX.group_linear(x, w, None, o, out=ob[:, off: off + N])
        assert torch.equal(y, EX.group_linear(x, w, None, o)) and not ob[:, :off].any() and not ob[:, off + N:].any()
        a, b = EX.group_wgrad(y, x, o), EX.group_wgrad(y.contiguous(), x.contiguous(), o)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        m = A8.pack(x)
        mb = torch.zeros(S, off + K + pad, dtype=torch.uint8, device=DEV)
        mb[:, off: off + K] = m.codes
        wt = w.transpose(1, 2).contiguous()
        mv = A8.Act8(mb[:, off: off + K], m.scales)
        assert torch.equal(EX.group_dgrad(y, wt, o, mask=mv), EX.group_dgrad(y.contiguous(), wt, o, mask=m))
        assert torch.equal(EX.group_wgrad(y, mv, o)[0], EX.group_wgrad(y, m, o)[0])
    shared = randn(g, 1, 64, 64, dtype=torch.bfloat16).to(DEV)      # one matrix for every expert
    x = randn(g, S, 64, dtype=torch.bfloat16).to(DEV)
    assert torch.equal(EX.group_linear(x, shared.expand(3, 64, 64), None, offs.to(DEV)),
                       EX.group_linear(x, shared.expand(3, 64, 64).contiguous(), None, offs.to(DEV)))


def test_far_rows():
    """Rows whose elements lie past 2^31 (row strides of 2^30 elements)."""
    EX, A8 = ops()
    g = gen(4)
    n, ld, D = 4, 1 << 30, 64
    big = torch.empty(n * ld, dtype=torch.bfloat16, device=DEV)
    x = big.view(n, ld)[:, :D]
    x.copy_(randn(g, n, D, dtype=torch.bfloat16))
    xc = x.contiguous()
    w = randn(g, 1, 64, D, dtype=torch.bfloat16).to(DEV)
    o = torch.tensor([0, n], dtype=torch.int32, device=DEV)
    assert torch.equal(EX.group_linear(x, w, None, o), EX.group_linear(xc, w, None, o))
    assert torch.equal(EX.group_wgrad(x, x, o)[0], EX.group_wgrad(xc, xc, o)[0])
    assert torch.equal(EX.group_dgrad(x, w, o, mask=x), EX.group_dgrad(xc, w, o, mask=xc))
    assert torch.equal(A8.pack(x).codes, A8.pack(xc).codes)
    r = EX.route(randn(g, n, 3).to(DEV), 1)
    assert torch.equal(EX.dispatch(x, r), EX.dispatch(xc, r)) and torch.equal(EX.combine(x, r), EX.combine(xc, r))


# ------------------------------------------------------------------ together
def layer(EX, A8, logits, x, w1, b1, w2, b2, dy, k, x8):
    """One expert layer, forward and backward, as a training step makes it."""
    r = EX.route(logits, k)
    h = EX.group_linear(x, w1, b1, r.offs, relu=True, src=r.src, top_k=k)
    ys = EX.group_linear(h, w2, b2, r.offs)
    y = EX.combine(ys, r)
    kept = A8.pack(h) if x8 else h
    dys, dweight = EX.combine_bwd(dy, ys, r)
    dw2, db2 = EX.group_wgrad(dys, kept, r.offs)
    dh = EX.group_dgrad(dys, w2.transpose(1, 2).contiguous(), r.offs, mask=kept)
    dw1, db1 = EX.group_wgrad(dh, x, r.offs, src=r.src, top_k=k)
    dxs = EX.group_dgrad(dh, w1.transpose(1, 2).contiguous(), r.offs)
    dx = EX.dispatch_bwd(dxs, r)
    return dict(y=y, dx=dx, dw1=dw1, db1=db1, dw2=dw2, db2=db2, dlogits=EX.route_bwd(logits, r, dweight))


def layer_inputs(seed, T=200, D=72, H=96, E=5):
    g = gen(seed)
    bf = torch.bfloat16
    return (randn(g, T, E), randn(g, T, D, dtype=bf), (randn(g, E, H, D) / D ** 0.5).to(bf), 0.1 * randn(g, E, H),
            (randn(g, E, D, H) / H ** 0.5).to(bf), 0.1 * randn(g, E, D), randn(g, T, D, dtype=bf))


@pytest.mark.parametrize("x8", [False, True])
def test_layer_gradients(x8):
    """The whole layer against fp64 autograd of its formula, and along a direction against differences.

    Bound: every bf16 tensor between the operators is off by half a step, 2^-8 of a value, at most 4 of
    them behind one another (h, ys, dys, dh), and e4m3 by 2^-4: relative errors in the 2-norm add up to
    at most 5 * 2^-8, and with 8 bits another 2^-4.  A relu that the rounding of h turns is none: h
    rounds to zero only from zero.  Sums of rounded terms do not raise the 2-norm's relative error
    but where terms cancel, which random signs do by sqrt(n) in terms and errors alike."""
    EX, A8 = ops()
    k = 2
    inp = layer_inputs(7)
    got = layer(EX, A8, *(t.to(DEV) for t in inp), k, x8)
    lg, x, w1, b1, w2, b2, dy = (t.double() for t in inp)
    leaves = [lg, x, w1, b1, w2, b2]
    expert = torch.argsort(-lg, dim=1, stable=True)[:, :k]

    def f(lg, x, w1, b1, w2, b2):
        w = torch.softmax(lg.gather(1, expert), 1)
        y = 0
        for j in range(k):
            e = expert[:, j]
            h = torch.relu((w1[e] @ x[:, :, None])[:, :, 0] + b1[e])
            y = y + w[:, j: j + 1] * ((w2[e] @ h[:, :, None])[:, :, 0] + b2[e])
        return y

    var = [t.clone().requires_grad_() for t in leaves]
    y = f(*var)
    (y * dy).sum().backward()
    tol = 5 * 2.0 ** -8 + (2.0 ** -4 if x8 else 0.0)
    want = dict(zip(("dlogits", "dx", "dw1", "db1", "dw2", "db2"), (v.grad for v in var)), y=y.detach())
    for name, w in want.items():
        d = got[name].double().cpu() - w
        assert float(d.norm() / w.norm()) <= tol, name
    # differences of the formula along one direction, against the kernels' gradients
    g = gen(11)
    u = [torch.randn(t.shape, generator=g, dtype=torch.float64) for t in leaves]
    eps = 1e-6
    hi, lo = (f(*(t + s * eps * q for t, q in zip(leaves, u))) for s in (1, -1))
    num = float((((hi - lo) / (2 * eps)) * dy).sum())
    ana = sum(float((got[n].double().cpu() * q).sum()) for n, q in zip(("dlogits", "dx", "dw1", "db1", "dw2", "db2"), u))
    # an error vector of norm tol |grad| against a random direction: 6 of its standard deviations
    assert abs(num - ana) <= 6 * tol * math.sqrt(sum(float(v.grad.norm()) ** 2 for v in var))


def test_layer_again_other_stream_and_graph():
    """The same bits: called again, on another stream, and replayed from a graph with new inputs in
    between; two graphs alive at once."""
    EX, A8 = ops()
    a, b = (tuple(t.to(DEV) for t in layer_inputs(s)) for s in (1, 2))
    ea, eb = layer(EX, A8, *a, 2, True), layer(EX, A8, *b, 2, True)

    def same(p, q):
        torch.cuda.synchronize()
        live = {n: torch.equal(p[n], q[n]) for n in p}
        assert all(live.values()), live

    same(layer(EX, A8, *a, 2, True), ea)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = layer(EX, A8, *a, 2, True)
    torch.cuda.current_stream().wait_stream(s)
    same(got, ea)
    runs = []
    for first in (a, b):
        inp = tuple(t.clone() for t in first)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layer(EX, A8, *inp, 2, True)
        runs.append((graph, inp, out))
    for rounds in range(3):
        for (graph, inp, out), which, want in ((runs[0], (a, b)[rounds % 2], (ea, eb)[rounds % 2]),
                                               (runs[1], (b, a)[rounds % 2], (eb, ea)[rounds % 2])):
            for t, v in zip(inp, which):
                t.copy_(v)
            graph.replay()
            layer(EX, A8, *b, 2, True)              # eager work between the replays
            same(out, want)


SHARED = [(9000, 1024, 512), (9000, 320, 600), (9000, 333, 601), (700, 256, 256), (150, 40, 72)]


@pytest.mark.parametrize("S,K,N", SHARED)
@pytest.mark.parametrize("stride", [0, 3, 8, 64])
def test_weights_whose_rows_share_memory(S, K, N, stride):
    """Rows a stride apart that is less than their length, in a weight of its own for every expert and in one for all,
    whichever tile the sizes take."""
    EX, _ = ops()
    g = torch.Generator(device=DEV).manual_seed(S + K + stride)
    offs = [0, S // 3, S - 7]
    o = torch.tensor(offs, dtype=torch.int32, device=DEV)
    x = torch.randn(S, K, device=DEV, generator=g).bfloat16()
    mask = torch.randn(S, N, device=DEV, generator=g).bfloat16()
    b = torch.randn(2, N, device=DEV, generator=g)
    src = torch.randperm(S, device=DEV, generator=g).int()
    es = -(-((N - 1) * stride + K) // 8) * 8
    buf = torch.randn(2 * es, device=DEV, generator=g).bfloat16()
    for step in (es, 0):
        w = buf.as_strided((2, N, K), (step, stride, 1))
        results = (("linear", EX.group_linear(x, w, b, o), x), ("through src", EX.group_linear(x, w, b, o, src=src), x[src.long()]),
                   ("gradient", EX.group_dgrad(x, w, o), x), ("masked", EX.group_dgrad(x, w, o, mask=mask), x))
        for what, y, a in results:
            for e in range(2):
                rows = slice(offs[e], offs[e + 1])
                ad, wd = a[rows].double(), w[e].double().contiguous()
                want, mag = ad @ wd.T, ad.abs() @ wd.abs().T
                if what in ("linear", "through src"):
                    want = want + b[e].double()
                if what == "masked":
                    want = torch.where(mask[rows] > 0, want, 0.0)
                bound = HALF[torch.bfloat16] * want.abs() + 1.01 * 2.0 ** -23 * ((K + 4) * mag + want.abs())
                assert bool(((y[rows].double() - want).abs() <= bound).all()), (what, step, e)


@pytest.mark.parametrize("K,off", [(384, 128), (1040, 64), (528, 48), (4000, 96), (1001, 40)])
def test_weight_gradient_from_columns_of_wider_codes(K, off):
    """Codes that are columns of wider rows, up to the last element of their storage: nothing beside them is taken."""
    EX, A8 = ops()
    g = torch.Generator(device=DEV).manual_seed(K)
    S, N = 16384, 520
    offs = [0, 9001, S]
    dz, x = (torch.randn(*s, device=DEV, generator=g).bfloat16() for s in ((S, N), (S, K)))
    a = A8.pack(x)
    wide = torch.full((S, off + K), 127, dtype=torch.uint8, device=DEV)         # (127: NaN)
    wide[:, off:] = a.codes
    o = torch.tensor(offs, dtype=torch.int32, device=DEV)
    src = torch.arange(S, dtype=torch.int32, device=DEV)
    v = A8.unpack(a, torch.float32).double()
    for kw in (dict(), dict(src=src)):
        dw, db = EX.group_wgrad(dz, A8.Act8(wide[:, off:], a.scales), o, **kw)
        for e in range(2):
            lo, hi = offs[e], offs[e + 1]
            z = dz[lo:hi].double()
            c = 1.01 * (hi - lo + 4) * 2.0 ** -23
            assert bool(((dw[e].double() - z.T @ v[lo:hi]).abs() <= c * (z.abs().T @ v[lo:hi].abs())).all()), (len(kw), e)
            assert bool(((db[e].double() - z.sum(0)).abs() <= c * z.abs().sum(0)).all()), (len(kw), e)


def next_to_the_largest(g, S, K, dtype):
    """Rows of ordinary values, some with one of the largest magnitudes in blocks here and there."""
    x = torch.randn(S, K, device=DEV, generator=g)
    big = torch.tensor([3.4028234e38, -3.4028234e38, 248 * 2.0 ** 120, -247.9 * 2.0 ** 120, 255.0 * 2.0 ** 120, 3.3895314e38], device=DEV)
    for i in range(0, S, 97):
        x[i, (7 * i) % K] = big[i % 6]
    x[5 % S, 3 % K] = math.nan
    return x.clamp(-3.3895314e38, 3.3895314e38).to(dtype) if dtype == torch.bfloat16 else x


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,N", [(300, 36), (1000, 401), (64, 4096)])
def test_finite_values_stay_finite_in_8_bits(M, N, dtype):
    """Up to the type's largest: half an e4m3 step, 2^-4 of a value in the format's normal range."""
    _, A8 = ops()
    x = next_to_the_largest(torch.Generator(device=DEV).manual_seed(N), M, N, dtype)
    a = A8.pack(x)
    u, v = A8.unpack(a, torch.float32), A8.unpack(a, torch.bfloat16)
    assert torch.equal(torch.isnan(u), torch.isnan(x)) and not torch.isinf(u).any()
    assert torch.equal(u.nan_to_num(nan=7.0), v.float().nan_to_num(nan=7.0))
    large = x.abs() >= 2.0 ** 115
    assert large.any() and bool(((u.double() - x.double()).abs() <= 2.0 ** -4 * x.double().abs())[large].all())


@pytest.mark.parametrize("S,N,K", [(600, 64, 96), (600, 33, 100), (16384, 512, 256), (16384, 512, 600)])
def test_weight_gradient_from_8_bits_next_to_the_largest(S, N, K):
    EX, A8 = ops()
    g = torch.Generator(device=DEV).manual_seed(S + K)
    x = next_to_the_largest(g, S, K, torch.float32).nan_to_num(nan=0.0)
    dz = (torch.randn(S, N, device=DEV, generator=g) * 2.0 ** -12).bfloat16()
    dz[::3] = 0
    a = A8.pack(x)
    v = A8.unpack(a, torch.float32).double()
    assert bool((v.abs() >= 240 * 2.0 ** 120).any())
    o = torch.tensor([0, S // 2, S], dtype=torch.int32, device=DEV)
    src = torch.arange(S, dtype=torch.int32, device=DEV)
    for kw in (dict(), dict(src=src)):
        dw, _ = EX.group_wgrad(dz, a, o, **kw)
        for e, (lo, hi) in enumerate(((0, S // 2), (S // 2, S))):
            z = dz[lo:hi].double()
            assert bool(((dw[e].double() - z.T @ v[lo:hi]).abs() <= 1.01 * (hi - lo + 4) * 2.0 ** -23 * (z.abs().T @ v[lo:hi].abs())).all())


@pytest.mark.parametrize("S,N,K", [(600, 64, 96), (16384, 512, 256), (16384, 512, 600)])
def test_places_without_a_row_read_zeros_whatever_row_0_holds(S, N, K):
    """Sources that are no slot of a row, beside a row 0 of x that nobody packed: codes and scales of any bits."""
    EX, A8 = ops()
    g = torch.Generator(device=DEV).manual_seed(S + K)
    dz, x = (torch.randn(*s, device=DEV, generator=g).bfloat16() for s in ((S, N), (S, K)))
    a = A8.pack(x)
    o = torch.tensor([0, S // 2, S], dtype=torch.int32, device=DEV)
    src = torch.randint(1, S, (S,), device=DEV, generator=g).int()
    src[::3] = -1
    src[1::5] = S
    want = EX.group_wgrad(dz, a, o, src=src)
    assert bool(torch.isfinite(want[0]).all())
    for code, scale in ((0x33, 255), (0x7F, 0), (0xFF, 255)):
        a.codes[0], a.scales[0] = code, scale
        got = EX.group_wgrad(dz, a, o, src=src)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), (code, scale)
