"""Measured cases of the expert and 8-bit-checkpoint operators (hipfm.ops.experts, hipfm.ops.act8).

Operators of a deep tower whose layers are mixtures of experts, and whose activations are kept
in 8 bits for the backward pass:

* ``route``    a gate's logits -> the top_k experts of every token, their weights, and the order that
               puts the (token, choice) slots of one expert side by side; and the gate's gradient
* ``exchange`` tokens copied into that order, the experts' rows brought back with the weights
               applied, and the gradients of both
* ``linear``   one layer of every expert over its own rows (bias, relu), forward
* ``backward`` its two gradient products: towards the input (masked by the relu of the layer below)
               and towards the weights and biases; the input kept in bf16, or in 8 bits
* ``pack``     activations to 8 bits (e4m3 codes, one power-of-two scale per row and 32 columns) and back

``own`` chooses the side: the plain form in elementary torch operations, or the framework's calls.
"""
import math

import torch

own = False


# ------------------------------------------------------------------ cases
def listed():
    return [
        # a request of 48 candidates scored by 8 experts: launch latency is all there is
        dict(name="route serve", op="route", T=48, E=8, k=2, dtype="f32", renorm=True, masked=False, grad=False),
        # a training batch of 16384 rows (the benchmark's), its last part padding, and the gate's gradient
        dict(name="route train", op="route", T=16384, E=64, k=2, dtype="f32", renorm=False, masked=True, grad=True),
        # many fine-grained experts, a ragged batch, bf16 gate logits (equal logits occur)
        dict(name="route fine experts", op="route", T=20011, E=256, k=8, dtype="bf16", renorm=True, masked=True, grad=True),
        # the same request's rows to its experts and back (a 400-wide layer), forward only
        dict(name="exchange serve", op="exchange", T=96, D=400, E=8, k=2, dtype="bf16", masked=False, grad=False),
        # a training batch of 39 fields x 32 = 1248 inputs per row, both directions
        dict(name="exchange train", op="exchange", T=16384, D=1248, E=16, k=2, dtype="bf16", masked=True, grad=True),
        # fp32 rows whose length fits no vector load, every row sent to every expert (multi-gate towers)
        dict(name="exchange odd f32", op="exchange", T=10007, D=313, E=4, k=4, dtype="f32", masked=True, grad=True),
        # the request's expert layer: few rows per expert, the weights' bytes are the time
        dict(name="linear serve", op="linear", S=192, K=1248, N=400, E=8, relu=True, gather=True, tail=0),
        # a training batch's expert layer, rows taken from the tokens through the order
        dict(name="linear train", op="linear", S=32768, K=1248, N=1024, E=16, relu=True, gather=True, tail=513),
        # its backward pass from bf16 activations
        dict(name="backward train", op="backward", S=32768, K=1024, N=1024, E=16, x8=False, tail=513),
        # the 4096-wide dense tower's layer (one expert) from activations kept in 8 bits
        dict(name="backward wide 8 bits", op="backward", S=16384, K=4096, N=4096, E=1, x8=True, tail=0),
        # activations of a small fp32 layer whose width is no multiple of the scale's 32 columns
        dict(name="pack odd f32", op="pack", M=1000, N=401, dtype="f32"),
        # a 4096-wide layer's activations of a training batch
        dict(name="pack wide", op="pack", M=16384, N=4096, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """A layer width: mostly a multiple of 8, sometimes any number."""
    n = _log_int(rng, lo, hi)
    return n if rng.random() < 0.25 else max(8, n // 8 * 8)


def draw(rng):
    op = rng.choice(["route", "exchange", "linear", "backward", "pack"])
    if op == "route":
        E = _log_int(rng, 2, 256)
        return dict(op=op, T=_log_int(rng, 1, 20011), E=E, k=rng.randint(1, min(8, E)), dtype=rng.choice(["f32", "bf16"]),
                    renorm=rng.random() < 0.5, masked=rng.random() < 0.5, grad=rng.random() < 0.7)
    if op == "exchange":
        E = _log_int(rng, 2, 64)
        k = rng.randint(1, min(4, E))
        D = _width(rng, 16, 4096)
        T = _log_int(rng, 1, min(16384, 40_000_000 // (D * k)))
        return dict(op=op, T=T, D=D, E=E, k=k, dtype=rng.choice(["f32", "bf16", "bf16"]), masked=rng.random() < 0.5,
                    grad=rng.random() < 0.7)
    if op == "pack":
        N = _width(rng, 16, 8192)
        return dict(op=op, M=_log_int(rng, 1, min(32768, 67_000_000 // N)), N=N, dtype=rng.choice(["f32", "bf16"]))
    E = _log_int(rng, 1, 64)
    K, N = _width(rng, 32, 4096), _width(rng, 32, 4096)
    while E * K * N > 1 << 26:
        E = max(1, E // 2)
    S = _log_int(rng, 1, min(32768, (1 << 38) // (K * N)))
    tail = rng.choice([0, 0, 77])
    if op == "linear":
        return dict(op=op, S=S, K=K, N=N, E=E, relu=rng.random() < 0.5, gather=rng.random() < 0.5, tail=tail)
    return dict(op=op, S=S, K=K, N=N, E=E, x8=rng.random() < 0.5, tail=tail)


_TYPE = {"f32": torch.float32, "bf16": torch.bfloat16}


# ------------------------------------------------------------------ inputs
def _order(expert, E):
    """The expert order of the slots ``expert`` [T, k] (-1: none): (pos [T, k], src [T k], offs [E + 1])."""
    T, k = expert.shape
    flat = expert.reshape(-1).long()
    key = torch.where(flat < 0, torch.full_like(flat, E), flat)
    by = torch.sort(key, stable=True).indices
    offs = torch.zeros(E + 1, dtype=torch.int64, device=expert.device)
    offs[1:] = torch.cumsum(torch.bincount(key, minlength=E + 1)[:E], 0)
    rank = torch.arange(T * k, device=expert.device)
    live = rank < offs[E]
    src = torch.where(live, by, -1).int()
    pos = torch.empty_like(rank)
    pos[by] = rank
    pos = torch.where(flat < 0, -1, pos).int().reshape(T, k)
    return pos, src, offs.int()


def _valid(T, g, dev):
    """Rows that hold a sample: the batch's first nine tenths, but for a few rows that were refused."""
    v = torch.arange(T, device=dev) < max(1, T - T // 10)
    return v & (torch.rand(T, device=dev, generator=g) > 0.02)


def _ragged(S, E, g, dev):
    """Offsets of S rows over E experts, some much fuller than others."""
    share = torch.softmax(torch.randn(E, device=dev, generator=g), 0)
    cut = torch.cumsum(share.double(), 0)
    offs = torch.zeros(E + 1, dtype=torch.int64, device=dev)
    offs[1:] = torch.floor(cut / cut[-1] * S + 0.5).long()
    offs[E] = S
    return offs.int()


def _two_to(e):
    """2^e of whole e in [-126, 127], exactly: the bits of the fp32 value."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _pack_plain(x):
    """(codes uint8 [M, N], scales uint8 [M, ceil(N / 32)]) of x [M, N], in elementary operations.

    A block of 32 columns of a row has the scale 2^e with the smallest e that keeps its largest
    finite magnitude within 448, e in [-110, 120], stored as e + 127. A code is the e4m3 value
    nearest to x / 2^e (ties to even), but a value that is not zero never becomes a zero; what is
    not finite becomes NaN."""
    M, N = x.shape
    nb = -(-N // 32)
    xf = torch.zeros(M, nb * 32, dtype=torch.float32, device=x.device)
    xf[:, :N] = x.float()
    xb = xf.view(M, nb, 32)
    fin = torch.isfinite(xb)
    amax = torch.where(fin, xb.abs(), 0.0).amax(2)
    m, ex = torch.frexp(amax)                           # amax = m 2^ex, m in [0.5, 1); 448 = 0.875 2^9
    e = torch.where(amax > 0, torch.clamp(ex - 9 + (m > 0.875).int(), -110, 120), -110)
    q = xb * _two_to(-e)[:, :, None]
    c = q.to(torch.float8_e4m3fn).view(torch.uint8)
    c = torch.where((c & 127 == 0) & (xb != 0), c | 1, c)
    c = torch.where(fin, c, c | 127)
    return c.view(M, nb * 32)[:, :N].contiguous(), (e + 127).to(torch.uint8)


def _unpack_plain(codes, scales):
    N = codes.shape[1]
    s = _two_to(scales.int() - 127)
    return codes.view(torch.float8_e4m3fn).float() * s.repeat_interleave(32, 1)[:, :N]


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)

    def randn(*shape, dtype=torch.float32):
        return torch.randn(*shape, device=dev, generator=g).to(dtype)

    op, s = case["op"], {"case": case}
    if op == "route":
        T, E, k = case["T"], case["E"], case["k"]
        # a trained gate prefers some experts; a few choices are closed (-inf), rows and experts alike
        lg = randn(T, E) * 1.5 + randn(E)
        closed = torch.rand(T, E, device=dev, generator=g) < 0.02
        s["logits"] = torch.where(closed, float("-inf"), lg).to(_TYPE[case["dtype"]])
        s["valid"] = _valid(T, g, dev) if case["masked"] else None
        if case["grad"]:
            s["dweight"] = randn(T, k)
        return s
    if op == "exchange":
        T, D, E, k = case["T"], case["D"], case["E"], case["k"]
        dt = _TYPE[case["dtype"]]
        expert = (torch.rand(T, E, device=dev, generator=g) * torch.rand(E, device=dev, generator=g)).argsort(1)[:, :k].int()
        if case["masked"]:
            expert = torch.where(_valid(T, g, dev)[:, None], expert, -1)
        s["expert"], s["weight"] = expert, torch.where(expert < 0, 0.0, torch.softmax(randn(T, k), 1))
        s["pos"], s["src"], s["offs"] = _order(expert, E)
        s["x"], s["ys"] = randn(T, D, dtype=dt), randn(T * k, D, dtype=dt)
        s["xs_out"], s["y_out"] = torch.zeros(T * k, D, dtype=dt, device=dev), torch.zeros(T, D, dtype=dt, device=dev)
        if case["grad"]:
            s["dy"], s["dxs"] = randn(T, D, dtype=dt), randn(T * k, D, dtype=dt)
            s["dys_out"], s["dx_out"] = torch.zeros_like(s["xs_out"]), torch.zeros_like(s["y_out"])
        return s
    if op == "pack":
        # what a relu leaves: half of the values zero, columns of very different sizes
        x = randn(case["M"], case["N"]) * torch.exp(2 * randn(case["N"]))
        s["x"] = torch.relu(x).to(_TYPE[case["dtype"]])
        return s
    S, K, N, E, tail = (case[v] for v in ("S", "K", "N", "E", "tail"))
    s["offs"] = _ragged(S, E, g, dev)
    s["w"] = (randn(E, N, K) / math.sqrt(K)).to(torch.bfloat16)
    if op == "linear":
        s["b"] = randn(E, N)
        T = (S + 1) // 2 if case["gather"] else S + tail
        s["x"] = randn(T, K, dtype=torch.bfloat16)
        if case["gather"]:                               # two slots for each token
            s["src"] = torch.full((S + tail,), -1, dtype=torch.int32, device=dev)
            s["src"][:S] = torch.randperm(2 * T, device=dev, generator=g)[:S].int()
        s["out"] = torch.zeros(S + tail, N, dtype=torch.bfloat16, device=dev)
        return s
    s["wt"] = s["w"].transpose(1, 2).contiguous()       # the transposed copy that a training program keeps
    s["dz"] = randn(S + tail, N, dtype=torch.bfloat16)
    h = torch.relu(randn(S + tail, K)).to(torch.bfloat16)
    if case["x8"]:
        s["codes"], s["scales"] = _pack_plain(h)
    else:
        s["x"] = h
    s["dx_out"] = torch.zeros(S + tail, K, dtype=torch.bfloat16, device=dev)
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    case = s["case"]
    if own:
        return _OWN[case["op"]](s, case)
    return _PLAIN[case["op"]](s, case)


def _own_route(s, c):
    from hipfm.ops import experts as EX
    r = EX.route(s["logits"], c["k"], renormalize=c["renorm"], valid=s["valid"])
    out = dict(expert=r.expert, weight=r.weight, pos=r.pos, src=r.src, offs=r.offs)
    if c["grad"]:
        out["dlogits"] = EX.route_bwd(s["logits"], r, s["dweight"], renormalize=c["renorm"])
    return out


def _own_exchange(s, c):
    from hipfm.ops import experts as EX
    r = EX.Routes(s["expert"], s["weight"], s["pos"], s["src"], s["offs"])
    out = dict(xs=EX.dispatch(s["x"], r, out=s["xs_out"]), y=EX.combine(s["ys"], r, out=s["y_out"]))
    if c["grad"]:
        out["dx"] = EX.dispatch_bwd(s["dxs"], r, out=s["dx_out"])
        out["dys"], out["dweight"] = EX.combine_bwd(s["dy"], s["ys"], r, out=s["dys_out"])
    return out


def _own_linear(s, c):
    from hipfm.ops import experts as EX
    gather = dict(src=s["src"], top_k=2) if c["gather"] else {}
    return EX.group_linear(s["x"], s["w"], s["b"], s["offs"], relu=c["relu"], out=s["out"], **gather)


def _own_backward(s, c):
    from hipfm.ops import experts as EX
    from hipfm.ops import act8 as A8
    x = A8.Act8(s["codes"], s["scales"]) if c["x8"] else s["x"]
    dx = EX.group_dgrad(s["dz"], s["wt"], s["offs"], mask=x, scale=1.25, out=s["dx_out"])
    dw, db = EX.group_wgrad(s["dz"], x, s["offs"])
    return dict(dx=dx, dw=dw, db=db)


def _own_pack(s, c):
    from hipfm.ops import act8 as A8
    a = A8.pack(s["x"])
    return dict(values=A8.unpack(a, s["x"].dtype), scales=a.scales)


def _plain_route(s, c):
    T, E, k = c["T"], c["E"], c["k"]
    lg = s["logits"].float()
    lg = torch.where(torch.isnan(lg), float("-inf"), lg.clamp(max=torch.finfo(torch.float32).max))
    if s["valid"] is not None:
        lg = torch.where(s["valid"][:, None], lg, float("-inf"))
    top = torch.sort(lg, dim=1, descending=True, stable=True)
    tv, ti = top.values[:, :k], top.indices[:, :k]
    dead = tv == float("-inf")
    base = torch.where(dead[:, :1], 0.0, tv[:, :1])
    ex = torch.exp(lg - base)
    et = torch.where(dead, 0.0, torch.exp(tv - base))
    den = (et if c["renorm"] else ex).sum(1, keepdim=True)
    inv = torch.where(den > 0, 1.0 / den, 0.0)
    w = et * inv
    expert = torch.where(dead, -1, ti).int()
    pos, src, offs = _order(expert, E)
    out = dict(expert=expert, weight=w, pos=pos, src=src, offs=offs)
    if c["grad"]:
        dw = torch.where(dead, 0.0, s["dweight"])
        dot = (w * dw).sum(1, keepdim=True)
        d = torch.zeros_like(lg) if c["renorm"] else -(ex * inv) * dot
        d.scatter_add_(1, ti, w * (dw - dot) if c["renorm"] else w * dw)
        out["dlogits"] = d.to(s["logits"].dtype)
    return out


def _back(rows, pos):
    """rows[pos] with zeros where pos is -1, in fp32: [T, k, D]."""
    got = rows.float()[pos.clamp(min=0).long()]
    return torch.where(pos[:, :, None] < 0, 0.0, got)


def _plain_exchange(s, c):
    dt, k, pos = s["x"].dtype, c["k"], s["pos"]
    live = s["src"] >= 0
    tok = s["src"].clamp(min=0).long() // k

    def sorted_rows(rows):
        return torch.where(live[:, None], rows, torch.zeros((), dtype=rows.dtype, device=rows.device))

    out = dict(xs=sorted_rows(s["x"][tok]), y=(_back(s["ys"], pos) * s["weight"][:, :, None]).sum(1).to(dt))
    if c["grad"]:
        out["dx"] = _back(s["dxs"], pos).sum(1).to(dt)
        w = s["weight"].reshape(-1)[s["src"].clamp(min=0).long()]
        out["dys"] = sorted_rows((s["dy"][tok].float() * w[:, None]).to(dt))
        out["dweight"] = (_back(s["ys"], pos) * s["dy"].float()[:, None, :]).sum(2)
    return out


def _padded(offs, rows, S):
    """Where the sorted rows lie in [E, cap, .], cap the fullest expert's rows: (place [rows], live [rows], cap)."""
    E = offs.numel() - 1
    cap = max(1, int((offs[1:] - offs[:-1]).max()))
    p = torch.arange(rows, device=offs.device)
    e = torch.searchsorted(offs[1:].contiguous(), p.int(), right=True).clamp(max=E - 1)
    live = p < S
    return e * cap + (p - offs[e]), live, cap


def _by_expert(rows, place, live, E, cap):
    out = torch.zeros(E * cap, rows.shape[1], dtype=torch.float32, device=rows.device)
    out[place[live]] = rows[live].float()
    return out.view(E, cap, -1)


def _from_experts(y, place, live, like):
    out = torch.zeros_like(like)
    out[live] = y.reshape(-1, y.shape[2])[place[live]].to(like.dtype)
    return out


def _plain_linear(s, c):
    S, E, rows = c["S"], c["E"], c["S"] + c["tail"]
    place, live, cap = _padded(s["offs"], rows, S)
    x = s["x"][s["src"].clamp(min=0).long() // 2] if c["gather"] else s["x"]
    y = torch.bmm(_by_expert(x, place, live, E, cap), s["w"].float().transpose(1, 2).contiguous()) + s["b"][:, None, :]
    if c["relu"]:
        y = torch.relu(y)
    return _from_experts(y, place, live, s["out"])


def _plain_backward(s, c):
    S, E, rows = c["S"], c["E"], c["S"] + c["tail"]
    place, live, cap = _padded(s["offs"], rows, S)
    x = _unpack_plain(s["codes"], s["scales"]) if c["x8"] else s["x"].float()
    dz = _by_expert(s["dz"], place, live, E, cap)
    dx = torch.bmm(dz, s["w"].float()) * 1.25
    dx = torch.where(_by_expert(x, place, live, E, cap) > 0, dx, 0.0)
    dw = torch.bmm(dz.transpose(1, 2).contiguous(), _by_expert(x, place, live, E, cap))
    return dict(dx=_from_experts(dx, place, live, s["dx_out"]), dw=dw, db=dz.sum(1))


def _plain_pack(s, c):
    codes, scales = _pack_plain(s["x"])
    return dict(values=_unpack_plain(codes, scales).to(s["x"].dtype), scales=scales)


_PLAIN = dict(route=_plain_route, exchange=_plain_exchange, linear=_plain_linear, backward=_plain_backward, pack=_plain_pack)
_OWN = dict(route=_own_route, exchange=_own_exchange, linear=_own_linear, backward=_own_backward, pack=_own_pack)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    op = case["op"]
    if op == "route":
        T, E, k = case["T"], case["E"], case["k"]
        el = _TYPE[case["dtype"]].itemsize
        b = T * E * el + T * k * 16 + (E + 1) * 4 + (T if case["masked"] else 0)
        f = T * E * (3 + k)
        if case["grad"]:
            b, f = b + T * E * el + T * k * 4, f + 4 * T * E
        return {"bytes": b, "flops": f}
    if op == "exchange":
        T, D, k = case["T"], case["D"], case["k"]
        row = D * _TYPE[case["dtype"]].itemsize
        b, f = 2 * (T + T * k) * row + T * k * 12, 2 * T * k * D
        if case["grad"]:
            b, f = 2 * b + T * k * 4, 3 * f
        return {"bytes": b, "flops": f}
    if op == "pack":
        M, N = case["M"], case["N"]
        return {"bytes": M * N * (2 * _TYPE[case["dtype"]].itemsize + 2) + 2 * M * -(-N // 32), "flops": 4 * M * N}
    S, K, N, E = (case[v] for v in ("S", "K", "N", "E"))
    if op == "linear":
        T = (S + 1) // 2 if case["gather"] else S
        return {"bytes": 2 * (T * K + E * N * K + S * N) + 4 * E * N, "flops": 2 * S * N * K}
    xb = S * K + S * -(-K // 32) if case["x8"] else 2 * S * K
    return {"bytes": 2 * (S * N + E * N * K + S * K) + xb + 4 * (E * N * K + E * N), "flops": 4 * S * N * K}


# ------------------------------------------------------------------ the definition, in 64 bits
def _power(e):
    """2^e of whole e, exactly: the bits of the fp64 value."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def exact(case, seed):
    s = prepare(case, seed)
    return _EXACT[case["op"]](s, case)


def _exact_route(s, c):
    lg = s["logits"].double()
    if s["valid"] is not None:
        lg[~s["valid"]] = -math.inf
    sel = torch.argsort(-lg, dim=1, stable=True)[:, : c["k"]]
    chosen = torch.zeros_like(lg, dtype=torch.bool).scatter_(1, sel, True) & torch.isfinite(lg)
    shown = torch.where(chosen, lg, -math.inf) if c["renorm"] else lg
    p = torch.nan_to_num(torch.softmax(shown, 1), nan=0.0)
    w = (p * chosen).gather(1, sel)
    out = dict(expert=None, weight=w, pos=None, src=None, offs=None)
    if c["grad"]:
        dp = torch.zeros_like(lg).scatter_(1, sel, s["dweight"].double()) * chosen
        out["dlogits"] = p * (dp - (p * dp).sum(1, keepdim=True))
    return out


def _exact_exchange(s, c):
    k, live = c["k"], s["expert"] >= 0
    t, j = torch.nonzero(live, as_tuple=True)
    at = s["pos"][t, j].long()
    w = s["weight"].double()[t, j]
    x, ys = s["x"].double(), s["ys"].double()
    xs = torch.zeros_like(ys)
    xs[at] = x[t]
    out = dict(xs=xs, y=torch.zeros_like(x).index_add_(0, t, ys[at] * w[:, None]))
    if c["grad"]:
        dy = s["dy"].double()
        out["dx"] = torch.zeros_like(x).index_add_(0, t, s["dxs"].double()[at])
        dys = torch.zeros_like(ys)
        dys[at] = dy[t] * w[:, None]
        out["dys"], out["dweight"] = dys, torch.zeros(c["T"], k, dtype=torch.float64, device=x.device)
        out["dweight"][t, j] = (ys[at] * dy[t]).sum(1)
    return out


def _exact_linear(s, c):
    y = torch.zeros(s["out"].shape, dtype=torch.float64, device=s["out"].device)
    o = s["offs"].tolist()
    for e in range(c["E"]):
        rows = slice(o[e], o[e + 1])
        x = s["x"][torch.div(s["src"][rows], 2, rounding_mode="floor").long()] if c["gather"] else s["x"][rows]
        y[rows] = x.double() @ s["w"][e].double().T + s["b"][e].double()
    return y.clamp(min=0) if c["relu"] else y


def _exact_backward(s, c):
    if c["x8"]:                                          # sign, exponent and mantissa of each code
        v = s["codes"].int()
        ex, man = (v >> 3) & 15, v & 7
        x = torch.where(ex > 0, (8 + man).double() * _power(ex - 10), man.double() * 2.0 ** -9)
        x = torch.where(v > 127, -x, x) * _power(s["scales"].int() - 127).repeat_interleave(32, 1)[:, : c["K"]]
    else:
        x = s["x"].double()
    dx = torch.zeros_like(x)
    dw = torch.zeros(c["E"], c["N"], c["K"], dtype=torch.float64, device=x.device)
    db = torch.zeros(c["E"], c["N"], dtype=torch.float64, device=x.device)
    o = s["offs"].tolist()
    for e in range(c["E"]):
        rows = slice(o[e], o[e + 1])
        dz = s["dz"][rows].double()
        dx[rows] = (dz @ s["w"][e].double()) * 1.25 * (x[rows] > 0)
        dw[e], db[e] = dz.T @ x[rows], dz.sum(0)
    return dict(dx=dx, dw=dw, db=db)


def _exact_pack(s, c):
    x = s["x"].double()
    b = torch.nn.functional.pad(x, (0, -c["N"] % 32)).view(c["M"], -1, 32)
    big = b.abs().amax(2, keepdim=True)
    _, e = torch.frexp(big / 448)                        # big / 448 = m 2^e, m in [0.5, 1)
    e = torch.where(big <= 448 * _power(e - 1), e - 1, e).clamp(-110, 120)
    q = b / _power(e)
    step = _power(torch.frexp(q.abs().clamp(min=2.0 ** -6))[1] - 4)
    r = torch.round(q / step) * step
    r = torch.where((r == 0) & (q != 0), torch.sign(q) * 2.0 ** -9, r)
    return dict(values=(r * _power(e)).view(c["M"], -1)[:, : c["N"]], scales=None)


_EXACT = dict(route=_exact_route, exchange=_exact_exchange, linear=_exact_linear, backward=_exact_backward, pack=_exact_pack)
