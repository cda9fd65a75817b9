"""Expert operators in 64 bits, written from their definitions (oracle of the expert tests)."""
import math

import torch

E4M3 = [(-1 if c & 128 else 1) * ((8 + (c & 7)) * 2.0 ** ((c >> 3 & 15) - 10) if c >> 3 & 15 else (c & 7) * 2.0 ** -9)
        if c & 127 != 127 else math.nan for c in range(256)]


def order(expert, E):
    """(pos, src, offs) of the slots ``expert`` [T, k] on the host."""
    T, k = expert.shape
    src = [s for e in range(E) for s in range(T * k) if int(expert.view(-1)[s]) == e] if T * k < 4000 else None
    flat = expert.reshape(-1).long().cpu()
    if src is None:
        key = torch.where(flat < 0, E, flat)
        src = torch.argsort(key, stable=True)[: int((flat >= 0).sum())].tolist()
    offs = torch.zeros(E + 1, dtype=torch.int32)
    for e in range(E):
        offs[e + 1] = offs[e] + int((flat == e).sum())
    pos = torch.full((T * k,), -1, dtype=torch.int32)
    pos[torch.tensor(src, dtype=torch.long)] = torch.arange(len(src), dtype=torch.int32)
    full = torch.full((T * k,), -1, dtype=torch.int32)
    full[: len(src)] = torch.tensor(src, dtype=torch.int32)
    return pos.view(T, k), full, offs


def route(logits, k, renorm, valid=None):
    """(expert, weight, pos, src, offs); selection one by one, weights in fp64."""
    l = logits.double().cpu()
    T, E = l.shape
    l = torch.where(torch.isnan(l), -math.inf, l.clamp(max=float(torch.finfo(torch.float32).max)))
    if valid is not None:
        l[~valid.cpu()] = -math.inf
    idx = torch.argsort(-l, dim=1, stable=True)[:, :k]
    val = l.gather(1, idx)
    dead = val == -math.inf
    m = torch.where(dead[:, :1], 0.0, val[:, :1])
    num = torch.where(dead, 0.0, torch.exp(val - m))
    den = num.sum(1, keepdim=True) if renorm else torch.exp(l - m).sum(1, keepdim=True)
    w = torch.where(den > 0, num / den, 0.0)
    expert = torch.where(dead, -1, idx).int()
    return (expert, w) + order(expert, E)


def group_ids(offs, S):
    """Expert of each row (-1 behind the last) from valid offsets."""
    o = offs.tolist()
    e = torch.full((S,), -1, dtype=torch.long)
    for i in range(len(o) - 1):
        e[o[i]: o[i + 1]] = i
    return e


def pack(x):
    """(codes, scales, values): every block's scale and every code by search over the 256 codes' values."""
    x = x.double().cpu()
    M, N = x.shape
    nb = -(-N // 32)
    fin = torch.isfinite(x)
    xb = torch.zeros(M, nb * 32, dtype=torch.float64)
    xb[:, :N] = torch.where(fin, x, 0.0)
    amax = xb.view(M, nb, 32).abs().amax(2)
    e = torch.full((M, nb), -110, dtype=torch.long)
    for c in range(-109, 121):
        e = torch.where(amax > 448 * 2.0 ** (c - 1), c, e)
    e = e.clamp(max=120)
    s = 2.0 ** e.double()
    q = x / s.repeat_interleave(32, 1)[:, :N]
    grid = torch.tensor(E4M3[:127], dtype=torch.float64)
    a = q.abs()
    hi = torch.searchsorted(grid, a.clamp(max=448)).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    dl, dh = a - grid[lo], grid[hi] - a
    code = torch.where((dh < dl) | ((dh == dl) & (hi % 2 == 0)), hi, lo)
    code = torch.where((code == 0) & (x != 0), 1, code)
    code = torch.where(x < 0, code + 128, code)
    neg0 = (x == 0) & torch.signbit(x)
    code = torch.where(neg0, 128, code)
    code = torch.where(fin, code, code * 0 + 127)
    vals = torch.tensor(E4M3, dtype=torch.float64)[code] * s.repeat_interleave(32, 1)[:, :N]
    return code.to(torch.uint8), (e + 127).to(torch.uint8), vals
