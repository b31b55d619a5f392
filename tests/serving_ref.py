"""The serving operators' definitions in 64 bits, on the CPU, one sequence, page and head at a time (test aid)."""
import math

import torch

MIN_EXP = -60
STEP = {torch.bfloat16: 2.0 ** -8, torch.float8_e4m3fn: 2.0 ** -4}   # the most that one rounding moves a value, relative to it


def to_e4m3(x):
    """x (float64) to the nearest e4m3 number, ties to even; NaN and infinities are NaN."""
    _, e = torch.frexp(torch.where(torch.isfinite(x), x, torch.zeros_like(x)))
    step = torch.exp2((e - 1).clamp(min=-6).double() - 3)
    return torch.where(torch.isfinite(x), (torch.round(x / step) * step).clamp(-448, 448), torch.full_like(x, math.nan))


def scale_for(y):
    """Smallest 2^n, n >= -60, with every finite |y| <= 448 2^n."""
    top = float(torch.where(torch.isfinite(y), y, torch.zeros_like(y)).abs().max()) if y.numel() else 0.0
    n = MIN_EXP
    while top > 448 * 2.0 ** n:
        n += 1
    return 2.0 ** n


def rotate(x, cos, sin):
    """x [T, heads, hd] by the rows cos, sin [T, hd/2], in the precision of x."""
    h = x.shape[-1] // 2
    x1, x2, c, s = x[..., :h], x[..., h:], cos[:, None].to(x.dtype), sin[:, None].to(x.dtype)
    return torch.cat((x1 * c - x2 * s, x2 * c + x1 * s), -1)


def append(codes, scales, y, before, new, table):
    """In place: codes [pages, kv, P, hd] and scales [pages, kv] as float64; y [T, kv, hd] (float64, rotated)."""
    P, first = codes.shape[2], 0
    for b, (n0, n) in enumerate(zip(before, new)):
        for j in range(n0 // P, (n0 + n + P - 1) // P) if n0 >= 0 else ():
            lo, hi = max(n0, j * P), min(n0 + n, (j + 1) * P)
            if lo >= hi:
                continue
            page, had = int(table[b][j]), lo - j * P
            for h in range(codes.shape[1]):
                rows = y[first + lo - n0:first + hi - n0, h]
                now = max(scale_for(rows), float(scales[page, h]) if had else 0.0)
                codes[page, h, :had] = to_e4m3(codes[page, h, :had] * (float(scales[page, h]) / now))
                codes[page, h, had:had + hi - lo] = to_e4m3(rows / now)
                scales[page, h] = now
        first += n


def attend(q, k, v, visible, scale):
    """q [rows, hd], k, v [keys, hd] float64, visible [rows, keys] -> (o, lse); what is not visible is not touched, whatever it holds."""
    o, lse = torch.zeros_like(q), torch.full((q.shape[0],), -math.inf, dtype=torch.float64)
    for r in range(q.shape[0]):
        at = visible[r].nonzero()[:, 0]
        if at.numel() == 0:
            continue
        x = (k[at] @ q[r]) * scale
        lse[r] = torch.logsumexp(x, 0)
        o[r] = torch.exp(x - lse[r]) @ v[at]
    return o, lse


def attend_causal(q, k, v, scale, causal=True):
    """The same for whole heads q [lq, H, hd], k, v [lk, kv, hd]; causal from the lower right corner."""
    lq, H, lk, kv = q.shape[0], q.shape[1], k.shape[0], k.shape[1]
    vis = torch.ones(lq, lk, dtype=torch.bool)
    if causal:
        vis = torch.arange(lk)[None] <= torch.arange(lq)[:, None] + (lk - lq)
    o, lse = torch.zeros_like(q), torch.zeros(lq, H, dtype=torch.float64)
    for h in range(H):
        g = h // (H // kv)
        x = (q[:, h] @ k[:, g].T * scale).masked_fill(~vis, -math.inf)
        l = torch.logsumexp(x, -1) if lk else torch.full((lq,), -math.inf, dtype=torch.float64)
        w = torch.nan_to_num(torch.exp(x - l[:, None]), nan=0.0)
        o[:, h], lse[:, h] = w @ v[:, g], l
    return o, lse


def ints(values, device="cuda"):
    return torch.tensor(values, dtype=torch.int32, device=device)


def tables(n, hd, device="cuda", theta=10000.0):
    ang = torch.arange(n).double()[:, None] / theta ** (torch.arange(0, hd, 2).double() / hd)
    return ang.cos().float().to(device), ang.sin().float().to(device)


def page_tables(total, P, spare=2, seed=0, unused=-1):
    """(rows of page numbers for sequences of `total` tokens, in random order; pages in the pool)."""
    need = [-(-max(n, 0) // P) for n in total]
    order = torch.randperm(sum(need) + spare, generator=torch.Generator().manual_seed(seed)).tolist()
    width, rows = max(need + [1]) + 1, []
    for n in need:
        rows.append([order.pop() for _ in range(n)] + [unused] * (width - n))
    return rows, sum(need) + spare
