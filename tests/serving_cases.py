"""Plain 64-bit forms of the serving operators (page plan, 8-bit paged cache,
attention over it, sampling) for the tests, one value at a time where that is
clearest."""
import math

import numpy as np
import torch


def plan(cached, new, ended, table, free, count, page, tokens):
    """The page plan on lists and numpy arrays; table and free are changed in place."""
    top = count
    for r, n in enumerate(ended):
        for j in range(-(-n // page)):
            free[top] = table[r][j]
            top += 1
    starts, positions, slots = [0], [], []
    for r in range(len(cached)):
        for j in range(-(-cached[r] // page), -(-(cached[r] + new[r]) // page)):
            top -= 1
            table[r][j] = free[top]
        for p in range(cached[r], cached[r] + new[r]):
            positions.append(p)
            slots.append(table[r][p // page] * page + p % page)
        starts.append(starts[-1] + new[r])
    pad = [-1] * (tokens - len(slots))
    return starts, [a + b for a, b in zip(cached, new)], positions + pad, slots + pad, top


def scale_exponent(big):
    """The smallest e >= -126 with big <= 127 * 2^e (None for 0)."""
    if big == 0:
        return None
    e = max(-126, math.frexp(big)[1] - 8)
    while big > math.ldexp(127, e):
        e += 1
    return e


def store(x, slots, codes, scales):
    """Rows x [tokens, heads, dim] (float64) into codes and scales (float64 arrays), in place."""
    page = codes.shape[2]
    at = 0
    while at < len(slots):
        if slots[at] < 0:
            at += 1
            continue
        p, off = divmod(int(slots[at]), page)
        n = 1
        while at + n < len(slots) and off + n < page and slots[at + n] == slots[at] + n:
            n += 1
        for h in range(codes.shape[1]):
            rows = x[at:at + n, h]
            old = scales[p, h] if off else 0.0
            if not np.isfinite(rows).all() or np.isnan(old):
                scales[p, h] = np.nan
                codes[p, h, off:off + n] = 0
                continue
            e = scale_exponent(np.abs(rows).max())
            scale = max(math.ldexp(1.0, e) if e is not None else 0.0, old)
            if off and old > 0 and scale != old:
                codes[p, h, :off] = np.rint(codes[p, h, :off] * (old / scale))
            codes[p, h, off:off + n] = np.rint(rows / scale) if scale else 0
            scales[p, h] = scale
        at += n


def attention(q, starts, lens, table, codes, scales, scale):
    """(out, tolerance) of [rows, heads, dim] float64: codes, scales = (k, v) pairs of tensors.

    The tolerance is that of f32 sums over parts of 22 bits: a score's sum over
    dim rounds at most dim / 8 + 4 times at 2^-23 of sum |q k|; a weight is off by
    ln 2 of that (in bits) and by 2^-20 (its power, its parts, the sum); the
    sum over keys rounds once for each 16 of them."""
    rows, heads, dim = q.shape
    kv_heads, page = codes[0].shape[1:3]
    group = heads // kv_heads
    out = torch.zeros(rows, heads, dim, dtype=torch.float64, device=q.device)
    tol = torch.zeros(rows, heads, 1, dtype=torch.float64, device=q.device)
    q = q.double()
    for r, L in enumerate(lens):
        a, b = starts[r], starts[r + 1]
        if b == a or L == 0:
            continue
        ids = table[r, : -(-L // page)].long()
        seen = torch.arange(L, device=q.device)[None, :] <= torch.arange(L - (b - a), L, device=q.device)[:, None]
        for g in range(kv_heads):
            k, v = ((c[ids, g].double() * s[ids, g].double()[:, None, None]).reshape(-1, dim)[:L]
                    for c, s in zip(codes, scales))
            for h in range(g * group, (g + 1) * group):
                x = (q[a:b, h] @ k.T * scale).masked_fill(~seen, -math.inf)
                w = torch.softmax(x, 1).nan_to_num(0.0) if not x.isnan().any() else torch.softmax(x, 1)
                w = torch.where(seen, w, torch.zeros_like(w))
                out[a:b, h] = torch.where(seen.any(1)[:, None], w @ torch.where(seen.any(0)[:, None], v, torch.zeros_like(v)), 0)
                mass = (q[a:b, h].abs() @ k.abs().T * abs(scale) * 1.4427).masked_fill(~seen, 0).amax(1, keepdim=True)
                ew = 0.6932 * mass * 2.0 ** -23 * (dim / 8 + 4) + 2.0 ** -20 + (L / 16 + 8) * 2.0 ** -23
                tol[a:b, h] = 2 * ew * v.abs().max()
    return out, tol


def pick(logits, temperature, k, p, m, u):
    """(token, kept, prob) of one row of float64 logits."""
    x = np.where(np.isnan(logits), -np.inf, logits)
    alive = int((x > -np.inf).sum())
    if alive == 0:
        return -1, 0, 0.0
    if not temperature > 0:
        return int(np.argmax(x)), 1, 1.0
    order = np.argsort(-x, kind="stable")[:alive]
    top = x[order[0]]
    with np.errstate(invalid="ignore"):
        w = (x[order] == np.inf).astype(np.float64) if top == np.inf else np.exp((x[order] - top) / temperature)
    n = alive
    if 0 < k < len(x):
        n = min(n, k)
    if p < 1:
        n = min(n, max(1, 1 + int(np.searchsorted(np.cumsum(w), p * w[:n].sum(), side="left"))))
    if m > 0:
        n = min(n, int((w >= min(m, 1.0)).sum()))
    some = np.argsort(order[:n])
    mass = np.cumsum(w[some])
    i = min(int(np.searchsorted(mass, u * mass[-1], side="right")), n - 1)
    while w[some[i]] == 0:
        i -= 1
    return int(order[some[i]]), n, float(w[some[i]] / mass[-1])
