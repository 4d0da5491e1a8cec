"""The paged cache's operators from their definitions, in 64 bits and with
loops, on the CPU."""
import math

import torch


def place(table, pages, page, b, p):
    """(page, row) of place p of sequence b; None where there is no page."""
    if p // page >= table.shape[1]:
        return None
    at = int(table[b, p // page])
    return (at, p % page) if 0 <= at < pages else None


def turn(x, positions, inv_freq):
    """Rotate adjacent pairs of x [rows, heads, D]."""
    if inv_freq is None:
        return x.double()
    angle = positions.double()[:, None] * inv_freq.double()
    x = x.double().reshape(*x.shape[:2], -1, 2)
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    return torch.stack((x[..., 0] * c - x[..., 1] * s,
                        x[..., 0] * s + x[..., 1] * c), -1).flatten(-2)


def keys_values(pool, table, b, n):
    """K, V [kv heads, n, D] of sequence b, and which places are there."""
    page = pool.shape[-2]
    k = torch.zeros(pool.shape[1], n, pool.shape[-1], dtype=torch.float64)
    v, there = k.clone(), torch.zeros(n, dtype=torch.bool)
    for p in range(n):
        at = place(table, pool.shape[0], page, b, p)
        if at:
            there[p] = True
            k[:, p] = pool[at[0], :, 0, at[1]].double()
            v[:, p] = pool[at[0], :, 1, at[1]].double()
    return k, v, there


def weights(q, k, there, scale, seen=None):
    """Softmax of q [G, rows, D] over k [n, D]; zeros where nothing is seen.
    Also the largest |q||k| sum, which bounds the rounding of the scores."""
    s = q @ k.T * scale
    size = float((q.abs() @ k.abs().T).max() * abs(scale)) if k.numel() else 0.
    hidden = ~there if seen is None else ~(there & seen)
    s = s.masked_fill(hidden, -math.inf)
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(top == -math.inf, 0., top))
    e = torch.where(hidden, torch.zeros_like(e), e)
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total == 0, 1., total), size


def attend(q, pool, table, lens, scale):
    """out [B, heads, D], added mass [B, kv heads, most], sum w|V|, size."""
    B, H, D = q.shape
    heads = pool.shape[1]
    G, most = H // heads, table.shape[1] * pool.shape[-2]
    out = torch.zeros(B, H, D, dtype=torch.float64)
    big, mass = out.clone(), torch.zeros(B, heads, most, dtype=torch.float64)
    size = 0.
    for b in range(B):
        n = max(0, min(int(lens[b]), most))
        if not n:
            continue
        k, v, there = keys_values(pool, table, b, n)
        for h in range(heads):
            w, s = weights(q[b, h * G:(h + 1) * G].double(), k[h], there,
                           scale)
            size = max(size, s)
            out[b, h * G:(h + 1) * G] = w @ v[h]
            big[b, h * G:(h + 1) * G] = w @ v[h].abs()
            mass[b, h, :n] = w.sum(0)
    return out, mass, big, size


def observe(q, pool, table, lens, starts, scale):
    """Added mass [B, kv heads, most], and size as above."""
    H, heads = q.shape[1], pool.shape[1]
    B, G, most = table.shape[0], H // heads, table.shape[1] * pool.shape[-2]
    mass, size = torch.zeros(B, heads, most, dtype=torch.float64), 0.
    for b in range(B):
        t0, t1 = int(starts[b]), int(starts[b + 1])
        n, m = max(0, min(int(lens[b]), most)), t1 - t0
        if not n or m <= 0:
            continue
        k, _, there = keys_values(pool, table, b, n)
        seen = torch.arange(n)[None] <= (n - m + torch.arange(m))[:, None]
        for h in range(heads):
            x = q[t0:t1, h * G:(h + 1) * G].double().transpose(0, 1)
            w, s = weights(x, k[h], there, scale, seen)
            size = max(size, s)
            mass[b, h, :n] = w.sum((0, 1))
    return mass, size


def survivors(mass, pos, late, keep):
    """The places that stay of one row, by the order's definition."""
    def rank(p):
        w = float(mass[p])
        if int(pos[p]) >= late:
            return (0, 0., p)
        return (1, math.inf if math.isnan(w) else -w, p)
    return set(sorted(range(len(mass)), key=rank)[:keep])


def evict(pool, table, lens, next_pos, mass, pos, keep, recent, limit):
    """In place, on the CPU."""
    page, cap = pool.shape[-2], mass.shape[-1]
    for b in range(table.shape[0]):
        n = max(0, min(int(lens[b]), cap))
        if n <= limit:
            continue
        for l in range(pool.shape[1]):
            for h in range(pool.shape[2]):
                stay = survivors(mass[l, b, h, :n], pos[l, b, h, :n],
                                 int(next_pos[b]) - recent, keep)
                free = [p for p in range(keep) if p not in stay]
                come = [p for p in range(keep, n) if p in stay]
                assert len(free) == len(come)
                for d, s in zip(free, come):
                    mass[l, b, h, d] = mass[l, b, h, s]
                    pos[l, b, h, d] = pos[l, b, h, s]
                    a = place(table, pool.shape[0], page, b, d)
                    c = place(table, pool.shape[0], page, b, s)
                    if a and c:
                        pool[a[0], l, h, :, a[1]] = pool[c[0], l, h, :, c[1]]
        lens[b] = keep
