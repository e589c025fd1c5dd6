"""The serving operators from their definitions, in 64 bits on the CPU."""
import math

import torch


def norm_rotate(x, w, table, pos, eps, interleaved):
    """x [B,N,H,D] float64, pos [B,N] long -> float64."""
    y = x
    if w is not None:
        y = x * (x.pow(2).mean(-1, keepdim=True) + eps).rsqrt() * w
    if table is None:
        return y
    rot = table.shape[1]
    c, s = table[pos][..., None, : rot // 2], table[pos][..., None, rot // 2:]
    z = y.clone()
    if interleaved:
        a, b = y[..., 0:rot:2], y[..., 1:rot:2]
        z[..., 0:rot:2], z[..., 1:rot:2] = a * c - b * s, a * s + b * c
    else:
        a, b = y[..., : rot // 2], y[..., rot // 2: rot]
        z[..., : rot // 2], z[..., rot // 2: rot] = a * c - b * s, a * s + b * c
    return z


def visible(n, window, sinks):
    return [e for e in range(n) if not window or e < sinks or e >= n - window]


def rows_of(pool, page_table, b, slots):
    """The rows [len(slots), Hkv, D] of sequence b, one at a time, with the last dimensions of any pool."""
    size = pool.shape[1]
    return torch.stack([pool[int(page_table[b, e // size]), e % size] for e in slots]) if slots else pool.new_zeros((0, *pool.shape[2:]))


def decode(Q, pools, page_table, lengths, window=0, sinks=0):
    """(Y, sum of P |Vr o Vs|, shares as {(page, slot, head): share}) in float64."""
    B, Hq, D = Q.shape
    Hkv, size = pools[0].shape[2], pools[0].shape[1]
    G = Hq // Hkv
    Y, A, share = torch.zeros(B, Hq, D, dtype=torch.float64), torch.zeros(B, Hq, D, dtype=torch.float64), {}
    for b in range(B):
        slots = visible(int(lengths[b]), window, sinks)
        if not slots:
            continue
        R, S, Vr, Vs = (rows_of(p, page_table, b, slots).double() for p in pools)
        for h in range(Hq):
            k = h // G
            x = (Q[b, h].double() * R[:, k]) @ S[:, k].T / math.sqrt(D)
            p = torch.softmax(x.flatten(), 0).view_as(x)
            Y[b, h] = ((p @ Vs[:, k]) * Vr[:, k]).sum(0)
            A[b, h] = ((p @ Vs[:, k].abs()) * Vr[:, k].abs()).sum(0)
            part = (p.sum(0) + p.sum(1)) / (2 * G)
            for e, v in zip(slots, part.tolist()):
                at = (int(page_table[b, e // size]), e % size, k)
                share[at] = share.get(at, 0.0) + v
    return Y, A, share


def evict(mass, page_table, lengths, keep, sinks, recent):
    """Kept slots per sequence and key head, as lists."""
    out = []
    for b in range(page_table.shape[0]):
        n, row = int(lengths[b]), []
        m = rows_of(mass, page_table, b, list(range(n)))
        for h in range(mass.shape[2]):
            def rank(e):
                v = float(m[e, h])
                return (0 if e < sinks or e >= n - recent else 1, -math.inf if math.isnan(v) else -v, 0 if math.isnan(v) else 1, e)
            row.append(sorted(sorted(range(n), key=rank)[:keep]) if n > keep else list(range(n)))
        out.append(row)
    return out
