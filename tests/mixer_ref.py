"""The token mixer's operators in 64 bits on the CPU, from their definitions,
with the magnitudes that error bounds go by.  Test infrastructure only."""

import numpy as np
import torch


def tables(cached, added, table, free, page, rows):
    """paged_tables, request by request: (table, slots, positions, requests,
    cu, lengths, counts) as lists / numpy."""
    table = table.copy()
    R, P = table.shape
    f, wanted = 0, 0
    cu, lengths, tokens = [0], [], []
    for r in range(R):
        c, n = max(int(cached[r]), 0), max(int(added[r]), 0)
        have, need = -(-c // page), -(-(c + n) // page)
        for e in range(have, min(need, P)):
            table[r, e] = free[f] if f < len(free) else -1
            f += f < len(free)
            wanted += 1
        for pos in range(c, c + n):
            p = int(table[r, pos // page]) if pos // page < P else -1
            tokens.append((p * page + pos % page if p >= 0 else -1, pos, r))
        cu.append(cu[-1] + n)
        lengths.append(c + n)
    tokens = (tokens + [(-1, 0, -1)] * rows)[:max(rows, 0)] if len(tokens) < rows else tokens[:rows]
    slots, positions, requests = (np.array([t[i] for t in tokens], dtype=np.int64)
                                  for i in range(3))
    return (table, slots, positions, requests, np.array(cu), np.array(lengths),
            np.array([cu[-1], min(wanted, len(free)), max(wanted - len(free), 0)]))


def axis_of(i, half, sections, woven):
    if woven:
        a = i % len(sections)
        return a if i // len(sections) < sections[a] else 0
    for a, n in enumerate(sections):
        if i < n:
            return a
        i -= n


def rotary(x, positions, inv_freq, sections, woven=False, adjacent=False):
    """x [N, H, D], positions [A, N] -> float64 [N, H, D]."""
    half = len(inv_freq)
    x = x.double().clone()
    y = x.clone()
    for i in range(half):
        a = axis_of(i, half, sections, woven)
        angle = positions[a].double() * inv_freq[i].double()
        c, s = angle.cos()[:, None], angle.sin()[:, None]
        lo, hi = (2 * i, 2 * i + 1) if adjacent else (i, i + half)
        y[..., lo] = x[..., lo] * c - x[..., hi] * s
        y[..., hi] = x[..., lo] * s + x[..., hi] * c
    return y


def attention(q, k_cache, v_cache, table, lengths, scale, window=0, k_scale=1.0, v_scale=1.0):
    """(out, lse, weighted |v|, largest error unit of a score) in float64:
    q [R, Hq, D], caches [pages, Hk, page, D]."""
    R, hq, D = q.shape
    pages, hk, page, _ = k_cache.shape
    out = torch.zeros(R, hq, D, dtype=torch.float64)
    lse = torch.full((R, hq), -torch.inf, dtype=torch.float64)
    size, unit = torch.zeros_like(out), torch.zeros_like(lse)
    for r in range(R):
        n = min(int(lengths[r]), table.shape[1] * page)
        keys = [j for j in range(max(0, n - window) if window else 0, n)
                if 0 <= int(table[r, j // page]) < pages]
        if not keys:
            continue
        at = torch.tensor([int(table[r, j // page]) for j in keys])
        off = torch.tensor([j % page for j in keys])
        k, v = k_cache[at, :, off].double() * k_scale, v_cache[at, :, off].double() * v_scale
        for h in range(hq):
            kk, vv, x = k[:, h * hk // hq], v[:, h * hk // hq], q[r, h].double()
            s = kk @ x * scale
            p = torch.softmax(s, 0)
            out[r, h], size[r, h] = p @ vv, p @ vv.abs()
            lse[r, h] = torch.logsumexp(s, 0)
            unit[r, h] = (kk.abs() @ x.abs()).max() * abs(scale) + s.abs().max()
    return out, lse, size, unit


def linear(q, k, v, g, cu, state, beta=None, index=None, scale=None):
    """Token by token in float64: (out, state_out, bound of |out|'s terms,
    bound of |state|'s terms).  The bounds follow the recurrence with every
    factor's absolute value."""
    N, vh, dv = v.shape
    dk = q.shape[2]
    each = vh // q.shape[1]
    scale = dk ** -0.5 if scale is None else scale
    out, size = torch.zeros(N, vh, dv, dtype=torch.float64), torch.zeros(N, vh, dv, dtype=torch.float64)
    final, fsize = state.double().clone(), state.double().abs()
    q, k = (x.double().repeat_interleave(each, dim=1) for x in (q, k))
    v, g = v.double(), g.double()
    for r in range(len(cu) - 1):
        i = r if index is None else int(index[r])
        keep = 0 <= i < len(state)
        S = state[i].double().clone() if keep else torch.zeros(vh, dk, dv, dtype=torch.float64)
        B = S.abs()
        for t in range(int(cu[r]), int(cu[r + 1])):
            a = g[t].exp()[:, None, None]
            u, ub = v[t], v[t].abs()
            if beta is not None:
                b = beta[t].double()[:, None]
                u = b * (u - ((a * S) * k[t][..., None]).sum(1))
                # |u| <= beta (|v| + |k| |S|); the update shrinks S along k by
                # 1 - beta, so |k| |S| of the state as it is bounds that term
                ub = b * (ub + ((a * S).abs() * k[t].abs()[..., None]).sum(1))
            S = a * S + k[t][..., None] * u[:, None]
            B = torch.maximum(a * B, S.abs()) + k[t].abs()[..., None] * ub[:, None]
            out[t] = scale * (S * q[t][..., None]).sum(1)
            size[t] = abs(scale) * (B * q[t].abs()[..., None]).sum(1)
        if keep:
            final[i], fsize[i] = S, B
    return out, final, size, fsize
