"""The paged operators in 64 bits, slot by slot, on CPU tensors (test infrastructure).

``Pages`` reads and writes slots of rows through a table; every function takes the inputs of an operator and returns what it has to give,
with bounds on what 32-bit arithmetic and the roundings to the storage type may add."""
import math

import torch

U32 = 2.0 ** -24                                    # half a step of fp32, relative


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def place(table, P, page, row, slot):
    """(page id, offset) of a slot, or None where the table names no place."""
    if not (0 <= row < table.shape[0]) or not (0 <= slot < table.shape[1] * page):
        return None
    p = int(table[row, slot // page])
    return (p, slot % page) if 0 <= p < P else None


def visible(n, first, window):
    return [j for j in range(n) if window == 0 or j < first or j >= n - window]


def append(qkv, k, v, mass, table, t_row, t_slot, t_pos, H, rates, pairs, qw, kw, eps):
    """-> (q [M, H, D] or NaN for idle tokens, k, v, mass, bound of q's and k's error beyond their rounding), all float64."""
    P, G, page, D = k.shape
    M = t_row.numel()
    x = qkv.double()[:, :(H + 2 * G) * D].reshape(M, H + 2 * G, D)
    k, v = k.double().clone(), v.double().clone()
    mass = None if mass is None else mass.double().clone()
    q = torch.full((M, H, D), math.nan, dtype=torch.float64)
    bound = 0.0
    n = 0 if rates is None else rates.numel()
    for t in range(M):
        r, s = int(t_row[t]), int(t_slot[t])
        if r < 0 or r >= table.shape[0]:
            continue
        y = x[t].clone()
        for lo, hi, w in ((0, H, qw), (H, H + G, kw)):
            if w is not None:
                y[lo:hi] = y[lo:hi] / torch.sqrt(y[lo:hi].square().mean(-1, keepdim=True) + eps) * w.double()
        if n:
            ang = float(t_pos[t]) * rates.double()
            a, b = (slice(0, n), slice(n, 2 * n)) if pairs == 0 else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
            z = y[:H + G].clone()
            y[:H + G, a] = z[:, a] * ang.cos() - z[:, b] * ang.sin()
            y[:H + G, b] = z[:, a] * ang.sin() + z[:, b] * ang.cos()
        # norm: the sum of D squares, root, quotient and two products; rotation: sine and cosine to 2 steps of an angle that is right to one step of a
        # half-turn (pi * U32), two products and a sum
        bound = max(bound, float(y[:H + G].abs().max()) * 2 * (D / 8 + 8 + 12) * U32)
        q[t] = y[:H]
        at = place(table, P, page, r, s)
        if at is not None:
            k[at[0], :, at[1]], v[at[0], :, at[1]] = y[H:H + G], y[H + G:]
            if mass is not None:
                mass[at[0], :, at[1]] = 0.0
    return q, k, v, mass, bound


def attn(q, k, v, mass, table, t_row, t_slot, H, scale, first, window, p_bits):
    """-> (out [M, H, D] with NaN for idle tokens, its error bound beyond the rounding of the result, mass, its error bound).  ``p_bits``: relative error
    of the weights' form that multiplies the values."""
    P, G, page, D = k.shape
    M, per = t_row.numel(), H // G
    out = torch.full((M, H, D), math.nan, dtype=torch.float64)
    tol = torch.zeros((M, H, D), dtype=torch.float64)
    q = q.double().view(M, H, D)
    new = None if mass is None else mass.double().clone()
    off = None if mass is None else torch.zeros_like(new)
    for t in range(M):
        r, s = int(t_row[t]), int(t_slot[t])
        if r < 0 or r >= table.shape[0]:
            continue
        n = max(0, min(s + 1, table.shape[1] * page))
        at = [place(table, P, page, r, j) for j in visible(n, first, window)]
        at = [x for x in at if x is not None]
        if not at:
            out[t] = 0.0
            continue
        pid, o = torch.tensor([x[0] for x in at]), torch.tensor([x[1] for x in at])
        kk, vv = k[pid, :, o].double(), v[pid, :, o].double()                       # [n, G, D]
        for g in range(G):
            heads = slice(g * per, (g + 1) * per)
            qh = q[t, heads]
            sc = qh @ kk[:, g].T * scale
            # scores: D products and sums in fp32 in any order, the scale folded in (and a step for each of exp's argument and value)
            ds = (2 * (D + 4) * U32 * scale * (qh.abs() @ kk[:, g].abs().T) + 4 * U32 * sc.abs()).amax(-1) + 8 * U32
            p = torch.softmax(sc, -1)
            out[t, heads] = p @ vv[:, g]
            near = p @ vv[:, g].abs()
            tol[t, heads] = near * ((2 * ds)[:, None] + p_bits + 2 * (len(at) / 8 + 32) * U32)
            if new is not None:
                w = p.sum(0)
                new[pid, g, o] += w
                off[pid, g, o] += ((2 * ds)[:, None] * p).sum(0) + w * 2 * (len(at) / 8 + 32) * U32
    if new is not None:
        off += 4 * U32 * new.abs()
    return out, tol, new, off


def select(mass, table, lengths, keep, first, recent):
    P, G, page = mass.shape
    kept = torch.full((table.shape[0], G, keep), -1, dtype=torch.int64)
    for r in range(table.shape[0]):
        n = max(0, min(int(lengths[r]), table.shape[1] * page))
        for g in range(G):
            if n <= keep:
                kept[r, g, :n] = torch.arange(n)
                continue
            score = []
            for j in range(first, n - recent):
                at = place(table, P, page, r, j)
                x = -math.inf if at is None else float(mass[at[0], g, at[1]])
                score.append(((-math.inf, 0) if at is None or math.isnan(x) else (x, 1), -j))
            best = sorted(score, reverse=True)[:keep - first - recent]
            kept[r, g] = torch.tensor(sorted(list(range(first)) + [-b[1] for b in best] + list(range(n - recent, n))))
    return kept


def compact(k, v, mass, table, lengths, kept):
    P, G, page, D = k.shape
    old = [None if t is None else t.clone() for t in (k, v, mass)]
    new = [None if t is None else t.clone() for t in (k, v, mass)]
    for r in range(table.shape[0]):
        for g in range(G):
            for i, j in enumerate(kept[r, g].tolist()):
                a, b = place(table, P, page, r, j), place(table, P, page, r, i)
                if j > i and j < int(lengths[r]) and a is not None and b is not None:
                    for src, dst in zip(old, new):
                        if src is not None:
                            dst[b[0], g, b[1]] = src[a[0], g, a[1]]
    return new


def gather(pages, table, rows, lengths, dense, extra):
    P, G, page, D = pages.shape
    dense = dense.clone()
    for i, r in enumerate(rows.tolist()):
        if 0 <= r < table.shape[0]:
            for j in range(min(int(lengths[r]) + extra, dense.shape[2], table.shape[1] * page)):
                at = place(table, P, page, r, j)
                if at is not None:
                    dense[i, :, j] = pages[at[0], :, at[1]]
    return dense
