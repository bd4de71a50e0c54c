"""Operators of a server of many requests, in 64 bits with numpy: rotary
positions, head norms, cache page moves, low-rank adapters.  Plain loops from
the definitions; none of the package's code."""

import numpy as np


def rope_pairs(rd, layout):
    """(a, b): indices of the values that turn together."""
    i = np.arange(rd // 2)
    return (2 * i, 2 * i + 1) if layout == "interleaved" else (i, i + rd // 2)


def rope_row(x, cos, sin, layout):
    """x [..., D] float64 turned by cos, sin [rd / 2]."""
    a, b = rope_pairs(2 * len(cos), layout)
    y = x.copy()
    y[..., a] = x[..., a] * cos - x[..., b] * sin
    y[..., b] = x[..., a] * sin + x[..., b] * cos
    return y


def rope(x, cos, sin, positions, layout):
    """x [B,S,H,D], positions [B,S] (negative: a row of zeros)."""
    x, cos, sin = (np.asarray(t, np.float64) for t in (x, cos, sin))
    y = np.zeros_like(x)
    for b in range(x.shape[0]):
        for s in range(x.shape[1]):
            p = positions[b, s]
            if 0 <= p < len(cos):
                y[b, s] = rope_row(x[b, s], cos[p], sin[p], layout)
    return y


def head_norm(x, w, eps):
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w


def qk_norm_rope(qkv, cos, sin, positions, Hq, Hkv, D, wq, wk, eps, layout):
    """(q [T,Hq,D], k [T,Hkv,D], v, largest magnitude that each q and k value is a sum of)."""
    x = np.asarray(qkv, np.float64).reshape(len(qkv), Hq + 2 * Hkv, D)
    n = x.copy()
    if wq is not None:
        n[:, :Hq] = head_norm(x[:, :Hq], np.asarray(wq, np.float64), eps)
        n[:, Hq:Hq + Hkv] = head_norm(x[:, Hq:Hq + Hkv], np.asarray(wk, np.float64), eps)
    out, size = n.copy(), np.abs(n)
    for t, p in enumerate(positions):
        if not 0 <= p < len(cos):
            out[t, :Hq] = 0.0
            continue
        out[t, :Hq + Hkv] = rope_row(n[t, :Hq + Hkv], np.asarray(cos[p], np.float64), np.asarray(sin[p], np.float64),
                                     layout)
        a, b = rope_pairs(2 * cos.shape[1], layout)
        both = np.abs(n[t][:, a]) + np.abs(n[t][:, b])
        size[t][:, a], size[t][:, b] = both, both
    return out[:, :Hq], out[:, Hq:Hq + Hkv], x[:, Hq + Hkv:], size[:, :Hq + Hkv]


def fork(table, lengths, refs, parents, P, reserve, num_pages):
    """Row b of the new table continues parents[b] (negative: nobody).  Returns
    (table, lengths, refs, ready, moves [(src, dst)])."""
    B, blocks = table.shape
    refs = refs.astype(np.int64).copy()
    valid = lambda p: 0 <= p < num_pages  # noqa: E731
    for p in table.reshape(-1):
        if valid(p):
            refs[p] -= 1
    n = len(parents)
    new = np.full((n, blocks), -1, np.int64)
    L = np.zeros(n, np.int64)
    for b, p in enumerate(parents):
        if not 0 <= p < B:
            continue
        L[b] = min(max(int(lengths[p]), 0), blocks * P)
        for j in range(-(-L[b] // P)):
            if valid(table[p, j]):
                new[b, j] = table[p, j]
                refs[table[p, j]] += 1
    live = np.array([0 <= p < B for p in parents], bool)
    ready = np.ones(n, bool)
    moves = []
    if reserve > 0:
        nb = -(-L // P)
        last = [int(new[b, nb[b] - 1]) if L[b] % P else -1 for b in range(n)]
        after = refs.copy()
        free = [int(p) for p in np.nonzero(refs == 0)[0]]
        used = 0
        for b in range(n):
            if not live[b]:
                continue
            if L[b] + reserve > blocks * P:
                ready[b] = False
                continue
            copy = False
            if last[b] >= 0:
                rows = [r for r in range(n) if last[r] == last[b]]
                keeper = max(rows, key=lambda r: (L[r] % P, -r))
                copy = not (keeper == b and refs[last[b]] == len(rows))
            need = int(copy) + int(-(-(L[b] + reserve) // P) - nb[b])
            got = free[used:used + need]
            used += need
            if need and used > len(free):
                ready[b] = False
                continue
            for p in got:
                after[p] = 1
            if copy:
                after[last[b]] -= 1
                moves.append((last[b], got[0]))
                new[b, nb[b] - 1] = got[0]
                got = got[1:]
            new[b, nb[b]:nb[b] + len(got)] = got
        refs = after
    return new, L, refs, ready, moves


def compact(table, refs):
    """(table, refs, page map, live pages, moves) with the live pages at ids [0, live)."""
    held = refs > 0
    n = int(held.sum())
    src = [p for p in range(len(refs)) if held[p] and p >= n]
    dst = [p for p in range(len(refs)) if not held[p] and p < n]
    page_map = np.where(held, np.arange(len(refs)), -1)
    page_map[src] = dst
    new_refs = np.zeros_like(refs)
    for p in range(len(refs)):
        if held[p]:
            new_refs[page_map[p]] = refs[p]
    new = np.full(table.shape, -1, np.int64)
    for i in np.ndindex(*table.shape):
        if 0 <= table[i] < len(refs):
            new[i] = page_map[table[i]]
    return new, new_refs, page_map, n, list(zip(src, dst))


def lora(x, base, a, b, ids, scales):
    """(base + s (x A^T) B^T, sum of the magnitudes that an output is a sum of)."""
    x, base, a, b = (np.asarray(t, np.float64) for t in (x, base, a, b))
    out, size = base.copy(), np.abs(base)
    for m, i in enumerate(ids):
        if 0 <= i < len(a):
            s = 1.0 if scales is None else float(scales[i])
            out[m] += s * (b[i] @ (a[i] @ x[m]))
            size[m] += abs(s) * (np.abs(b[i]) @ (np.abs(a[i]) @ np.abs(x[m])))
    return out, size
