"""Plain forms, in 64 bits, of what a step with drafted trees adds to the 8-bit
paged cache: norm and rotation, attention under a mask, rows kept and copied,
pages trimmed. And trees to test them with."""
import math

import numpy as np
import torch

import paged_fp8_ref as ref

BLOCK = ref.BLOCK


def parents(n, rng):
    """A random tree: each token hangs on one of those before it (-1: the root)."""
    return [-1] + [int(rng.integers(0, i)) for i in range(1, n)]


def paths(par):
    """Ancestors of each token, itself the last."""
    out = []
    for i, p in enumerate(par):
        out.append((out[p] if p >= 0 else []) + [i])
    return out


def mask_words(seen, words):
    """seen: for each token of the batch the drafted tokens that it attends -> int64 [T, words]."""
    m = np.zeros((len(seen), words), np.uint64)
    for t, js in enumerate(seen):
        for j in js:
            if j < 64 * words:
                m[t, j // 64] |= np.uint64(1) << np.uint64(j % 64)
    return torch.from_numpy(m.view(np.int64))


def norm_rotate(x, w, pos, rot, theta, eps, inv_freq=None):
    """x [T, H, D] float64; pos [T, rot / 2] or [T, 1] positions of each pair. -> y, and for each
    value the sum of the sizes of the terms that it is the sum of."""
    x = np.asarray(x, np.float64)
    D = x.shape[-1]
    with np.errstate(invalid="ignore", over="ignore"):
        y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * (1.0 if w is None else w)
    size = np.abs(y)
    if rot:
        f = theta ** (-2.0 * np.arange(rot // 2) / rot) if inv_freq is None else np.asarray(inv_freq, np.float64)
        ang = np.asarray(pos, np.float64) * f
        c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
        a, b = y[..., :rot // 2].copy(), y[..., rot // 2:rot].copy()
        y[..., :rot // 2], y[..., rot // 2:rot] = a * c - b * s, a * s + b * c
        size[..., :rot // 2] = size[..., rot // 2:rot] = np.abs(a) + np.abs(b)
    return y, size


def streams(pos3, sections, rot):
    """Positions [T, rot / 2] of the pairs of interleaved mRoPE."""
    j = np.arange(rot // 2)
    by = np.where((j % 3 == 1) & (j // 3 < sections[1]), 1, np.where((j % 3 == 2) & (j // 3 < sections[2]), 2, 0))
    return np.asarray(pos3)[by].T


def tree_attention(q, k, v, held, base, n, seen):
    """q [N, Hq, D] of one request; k, v [H, L, D] float64 of its rows, held [L]: rows that have a
    page; token i attends held rows [0, base) and base + j for j in seen[i]. As ref.attention."""
    N, Hq, D = q.shape
    H, L = k.shape[:2]
    G = Hq // H
    out = torch.zeros((N, Hq, D), dtype=torch.float64, device=q.device)
    mag, big = torch.zeros_like(out), torch.zeros((N, Hq, 1), dtype=torch.float64, device=q.device)
    for i in range(N):
        ok = torch.zeros(L, dtype=torch.bool)
        ok[:max(0, min(base, L))] = True
        for j in seen[i]:
            if j < n and 0 <= base + j < L:
                ok[base + j] = True
        sel = (ok.to(held.device) & held).nonzero().view(-1)
        if not len(sel):
            continue
        x = q[i].double().view(H, G, D)
        s = (x[:, :, None] * k[:, None, sel]).sum(-1) / math.sqrt(D)
        w = torch.softmax(s, -1)
        out[i] = (w[..., None] * v[:, None, sel]).sum(2).reshape(Hq, D)
        mag[i] = (w[..., None] * v[:, None, sel].abs()).sum(2).reshape(Hq, D)
        big[i, :, 0] = ((x.abs()[:, :, None] * k[:, None, sel].abs()).sum(-1) / math.sqrt(D)).amax(2).reshape(Hq)
    return out, mag, big


def keep(cache, table, cached, kept, counts, page):
    """cache: a ref.Cache, changed in place; lists in. -> lens"""
    P, H = cache.val.shape[:2]
    mp, lens = len(table[0]), []
    for b, c in enumerate(cached):
        if c < 0:
            lens.append(c)
            continue
        n = max(0, min(counts[b], len(kept[b]), mp * page - c))
        lens.append(c + n)
        path = kept[b][:n]
        first = next((i for i, k in enumerate(path) if k != i), n)

        def place(row):
            if not 0 <= row < mp * page:
                return None
            p = table[b][row // page]
            return (p, row % page) if 0 <= p < P else None

        at = (c + first) // BLOCK * BLOCK
        while first < n and at < c + n:
            dst = place(at)
            rows = {}
            for r in range(at, min(at + BLOCK, c + n)):
                src = place(r) if r < c + first else place(c + path[r - c]) if path[r - c] >= 0 else None
                if src is not None:
                    rows[r] = src
            if dst is not None and rows:
                for h in range(H):
                    sc = {r: (cache.scale[dst[0], h, dst[1] // BLOCK] if r < c + first else cache.scale[p, h, x // BLOCK]) for r, (p, x) in rows.items()}
                    top = max(sc.values())
                    val = {r: ref.e4m3(cache.val[p, h, x] * (sc[r] / top)) for r, (p, x) in rows.items()}
                    for r, x in val.items():
                        cache.val[dst[0], h, dst[1] + r - at] = x
                    cache.scale[dst[0], h, dst[1] // BLOCK] = top
            at += BLOCK
    return lens


def copy(cache, table, src, dst, lens, max_len, page):
    P = cache.val.shape[0]
    for s, d, n in zip(src, dst, lens):
        n = min(n, max_len)
        if not (0 <= s < len(table) and 0 <= d < len(table)):
            continue
        for r in range(0, max(n, 0), BLOCK):
            a, z = table[s][r // page], table[d][r // page]
            if 0 <= a < P and 0 <= z < P:
                x = r % page
                cache.val[z, :, x:x + BLOCK] = cache.val[a, :, x:x + BLOCK]
                cache.scale[z, :, x // BLOCK] = cache.scale[a, :, x // BLOCK]


def trim(lens, table, free, count, page):
    table, free = [list(r) for r in table], list(free)
    for b, n in enumerate(lens):
        for p in range(-(-n // page) if n >= 0 else len(table[b]), len(table[b])):
            e = table[b][p]
            if e < 0:
                break
            if count < len(free):
                free[count] = e
                count += 1
            table[b][p] = -1
    return table, free, count
