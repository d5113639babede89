"""Plain forms of the 8-bit paged cache's operators, in 64 bits: the page tables
request by request, the quantisation row by row, attention token by token."""
import math

import numpy as np
import torch

BLOCK = 16


def e4m3(x):
    """Nearest e4m3 value of x (float64 array), ties to even, saturated."""
    a = np.abs(x)
    with np.errstate(divide="ignore", invalid="ignore"):
        unit = np.exp2(np.maximum(np.floor(np.log2(np.where(a > 0, a, 1.0))), -6.0) - 3.0)
        y = np.clip(np.rint(x / unit) * unit, -448.0, 448.0)
    return np.where(np.isfinite(x), y, np.nan)


def code_values():
    """The 256 codes' values, from the format: 1 sign, 4 exponent (bias 7), 3 mantissa bits."""
    v = np.empty(256)
    for c in range(256):
        e, m = c >> 3 & 15, c & 7
        x = math.nan if e == 15 and m == 7 else m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        v[c] = -x if c & 128 else x
    return v


def scale_exp(amax):
    """Smallest integer e with amax <= 448 * 2^e, within [-100, 119]."""
    if amax == 0:
        return -100
    e = math.frexp(amax / 448.0)[1] - 1
    while amax > 448.0 * 2.0 ** e:
        e += 1
    return min(max(e, -100), 119)


class Cache:
    """One of K and V: values [P, H, page, D] and exponents [P, H, page / 16]."""

    def __init__(self, codes, scale):
        self.val = code_values()[codes.view(torch.uint8).cpu().numpy()]
        self.scale = scale.double().cpu().numpy().copy()

    def append(self, x, slots):
        """x [T, H, D] float64."""
        page = self.val.shape[2]
        t, T = 0, len(slots)
        while t < T:
            s = slots[t]
            if s < 0 or s >= self.val.shape[0] * page:
                t += 1
                continue
            r0, n = s % BLOCK, 1
            while t + n < T and r0 + n < BLOCK and slots[t + n] == s + n:
                n += 1
            p, r, blk = s // page, s % page, s % page // BLOCK
            for h in range(self.val.shape[1]):
                rows = x[t:t + n, h]
                e = scale_exp(float(np.max(np.where(np.isfinite(rows), np.abs(rows), 0.0))))
                if r0 > 0:
                    old = min(max(math.frexp(self.scale[p, h, blk])[1] - 1, -100), 119)
                    if e > old:
                        head = self.val[p, h, r - r0:r]
                        self.val[p, h, r - r0:r] = e4m3(head * 2.0 ** (old - e))
                    e = max(e, old)
                with np.errstate(over="ignore"):
                    self.val[p, h, r:r + n] = e4m3(rows * 2.0 ** -e)
                self.scale[p, h, blk] = 2.0 ** e
            t += n

    def rows(self, slots):
        page = self.val.shape[2]
        out = np.zeros((len(slots), self.val.shape[1], self.val.shape[3]))
        for i, s in enumerate(slots):
            if 0 <= s < self.val.shape[0] * page:
                out[i] = self.val[s // page, :, s % page] * self.scale[s // page, :, s % page // BLOCK][:, None]
        return out


def reserve(cached, new, table, free, count, page, capacity):
    """Lists in, (table, count, starts, lens, slots) out."""
    B, mp = len(cached), len(table[0])
    table = [list(r) for r in table]
    starts, lens, slots, need, taken = [0], [], [-1] * capacity, 0, 0
    for b in range(B):
        c, n = cached[b], new[b]
        if c < 0 or n < 0:
            starts.append(starts[-1])
            lens.append(0)
            continue
        starts.append(starts[-1] + n)
        fits = c + n <= mp * page
        holes = [p for p in range(c // page, -(-(c + n) // page)) if table[b][p] < 0] if fits else []
        need += len(holes)
        if not fits or starts[-1] > capacity or (holes and need > count):
            lens.append(0)
            continue
        for p in holes:
            table[b][p] = free[count - 1 - taken]
            taken += 1
        lens.append(c + n)
        for i in range(n):
            slots[starts[b] + i] = table[b][(c + i) // page] * page + (c + i) % page
    return table, count - taken, starts, lens, slots


def release(flags, table, free, count):
    table, free = [list(r) for r in table], list(free)
    for b, f in enumerate(flags):
        for p, e in enumerate(table[b]):
            if f and e >= 0:
                free[count] = e
                count += 1
                table[b][p] = -1
    return table, free, count


def gather(codes, scale, table, rows):
    """[H, rows, D] float64 of one request; rows without a page are NaN. -> values, held [rows]."""
    P, H, page, D = codes.shape
    n = -(-rows // page)
    t = table[:n].long()
    ok = (t >= 0) & (t < P)
    t = t.where(ok, 0)
    x = codes.view(torch.uint8)[t].view(codes.dtype).double() * scale[t].double().repeat_interleave(BLOCK, 2)[..., None]
    return x.permute(1, 0, 2, 3).reshape(H, n * page, D)[:, :rows], ok.repeat_interleave(page)[:rows]


def attention(q, k, v, held, first):
    """q [N, Hq, D] of one request whose token i attends held rows [0, first + i).
    Returns (out, bound on what the softmax weights carry: sum p |v|, and the
    largest sum of |q k| / sqrt(D) of a row), all in float64."""
    N, Hq, D = q.shape
    H, L = k.shape[:2]
    G = Hq // H
    out = torch.zeros((N, Hq, D), dtype=torch.float64, device=q.device)
    mag, big = torch.zeros_like(out), torch.zeros((N, Hq, 1), dtype=torch.float64, device=q.device)
    for i in range(N):
        n = max(0, min(first + i, L))
        sel = held[:n].nonzero().view(-1)
        if not len(sel):
            continue
        for h in range(H):
            kk, vv, qq = k[h, sel], v[h, sel], q[i, h * G:(h + 1) * G].double()
            s = (qq[:, None, :] * kk[None]).sum(-1) / math.sqrt(D)
            w = torch.softmax(s, -1)
            out[i, h * G:(h + 1) * G] = (w[:, :, None] * vv[None]).sum(1)
            mag[i, h * G:(h + 1) * G] = (w[:, :, None] * vv.abs()[None]).sum(1)
            big[i, h * G:(h + 1) * G, 0] = ((qq.abs()[:, None, :] * kk.abs()[None]).sum(-1) / math.sqrt(D)).amax(1)
    return out, mag, big


def attention_tolerance(out, mag, big, L, D, weight_step):
    """Derived bound per element: the output is rounded to bf16 (half a step:
    2^-8 of it); a score is a sum of D products in fp32, off by at most
    (D + 4) 2^-24 of the sum of their sizes, which moves a weight by that
    relative to it, once in the numerator and once in the sum; the sums run
    over L weights and the exponential is good to 2^-22; and a weight is rounded
    to `weight_step` of itself before it meets V."""
    rel = 2 * (D + 4) * 2.0 ** -24 * big + 2 * (L + 64) * 2.0 ** -24 + 2.0 ** -21 + weight_step
    return 2.0 ** -8 * out.abs() + rel * mag * (1 + 2.0 ** -8) + 1e-30
