"""Timed cases of a speculative step over the 8-bit paged KV cache, and of what forks and shortens a cache.

A step that verifies a tree of drafted tokens runs these in a row: pages and slots for the drafts; queries and
keys normalised, rotated at each token's depth and stored; attention in which a drafted token sees the rows before the draft
and its own ancestors; the rows of the accepted path moved together in every layer; the pages behind them given back.
A request that is answered several times is forked: its rows are copied to the pages of the others.

The cache: pages [P, Hkv, page, D] in e4m3, and for each block of 16 rows and head a scale, a power of two. The
pools of several layers lie in one tensor here, [layers * P, ...], so that one call reads all their rows back.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

BF = torch.bfloat16
F8 = torch.float8_e4m3fn
BLOCK = 16            # rows that share a scale
E_MIN, E_MAX = -100, 119
LARGEST = 448.0       # of e4m3
EPS = 1e-6
THETA = 1e6

# (query heads, KV heads, head dim) of the attention layers
HEADS = ((16, 8, 128), (32, 8, 128), (40, 8, 128), (16, 4, 256), (32, 8, 64))
PAGES = (16, 64, 128)


def listed():
    return [
        # the drafted tree of one chat sequence: launches and latency
        {"name": "prepare_tree", "kind": "prepare", "B": 1, "T": 26, "rows": 700, "prompt": False, "Hq": 32, "Hkv": 8, "D": 128, "rot": 128, "gate": False,
         "image": False, "page": 64},
        # a chunk of prompts, ragged, with an image in each, a quarter of each head rotated, gates between the queries
        {"name": "prepare_chunk", "kind": "prepare", "B": 5, "T": 8191, "rows": 900, "prompt": True, "Hq": 16, "Hkv": 4, "D": 256, "rot": 64, "gate": True,
         "image": True, "page": 64},
        # one sequence early in its context, a short draft: launches and latency
        {"name": "tree_one", "kind": "tree", "B": 1, "n": 8, "len": 612, "Hq": 16, "Hkv": 8, "D": 128, "page": 64},
        # one sequence deep in a long context, a full tree
        {"name": "tree_one_long", "kind": "tree", "B": 1, "n": 60, "len": 32768, "Hq": 16, "Hkv": 4, "D": 256, "page": 64},
        # a served batch, ragged lengths and trees, small pages
        {"name": "tree_batch", "kind": "tree", "B": 32, "n": 26, "len": 4001, "Hq": 40, "Hkv": 8, "D": 128, "page": 16},
        # few sequences, wide trees, long contexts
        {"name": "tree_wide", "kind": "tree", "B": 8, "n": 120, "len": 16384, "Hq": 32, "Hkv": 8, "D": 128, "page": 64},
        # the accepted paths of a served batch in the attention layers of a hybrid stack
        {"name": "keep_hybrid", "kind": "keep", "B": 8, "n": 26, "len": 1000, "layers": 8, "Hkv": 4, "D": 256, "page": 64},
        # the same for many requests in every layer of a deep stack
        {"name": "keep_deep", "kind": "keep", "B": 64, "n": 60, "len": 300, "layers": 32, "Hkv": 8, "D": 128, "page": 16},
        # pages of a step: for the drafts of a batch, and back behind the accepted rows
        {"name": "pages_draft", "kind": "pages", "B": 32, "n": 26, "len": 4096, "page": 64},
        # the same for many requests of wide trees on small pages
        {"name": "pages_wave", "kind": "pages", "B": 256, "n": 60, "len": 8192, "page": 16},
        # a short prompt answered four times, one layer's copy
        {"name": "fork_short", "kind": "fork", "B": 1, "copies": 3, "len": 213, "layers": 1, "Hkv": 8, "D": 128, "page": 64},
        # long prompts answered four times, the attention layers of a hybrid stack
        {"name": "fork_long", "kind": "fork", "B": 2, "copies": 3, "len": 4001, "layers": 8, "Hkv": 4, "D": 256, "page": 64},
    ]


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 8e12, w["flops"] / 2.5e15)


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    limits = {}
    for c in listed():
        limits[c["kind"]] = max(limits.get(c["kind"], 0.0), _cost(c))
    kind = rng.choice(sorted(limits))
    while True:
        Hq, Hkv, D = rng.choice(HEADS)
        page = rng.choice(PAGES)
        if kind == "prepare":
            B = _log_int(rng, 1, 64)
            prompt = rng.random() < 0.5
            case = {"kind": kind, "B": B, "T": B + _log_int(rng, 1, 8000 if prompt else 60 * B) - 1, "rows": _log_int(rng, 1, 6000), "prompt": prompt, "Hq": Hq,
                    "Hkv": Hkv, "D": D, "rot": rng.choice((D, D // 2, D // 4)), "gate": rng.random() < 0.4, "image": prompt and rng.random() < 0.5, "page": page}
        elif kind == "tree":
            case = {"kind": kind, "B": _log_int(rng, 1, 64), "n": _log_int(rng, 1, 128), "len": _log_int(rng, 1, 32768), "Hq": Hq, "Hkv": Hkv, "D": D, "page": page}
            if case["B"] * case["n"] * case["len"] * Hq > 4e9:     # scores of the plain form, padded
                continue
        elif kind == "keep":
            case = {"kind": kind, "B": _log_int(rng, 1, 100), "n": _log_int(rng, 2, 128), "len": _log_int(rng, 1, 2000), "layers": _log_int(rng, 1, 40), "Hkv": Hkv,
                    "D": D, "page": page}
            if case["B"] * (case["len"] + 192) * case["layers"] * Hkv * D > 4e9:     # bytes of a pool
                continue
        elif kind == "pages":
            case = {"kind": kind, "B": _log_int(rng, 1, 400), "n": _log_int(rng, 1, 128), "len": _log_int(rng, 1, 16000), "page": page}
        else:
            case = {"kind": kind, "B": _log_int(rng, 1, 8), "copies": rng.randint(1, 7), "len": _log_int(rng, 1, 8000), "layers": _log_int(rng, 1, 40), "Hkv": Hkv,
                    "D": D, "page": page}
        if _cost(case) <= limits[kind]:
            return case


# ---- lengths and trees: ragged, of the case alone, so that work() counts them ------------------
def _part(b, lo=0.5):
    """1 for the first, then spread over [lo, 1]."""
    return 1.0 if b == 0 else lo + (1.0 - lo) * ((b * 0.6180339887) % 1.0)


def _ceil(a, b):
    return -(-a // b)


def _lens(case):
    """Rows of each request before its new tokens."""
    return [max(0, int(case["len"] * _part(b))) for b in range(case["B"])]


def _drafts(case):
    """Drafted tokens of each request."""
    return [max(1, int(case["n"] * _part(b, 0.3))) for b in range(case["B"])]


def _prepare_lens(case):
    """(rows already there, new rows) of each request."""
    B, T = case["B"], case["T"]
    start = [int(case["rows"] * _part(b, 0.1)) for b in range(B)]
    share = [_part(b, 0.2) for b in range(B)]
    new = [1 + int((T - B) * s / sum(share)) for s in share]
    new[-1] += T - sum(new)
    return start, new


def _parents(n, b):
    """A tree of n drafted tokens: token 0 is its root, token i hangs on one of those before it."""
    g = np.random.RandomState(1000 + b)
    return [-1] + [int(g.randint(0, i)) for i in range(1, n)]


def _depths(parents):
    d = []
    for p in parents:
        d.append(0 if p < 0 else d[p] + 1)
    return d


def _paths(parents):
    """Ancestors of each token, itself among them, in order."""
    out = []
    for i, p in enumerate(parents):
        out.append((out[p] if p >= 0 else []) + [i])
    return out


def _accepted(case):
    """The accepted path of each request: the ancestors of one of its tokens."""
    out = []
    for b, n in enumerate(_drafts(case)):
        paths = _paths(_parents(n, b))
        out.append(paths[int((b * 0.7548776662 + 0.9) % 1.0 * n)])
    return out


def _starts(new):
    s = [0]
    for n in new:
        s.append(s[-1] + n)
    return s


# ---- inputs -------------------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _exponent(amax):
    """The smallest e with amax <= 448 * 2^e, bounded: 448 = 0.875 * 2^9."""
    m, e = torch.frexp(amax)
    return (e - 9 + (m > 0.875)).where(amax > 0, torch.full_like(e, E_MIN)).clamp(E_MIN, E_MAX)


def _pow2(e):
    """2^e in f32, from its bits: a power function may be off by a rounding."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _log2(scale):
    return torch.frexp(scale)[1] - 1


def _codes(x, e):
    """x (f32) over 2^e, rounded to e4m3."""
    y = (x * _pow2(-e)).clamp(-LARGEST, LARGEST)
    return torch.where(x.isfinite(), y, torch.full_like(y, math.nan)).to(F8)


def _filled(g, P, Hkv, page, D, spread):
    """Pages of random rows and their scales; `spread`: channels differ in size, as normalised keys' do."""
    pages, scale = torch.empty((P, Hkv, page, D), dtype=F8, device="cuda"), torch.empty((P, Hkv, page // BLOCK), device="cuda")
    w = torch.exp(spread * torch.randn((Hkv, 1, 1, D), generator=g, device="cuda"))
    step = max(1, (1 << 27) // (Hkv * page * D))
    for p in range(0, P, step):
        n = min(step, P - p)
        x = torch.randn((n, Hkv, page // BLOCK, BLOCK, D), generator=g, device="cuda") * w
        # tokens differ in size, and with them the blocks' scales
        x *= torch.exp(0.7 * torch.randn((n, Hkv, page // BLOCK, BLOCK, 1), generator=g, device="cuda"))
        e = _exponent(x.abs().amax((3, 4)))
        pages[p:p + n] = _codes(x, e[..., None, None]).view(n, Hkv, page, D)
        scale[p:p + n] = _pow2(e)
    return pages, scale


def _table(seed, rows, page, spare=3):
    """Pages of each request's rows, in shuffled order; -1 behind them. Returns the table, the pool's size and the pages left over."""
    held = [_ceil(r, page) for r in rows]
    mp, P = max(1, max(held)), sum(held) + spare
    g = torch.Generator()
    g.manual_seed(int(seed) + 5)
    order, table, at = torch.randperm(P, generator=g).to(torch.int32), torch.full((len(rows), mp), -1, dtype=torch.int32), 0
    for b, n in enumerate(held):
        table[b, :n] = order[at:at + n]
        at += n
    return table, P, order[at:]


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _slots(table, page, rows):
    """Slots of rows [from, to) of each request, one after the other."""
    t = table.cpu().numpy()
    out = []
    for b, (a, z) in enumerate(rows):
        r = np.arange(a, z)
        out.append(t[b, r // page].astype(np.int64) * page + r % page)
    return np.concatenate(out) if out else np.zeros(0, np.int64)


def _read(s, slots):
    """Read-back of the slots in every layer of the joined pools."""
    P, layers = s["P"], s["layers"]
    all_slots = (np.arange(layers)[:, None] * (P * s["case"]["page"]) + slots[None]).reshape(-1)
    s["read"] = torch.tensor(all_slots, dtype=torch.int32, device="cuda")
    _, Hkv, _, D = s["kp"].shape
    s["k_out"], s["v_out"] = (torch.empty((len(all_slots), Hkv, D), dtype=BF, device="cuda") for _ in range(2))


def _pools(s, g, P, layers, case):
    Hkv, D, page = case["Hkv"], case["D"], case["page"]
    s["P"], s["layers"] = P, layers
    s["kp"], s["ks"] = _filled(g, P * layers, Hkv, page, D, 0.4)
    s["vp"], s["vs"] = _filled(g, P * layers, Hkv, page, D, 0.0)
    s["caches"] = [tuple(x[i * P:(i + 1) * P] for x in (s["kp"], s["vp"], s["ks"], s["vs"])) for i in range(layers)]


def _first_moved(path):
    """The first kept row that does not stay where it is."""
    return next((i for i, k in enumerate(path) if k != i), len(path))


def prepare(case, seed):
    kind, g, s = case["kind"], _gen(seed), {"case": dict(case)}
    page = case["page"]
    if kind == "pages":
        cached, new = _lens(case), _drafts(case)
        table, P, _ = _table(seed, cached, page, 0)
        more = sum(_ceil(c + n, page) - _ceil(c, page) for c, n in zip(cached, new)) + 7
        mp = max(_ceil(c + n, page) for c, n in zip(cached, new))
        s["table"] = torch.full((case["B"], mp), -1, dtype=torch.int32, device="cuda")
        s["table"][:, :table.shape[1]] = table[:, :mp].cuda()
        s["free"] = torch.full((P + more,), -1, dtype=torch.int32, device="cuda")
        s["free"][:more] = P + torch.randperm(more, generator=g, device="cuda").to(torch.int32)
        s["count"] = _ints([more])
        s["cached"], s["new"] = _ints(cached), _ints(new)
        s["kept"] = _ints([c + len(p) for c, p in zip(cached, _accepted(case))])
        s["slots"] = torch.zeros(sum(new) + 5, dtype=torch.int32, device="cuda")
        s["starts"], s["lens"] = torch.empty(case["B"] + 1, dtype=torch.int32, device="cuda"), torch.empty(case["B"], dtype=torch.int32, device="cuda")
        return s
    Hkv, D = case["Hkv"], case["D"]
    if kind == "fork":
        B, copies, lens = case["B"], case["copies"], [max(1, n) for n in _lens(case)]
        table, P, _ = _table(seed, [n for n in lens for _ in range(copies + 1)], page)     # request b, then its copies
        _pools(s, g, P, case["layers"], case)
        s["table"] = table.cuda()
        pairs = [(b * (copies + 1), b * (copies + 1) + i) for b in range(B) for i in range(1, copies + 1)]
        s["src"], s["dst"], s["len"] = _ints([a for a, _ in pairs]), _ints([z for _, z in pairs]), _ints([lens[b] for b in range(B) for _ in range(copies)])
        s["max_len"] = max(lens)
        _read(s, _slots(table, page, [(0, lens[i // (copies + 1)]) if i % (copies + 1) else (0, 0) for i in range(B * (copies + 1))]))
        return s
    if kind == "keep":
        cached, new, paths = _lens(case), _drafts(case), _accepted(case)
        table, P, _ = _table(seed, [c + n for c, n in zip(cached, new)], page)
        _pools(s, g, P, case["layers"], case)
        s["table"], s["cached"] = table.cuda(), _ints(cached)
        most = max(len(p) for p in paths)
        s["kept"], s["kept_lens"] = _ints([p + [-1] * (most - len(p)) for p in paths]), _ints([len(p) for p in paths])
        s["lens"] = torch.empty(case["B"], dtype=torch.int32, device="cuda")
        # read back: the accepted rows and those before them in their first block
        _read(s, _slots(table, page, [(c // BLOCK * BLOCK, c + len(p)) for c, p in zip(cached, paths)]))
        return s
    Hq = case["Hq"]
    if kind == "prepare":
        start, new = _prepare_lens(case)
    else:
        start, new = _lens(case), _drafts(case)
    rows, T = [a + n for a, n in zip(start, new)], sum(new)
    table, P, _ = _table(seed, rows, page)
    _pools(s, g, P, 1, case)
    s["table"], s["lens"], s["max_len"], s["starts"] = table.cuda(), _ints(rows), max(rows), _ints(_starts(new))
    if kind == "prepare":
        # q, k and v are views of one fused projection's rows
        wide = 2 if case["gate"] else 1
        x = torch.randn((T, (wide * Hq + 2 * Hkv) * D), generator=g, device="cuda")
        x *= torch.exp(0.5 * torch.randn((T, 1), generator=g, device="cuda"))
        x = x.to(BF)
        s["q"] = x[:, :wide * Hq * D].view(T, Hq, wide * D)[..., :D]
        s["k"], s["v"] = (x[:, (wide * Hq + i * Hkv) * D:(wide * Hq + (i + 1) * Hkv) * D].view(T, Hkv, D) for i in range(2))
        s["q_norm"], s["k_norm"] = ((1.0 + 0.2 * torch.randn(D, generator=g, device="cuda")).to(BF) for _ in range(2))
        pos = []
        for b, (a, n) in enumerate(zip(start, new)):
            pos += list(range(a, a + n)) if case["prompt"] else [a + d for d in _depths(_parents(n, b))]
        s["pos"], s["sections"] = _ints(pos), None
        if case["image"]:
            # an image in the middle of each prompt: one time, its rows and columns
            pos = np.array([pos] * 3)
            for a, n, at in zip(start, new, _starts(new)):
                side = int(math.sqrt(n / 2))
                i = np.arange(side * side)
                pos[:, at + n // 4:at + n // 4 + side * side] = a + n // 4 + np.stack([0 * i, i // max(1, side), i % max(1, side)])
            s["pos"] = torch.tensor(pos, dtype=torch.int32, device="cuda")
            pairs = case["rot"] // 2
            s["sections"] = (pairs - 2 * (pairs // 3), pairs // 3, pairs // 3)
        s["slots"] = torch.tensor(_slots(table, page, list(zip(start, rows))), dtype=torch.int32, device="cuda")
        s["q_out"] = torch.empty((T, Hq, D), dtype=BF, device="cuda")
        _read(s, _slots(table, page, [(a // BLOCK * BLOCK, r) for a, r in zip(start, rows)]))
        return s
    q = torch.randn((T, Hq, D), generator=g, device="cuda") * 1.2
    s["q"], s["out"] = q.to(BF), torch.zeros((T, Hq, D), dtype=BF, device="cuda")
    words = _ceil(max(new), 64)
    mask = np.zeros((T, words * 64), dtype=np.uint8)
    at = 0
    for b, n in enumerate(new):
        for i, path in enumerate(_paths(_parents(n, b))):
            mask[at + i, path] = 1
        at += n
    s["mask"] = torch.from_numpy(np.packbits(mask, axis=1, bitorder="little").view(np.int64).copy()).cuda()
    s["n"] = max(new)
    return s


# ---- the plain forms ----------------------------------------------------------------------------
def _plain_reserve(s):
    page, table, free, count = s["case"]["page"], s["table"], s["free"], s["count"]
    B, mp = table.shape
    c, n = s["cached"].long(), s["new"].long()
    starts = torch.cat([n[:1] * 0, n.cumsum(0)])
    p = torch.arange(mp, device=table.device)
    fits = c + n <= mp * page
    holes = (p >= (c // page)[:, None]) & (p < ((c + n + page - 1) // page)[:, None]) & (table < 0) & fits[:, None]
    need = holes.sum(1)
    ok = fits & (starts[1:] <= s["slots"].numel()) & ((need == 0) | (need.cumsum(0) <= count))
    take = holes & ok[:, None]
    k = (count - take.view(-1).cumsum(0)).clamp(min=0)
    table.copy_(torch.where(take, free[k].view(B, mp), table))
    count -= take.sum()
    t = torch.arange(s["slots"].numel(), device=table.device)
    b = torch.searchsorted(starts[1:].contiguous(), t, right=True)
    inside = b < B
    b = b.clamp(max=B - 1)
    row = (c[b] + t - starts[b]).clamp(0, mp * page - 1)
    s["slots"].copy_(torch.where(inside & ok[b], table[b, row // page].long() * page + row % page, -1))
    s["starts"].copy_(starts)
    s["lens"].copy_(torch.where(ok, c + n, 0))


def _plain_trim(s):
    page, table, free, count, lens = s["case"]["page"], s["table"], s["free"], s["count"], s["kept"].long()
    P, p = free.numel(), torch.arange(table.shape[1], device=table.device)
    give = (p >= ((lens + page - 1) // page)[:, None]) & (lens >= 0)[:, None] & (table >= 0)
    at = count + give.view(-1).cumsum(0) - 1
    at = torch.where(give.view(-1) & (at < P), at, P)
    free.copy_(torch.cat([free, free[:1]]).scatter(0, at, table.view(-1))[:P])
    count += give.sum()
    count.clamp_(max=P)
    table.masked_fill_(give, -1)


def _pages_out(s):
    return {k: s[k] for k in ("table", "free", "count", "starts", "lens", "slots")}


def _plain_store(pages, scale, x, slots):
    """x [T, Hkv, D] in f32 into the rows `slots`: blocks whose scale grows are rescaled."""
    P, H, page, D = pages.shape
    slot = slots.long()
    pg, blk, row = slot // page, slot % page // BLOCK, slot % BLOCK
    fine = torch.where(x.isfinite(), x.abs(), 0.0).amax(2)                                                  # [T, H]
    ids = slot // BLOCK
    amax = torch.zeros((P * (page // BLOCK), H), device=x.device).index_reduce(0, ids, fine, "amax")[ids]
    first = torch.full((P * (page // BLOCK),), BLOCK, device=x.device, dtype=torch.long).index_reduce(0, ids, row, "amin")[ids]
    old = _log2(scale[pg, :, blk])
    e = _exponent(amax)
    e = torch.where((first == 0)[:, None], e, torch.maximum(e, old))
    # the block's earlier rows at the new scale; its other rows as they are
    view = pages.view(P, H, page // BLOCK, BLOCK, D)
    held = view.view(torch.uint8)[pg, :, blk]                                                               # [T, H, 16, D]
    value = held.view(F8).float() * _pow2(old)[..., None, None]
    before = (torch.arange(BLOCK, device=x.device) < first[:, None])[:, None, :, None] & (e > old)[..., None, None]
    view.view(torch.uint8)[pg, :, blk] = torch.where(before, _codes(value, e[..., None, None]).view(torch.uint8), held)
    scale[pg, :, blk] = _pow2(e)
    view.view(torch.uint8)[pg, :, blk, row] = _codes(x, e[..., None]).view(torch.uint8)


def _plain_rows(pages, scale, slots):
    """Rows by slot, in f32."""
    page = pages.shape[2]
    slot = slots.long()
    return pages.view(torch.uint8)[slot // page, :, slot % page].view(F8).float() * scale[slot // page, :, slot % page // BLOCK][..., None]


def _plain_read(s):
    s["k_out"].copy_(_plain_rows(s["kp"], s["ks"], s["read"]))
    s["v_out"].copy_(_plain_rows(s["vp"], s["vs"], s["read"]))
    return s["k_out"], s["v_out"]


def _plain_norm_rotate(x, w, cos, sin, rot):
    """Heads of x [T, H, D] normalised and their first `rot` dims rotated, in f32."""
    x = x.float()
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
    a, b = x[..., :rot // 2], x[..., rot // 2:rot]
    return torch.cat([a * cos - b * sin, a * sin + b * cos, x[..., rot:]], -1)


def _plain_prepare(s):
    rot, pos = s["case"]["rot"], s["pos"]
    j = torch.arange(rot // 2, device=pos.device)
    if s["sections"] is not None:     # pair j turns with one of the three positions
        stream = torch.where((j % 3 == 1) & (j // 3 < s["sections"][1]), 1, torch.where((j % 3 == 2) & (j // 3 < s["sections"][2]), 2, 0))
        pos = pos[stream].t()
    else:
        pos = pos[:, None]
    angle = pos.double() * torch.exp(j.double() * (-2.0 / rot * math.log(THETA)))
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    s["q_out"].copy_(_plain_norm_rotate(s["q"], s["q_norm"], cos, sin, rot))
    _plain_store(s["kp"], s["ks"], _plain_norm_rotate(s["k"], s["k_norm"], cos, sin, rot), s["slots"])
    _plain_store(s["vp"], s["vs"], s["v"].float(), s["slots"])
    return s["q_out"], _plain_read(s)


def _plain_cache(pages, scale, table):
    """[B, Hkv, rows, D] in f32: the pages of each request, as the values they stand for."""
    B, mp = table.shape
    P, H, page, D = pages.shape
    t = table.long().clamp(min=0)
    x = pages.view(torch.uint8)[t].view(F8).float().view(B, mp, H, page // BLOCK, BLOCK, D) * scale[t][..., None, None]
    return x.transpose(1, 2).reshape(B, H, mp * page, D)


def _plain_tree(s):
    k, v, q = _plain_cache(s["kp"], s["ks"], s["table"]), _plain_cache(s["vp"], s["vs"], s["table"]), s["q"]
    (B, H, L, D), Hq, N = k.shape, q.shape[1], s["n"]
    G = Hq // H
    start, new = s["starts"][:-1].long(), (s["starts"][1:] - s["starts"][:-1]).long()
    i = torch.arange(N, device=k.device)
    there = i < new[:, None]                                                                                # [B, N]
    tok = (start[:, None] + i).clamp(max=q.shape[0] - 1)
    # row r of the cache is drafted token r - (rows - new) of its request
    bits = s["mask"][tok].view(B, N, -1, 1) >> torch.arange(64, device=k.device) & 1                        # [B, N, words, 64]
    before = (s["lens"].long() - new)[:, None]
    r = torch.arange(L, device=k.device)
    drafted = (r - before).clamp(0, bits.shape[2] * 64 - 1)                                                 # [B, L]
    seen = bits.view(B, N, -1).gather(2, drafted[:, None].expand(B, N, L)) != 0
    valid = ((r < before)[:, None] | seen & (r < s["lens"].long()[:, None])[:, None]) & there[..., None]
    x = q.float()[tok].view(B, N, H, G, D).permute(0, 2, 3, 1, 4).reshape(B * H, G * N, D) * (1.0 / math.sqrt(D))
    w = torch.bmm(x, k.reshape(B * H, L, D).transpose(1, 2).contiguous()).view(B, H, G, N, L)
    w.masked_fill_(~valid[:, None, None], -math.inf)
    m = w.amax(-1, keepdim=True)
    w.sub_(m.masked_fill(m == -math.inf, 0.0)).exp_()
    total = w.sum(-1, keepdim=True).clamp(min=1e-38)
    o = torch.bmm(w.view(B * H, G * N, L), v.reshape(B * H, L, D).contiguous()).view(B, H, G, N, D) / total
    s["out"][tok[there]] = o.permute(0, 3, 1, 2, 4).reshape(B, N, Hq, D)[there].to(BF)
    return s["out"]


def _plain_moved(pages, scale, table, cached, kept, there, moves):
    """One of K and V, all layers at once: pages [layers, P, H, page, D]. The kept rows go to the front of the draft; a block's scale becomes the
    largest of those that its rows come from."""
    N, P, H, page, D = pages.shape
    B, M = kept.shape
    blocks, scales = pages.view(torch.uint8).view(N, P, H, page // BLOCK, BLOCK, D), scale.view(N, P, H, page // BLOCK)
    b = torch.arange(B, device=kept.device)[:, None]
    from_row, to_row = cached[:, None] + kept.clamp(min=0), cached[:, None] + torch.arange(M, device=kept.device)

    def place(row):
        row = row.clamp(max=table.shape[1] * page - 1)
        return table[b, row // page].long().clamp(min=0), row % page // BLOCK, row % BLOCK

    sp, sb, sr = place(from_row)
    dp, db, dr = place(to_row)
    code = blocks[:, sp, :, sb, sr]                                                                         # [B, M, N, H, D]
    e_from = _log2(scales[:, sp, :, sb])                                                                    # [B, M, N, H]
    e_held = _log2(scales[:, dp, :, db])
    # rows of a block that stay: those before the first moved row in it
    nb = M // BLOCK + 2                                                                                     # blocks that a draft may touch
    at = to_row // BLOCK - (cached // BLOCK)[:, None]
    ids = torch.where(moves, b * nb + at, B * nb).view(-1)
    first = torch.full((B * nb + 1,), BLOCK, device=kept.device, dtype=torch.long).index_reduce(0, ids, dr.reshape(-1), "amin")[ids].view(B, M)
    top = torch.full((B * nb + 1, N, H), E_MIN, device=kept.device, dtype=torch.int32).index_reduce(
        0, ids, e_from.reshape(B * M, N, H).to(torch.int32), "amax")[ids].view(B, M, N, H)
    e = torch.where((first > 0)[..., None, None], torch.maximum(top, e_held), top)
    held = blocks[:, dp, :, db]                                                                             # [B, M, N, H, 16, D]
    stays = (torch.arange(BLOCK, device=kept.device) < first[..., None])[:, :, None, None, :, None]
    again = _codes(held.view(F8).float() * _pow2(e_held)[..., None, None], e[..., None, None]).view(torch.uint8)
    held = torch.where(stays & (e > e_held)[..., None, None], again, held)
    moved = _codes(code.view(F8).float() * _pow2(e_from)[..., None], e[..., None]).view(torch.uint8)
    i, j = moves.nonzero(as_tuple=True)
    blocks[:, dp[i, j], :, db[i, j]] = held[i, j]
    scales[:, dp[i, j], :, db[i, j]] = _pow2(e)[i, j]
    blocks[:, dp[i, j], :, db[i, j], dr[i, j]] = moved[i, j]


def _plain_keep(s):
    cached, kept, n = s["cached"].long(), s["kept"].long(), s["kept_lens"].long()
    i = torch.arange(kept.shape[1], device=kept.device)
    there = i < n[:, None]
    moves = there & ((kept != i) & there).cummax(1)[0]      # from the first row that does not stay where it is
    shape = (s["layers"], s["P"], *s["kp"].shape[1:])
    _plain_moved(s["kp"].view(shape), s["ks"], s["table"], cached, kept, there, moves)
    _plain_moved(s["vp"].view(shape), s["vs"], s["table"], cached, kept, there, moves)
    s["lens"].copy_(cached + n)
    return s["lens"], _plain_read(s)


def _plain_copied(pages, scale, P, src, dst, blocks):
    """Blocks [0, blocks) of each pair, in all layers."""
    H, page, D = pages.shape[1:]
    nb = page // BLOCK
    view, scales = pages.view(torch.uint8).view(-1, P, H, nb, BLOCK, D), scale.view(-1, P, H, nb)
    x = torch.arange(src.shape[1] * nb, device=src.device)
    pair, x = (x < blocks[:, None]).nonzero(as_tuple=True)
    a, z = src[pair, x // nb].long(), dst[pair, x // nb].long()
    view[:, z, :, x % nb] = view[:, a, :, x % nb]
    scales[:, z, :, x % nb] = scales[:, a, :, x % nb]


def _plain_fork(s):
    src, dst, blocks = s["table"][s["src"].long()], s["table"][s["dst"].long()], (s["len"] + BLOCK - 1) // BLOCK
    _plain_copied(s["kp"], s["ks"], s["P"], src, dst, blocks)
    _plain_copied(s["vp"], s["vs"], s["P"], src, dst, blocks)
    return _plain_read(s)


def run(s):
    kind = s["case"]["kind"]
    if own:
        import aila_amd as A
        page = s["case"]["page"]
        if kind == "pages":
            A.kv_pages_reserve(s["cached"], s["new"], s["table"], s["free"], s["count"], page, s["slots"], s["starts"], s["lens"])
            A.kv_pages_trim(s["kept"], s["table"], s["free"], s["count"], page)
            return _pages_out(s)
        cache = (s["kp"], s["vp"], s["ks"], s["vs"])
        if kind == "prepare":
            A.prepare_qkv_paged_fp8(s["q"], s["k"], s["v"], *cache, s["slots"], s["pos"], q_norm=s["q_norm"], k_norm=s["k_norm"], rotary_dim=s["case"]["rot"],
                                    theta=THETA, eps=EPS, sections=s["sections"], q_out=s["q_out"])
            return s["q_out"], A.kv_read_paged_fp8(*cache, s["read"], s["k_out"], s["v_out"])
        if kind == "keep":
            A.kv_keep_paged_fp8(s["caches"], s["table"], s["cached"], s["kept"], s["kept_lens"], lens=s["lens"])
            return s["lens"], A.kv_read_paged_fp8(*cache, s["read"], s["k_out"], s["v_out"])
        if kind == "fork":
            A.kv_copy_paged_fp8(s["caches"], s["table"], s["src"], s["dst"], s["len"], s["max_len"])
            return A.kv_read_paged_fp8(*cache, s["read"], s["k_out"], s["v_out"])
        if "ws" not in s:      # the workspace that a program keeps for its calls of this size
            T, Hq, D = s["q"].shape
            size = A.gqa_tree_paged_fp8_workspace_size(T, s["case"]["B"], Hq, s["kp"].shape[1], D, s["max_len"], s["mask"].shape[1])
            s["ws"] = torch.empty(size, dtype=torch.uint8, device="cuda")
        return A.gqa_tree_paged_fp8(s["q"], *cache, s["table"], s["starts"], s["lens"], s["mask"], s["max_len"], out=s["out"], workspace=s["ws"])
    if kind == "pages":
        _plain_reserve(s)
        _plain_trim(s)
        return _pages_out(s)
    if kind == "prepare":
        return _plain_prepare(s)
    if kind == "keep":
        return _plain_keep(s)
    if kind == "fork":
        return _plain_fork(s)
    return _plain_tree(s)


def work(case):
    page = case["page"]
    if case["kind"] == "pages":
        cached, new = _lens(case), _drafts(case)
        moved = sum(2 * _ceil(c + n, page) - _ceil(c, page) - _ceil(c + len(p), page) for c, n, p in zip(cached, new, _accepted(case)))
        # lengths in, starts and lengths out, slots out, the pages taken and given back: table and free list
        return {"bytes": 4.0 * (5 * case["B"] + sum(new) + 2 * moved), "flops": 0.0}
    Hkv, D = case["Hkv"], case["D"]
    row, back = Hkv * (D + 4 / BLOCK) * 2, Hkv * D * 4            # a row of the cache, K and V; read back
    if case["kind"] == "fork":
        rows = sum(max(1, n) for n in _lens(case)) * case["copies"] * case["layers"]
        once = sum(max(1, n) for n in _lens(case)) * case["layers"]
        return {"bytes": once * row + rows * row + rows * (row + back), "flops": 0.0}
    if case["kind"] == "keep":
        cached, paths = _lens(case), _accepted(case)
        moved = sum(len(p) - _first_moved(p) for p in paths)
        read = sum(c % BLOCK + len(p) for c, p in zip(cached, paths))
        return {"bytes": case["layers"] * (moved * 2 * row + read * (row + back)) + 4.0 * (3 * case["B"] + sum(len(p) for p in paths)), "flops": 0.0}
    Hq = case["Hq"]
    if case["kind"] == "prepare":
        start, new = _prepare_lens(case)
        T, R = case["T"], sum(a % BLOCK + n for a, n in zip(start, new))
        return {"bytes": T * (Hq * D * 4 + Hkv * D * 4 + row + 8) + R * (row + back), "flops": 0.0}
    start, new = _lens(case), _drafts(case)
    pairs = sum(n * a + sum(d + 1 for d in _depths(_parents(n, b))) for b, (a, n) in enumerate(zip(start, new)))
    return {"bytes": sum(a + n for a, n in zip(start, new)) * row + sum(new) * (Hq * D * 4 + 8 * _ceil(max(new), 64)), "flops": 4.0 * pairs * Hq * D}


# ---- the definitions in 64 bits -----------------------------------------------------------------
def _step64(x):
    """Nearest e4m3 value of x (float64), ties to even."""
    a = np.abs(x)
    unit = np.exp2(np.maximum(np.floor(np.log2(np.where(a > 0, a, 1.0))), -6.0) - 3.0)
    return np.where(np.isfinite(x), np.clip(np.rint(x / unit) * unit, -LARGEST, LARGEST), np.nan)


def _block64(pages, scale, blocks):
    """Values [n, H, 16, D] and scales [n, H] of blocks (page * blocks of a page + block) in float64."""
    P, H, page, D = pages.shape
    nb = page // BLOCK
    at = torch.tensor(blocks, device=pages.device, dtype=torch.long)
    code = pages.view(torch.uint8).view(P, H, nb, BLOCK, D)[at // nb, :, at % nb].view(F8)
    old = scale[at // nb, :, at % nb].double().cpu().numpy()
    return code.float().double().cpu().numpy() * old[..., None, None], old


def _exact_rows(pages, scale, x, slots, read):
    """The rows `read` after x [T, H, D] (float64) went to `slots`, block by block of 16 rows."""
    slots, read = slots.tolist(), read.tolist()
    blocks = sorted({r // BLOCK for r in read} | {r // BLOCK for r in slots})
    value, old = _block64(pages, scale, blocks)
    where = {blk: i for i, blk in enumerate(blocks)}
    runs = {}
    for t, r in enumerate(slots):
        runs.setdefault(r // BLOCK, []).append(t)
    for blk, toks in runs.items():
        i, rows = where[blk], [slots[t] % BLOCK for t in toks]
        fresh = x[toks].transpose(1, 0, 2)                                                                  # [H, n, D]
        top = np.abs(fresh).max((1, 2))
        e = np.clip(np.ceil(np.log2(np.where(top > 0, top, 1e-300) / LARGEST)), E_MIN, E_MAX)
        s = np.exp2(e) if min(rows) == 0 else np.maximum(np.exp2(e), old[i])
        s = s[:, None, None]
        value[i][:, :min(rows)] = _step64(value[i][:, :min(rows)] / s) * s
        value[i][:, rows] = _step64(fresh / s) * s
    return np.stack([value[where[r // BLOCK]][:, r % BLOCK] for r in read])


def _exact_heads(x, w, turn, rot):
    """x [T, H, D], each head over its root mean square times w; pairs (d, d + rot / 2) as complex numbers times turn [T, rot / 2]."""
    x = x.double().cpu().numpy()
    x = x * w.double().cpu().numpy() / np.sqrt(np.square(x).sum(-1, keepdims=True) / x.shape[-1] + EPS)
    z = (x[..., :rot // 2] + 1j * x[..., rot // 2:rot]) * turn[:, None]
    x[..., :rot // 2], x[..., rot // 2:rot] = z.real, z.imag
    return x


def _exact_tree(q, kp, ks, vp, vs, table, before, paths):
    """q [n, Hq, D] of one request whose token i sees rows [0, before) and the drafted tokens paths[i]; in float64."""
    n, Hq, D = q.shape
    P, H, page, _ = kp.shape
    rows = before + n
    ids = table[:_ceil(rows, page)].long()

    def whole(pages, scale):
        x = pages.view(torch.uint8)[ids].view(F8).double() * scale[ids].double().repeat_interleave(BLOCK, 2)[..., None]
        return x.permute(1, 0, 2, 3).reshape(H, -1, D)[:, :rows].contiguous()

    k, v = whole(kp, ks), whole(vp, vs)
    seen = torch.zeros((n, rows), dtype=torch.bool)
    seen[:, :before] = True
    for i, path in enumerate(paths):
        seen[i, [before + j for j in path]] = True
    x = q.double().view(n, H, Hq // H, D).permute(1, 0, 2, 3).reshape(H, -1, D).contiguous()
    a = (torch.bmm(x, k.transpose(1, 2).contiguous()) / math.sqrt(D)).view(H, n, Hq // H, rows)
    a = torch.softmax(a.masked_fill(~seen.to(q.device)[None, :, None], -math.inf), -1).view(H, -1, rows)
    return torch.bmm(a, v).view(H, n, Hq // H, D).permute(1, 0, 2, 3).reshape(n, Hq, D)


def _exact_kept(pages, scale, s, layer, paths, cached):
    """Rows of one layer after each request's path moved to the front of its draft: (first block's beginning, new end)."""
    P, H, page, D = pages.shape
    table, out = s["table"].cpu().numpy(), []
    block = lambda b, row: int(table[b, row // page]) * (page // BLOCK) + row % page // BLOCK      # noqa: E731
    for b, (c, path) in enumerate(zip(cached, paths)):
        first, end = c // BLOCK * BLOCK, c + len(path)
        src = [r if r < c else c + path[r - c] for r in range(first, end)]
        need = sorted({r // BLOCK * BLOCK for r in src} | set(range(first, end, BLOCK)))
        value, sc = _block64(pages, scale, [block(b, r) for r in need])
        where = {r: i for i, r in enumerate(need)}
        moved = next((c + i for i, k in enumerate(path) if k != i), end)           # rows before it stay
        for at in range(first, end, BLOCK):
            rows = list(range(at, min(end, at + BLOCK)))
            got = np.stack([value[where[src[r - first] // BLOCK * BLOCK]][:, src[r - first] % BLOCK] for r in rows], 1)     # [H, n, D]
            if rows[-1] >= moved:
                es = np.stack([sc[where[(src[r - first] if r >= moved else at) // BLOCK * BLOCK]] for r in rows], 1).max(1)   # [H]
                got = _step64(got / es[:, None, None]) * es[:, None, None]
            out.append(got.transpose(1, 0, 2))
    return np.concatenate(out)


def exact(case, seed):
    kind = case["kind"]
    if kind == "pages":
        return None
    s = prepare(case, seed)
    if kind == "fork":
        # each copied row is the one of the table row that it was copied from
        page, lens, table = case["page"], [max(1, n) for n in _lens(case)], s["table"].cpu().numpy()
        copies, slots = case["copies"], []
        for b, n in enumerate(lens):
            r = np.arange(n)
            slots += [table[b * (copies + 1), r // page].astype(np.int64) * page + r % page] * copies
        slots, out = torch.from_numpy(np.concatenate(slots)).cuda(), []
        for i in (0, 1):
            out.append(torch.cat([c[i].view(torch.uint8)[slots // page, :, slots % page].view(F8).double()
                                  * c[i + 2].double()[slots // page, :, slots % page // BLOCK][..., None] for c in s["caches"]]))
        return tuple(out)
    if kind == "prepare":
        rot = case["rot"]
        pos = s["pos"].double().cpu().numpy()
        if case["image"]:
            by = [1 if j % 3 == 1 and j // 3 < s["sections"][1] else 2 if j % 3 == 2 and j // 3 < s["sections"][2] else 0 for j in range(rot // 2)]
            pos = np.stack([pos[i] for i in by], 1)
        else:
            pos = pos[:, None]
        turn = np.exp(1j * pos * THETA ** (-2.0 * np.arange(rot // 2) / rot))
        k, v = _exact_heads(s["k"], s["k_norm"], turn, rot), s["v"].double().cpu().numpy()
        return _exact_heads(s["q"], s["q_norm"], turn, rot), (_exact_rows(s["kp"], s["ks"], k, s["slots"], s["read"]),
                                                              _exact_rows(s["vp"], s["vs"], v, s["slots"], s["read"]))
    if kind == "keep":
        if case["layers"] * case["B"] > 2500:      # block by block on the host: too slow for more
            return None
        paths, cached = _accepted(case), _lens(case)
        both = [[_exact_kept(c[i], c[i + 2], s, layer, paths, cached) for layer, c in enumerate(s["caches"])] for i in range(2)]
        return None, (np.concatenate(both[0]), np.concatenate(both[1]))
    out, at = s["out"].double(), 0
    for b, (before, n) in enumerate(zip(_lens(case), _drafts(case))):
        out[at:at + n] = _exact_tree(s["q"][at:at + n], s["kp"], s["ks"], s["vp"], s["vs"], s["table"][b], before, _paths(_parents(n, b)))
        at += n
    return out
