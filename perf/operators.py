"""Timed cases of the 8-bit paged KV cache: its page tables, its rows, the attention that reads it.

A serving step runs these in a row: request lengths become page tables and slots, new K/V rows are quantised
into the pages, and attention reads them. Each case is one such call with the sizes an engine sends: one
sequence and a batch, contexts from some hundred rows to 32k, prompts from a turn to 8k, ragged lengths.

The cache: pages [P, Hkv, page, D] in e4m3, and for each block of 16 rows and head a scale, a power of two.
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

# (query heads, KV heads, head dim) of the attention layers
HEADS = ((16, 8, 128), (32, 8, 128), (40, 8, 128), (16, 4, 256), (32, 8, 64))
PAGES = (16, 64, 128)


def listed():
    return [
        # a decode step of a served batch in which one request ended and a new prompt took its row
        {"name": "pages_step", "kind": "pages", "B": 32, "page": 64, "rows": 4096, "ended": 1, "prompt": 213, "tight": False},
        # many requests on small pages, a wave of them replaced by new prompts, more than the batch holds
        {"name": "pages_wave", "kind": "pages", "B": 256, "page": 16, "rows": 8192, "ended": 32, "prompt": 1024, "tight": True},
        # the rows of one decode step, each in its own request's last block, and their read-back with that block
        {"name": "append_step", "kind": "append", "B": 32, "T": 32, "rows": 4001, "Hq": 32, "Hkv": 8, "D": 128, "page": 64},
        # the rows of a chunk of prompts, ragged
        {"name": "append_chunk", "kind": "append", "B": 5, "T": 8191, "rows": 900, "Hq": 16, "Hkv": 4, "D": 256, "page": 64},
        # one chat sequence early in its context: launches and latency
        {"name": "decode_one", "kind": "decode", "B": 1, "Hq": 16, "Hkv": 8, "D": 128, "len": 612, "page": 64},
        # one sequence deep in a long context
        {"name": "decode_one_long", "kind": "decode", "B": 1, "Hq": 16, "Hkv": 4, "D": 256, "len": 32768, "page": 64},
        # a served batch at long context, every sequence at its own length
        {"name": "decode_batch_long", "kind": "decode", "B": 8, "Hq": 16, "Hkv": 4, "D": 256, "len": 32768, "page": 64},
        # continuous batching: many sequences of ordinary, ragged lengths on small pages
        {"name": "decode_batch", "kind": "decode", "B": 64, "Hq": 40, "Hkv": 8, "D": 128, "len": 4001, "page": 16},
        # the next turn of a conversation: a short input over a cached prefix
        {"name": "prefill_turn", "kind": "prefill", "B": 1, "prompts": 1, "S": 250, "start": 7900, "Hq": 16, "Hkv": 4, "D": 256, "page": 64},
        # an ordinary prompt
        {"name": "prefill_2k", "kind": "prefill", "B": 1, "prompts": 1, "S": 2048, "start": 0, "Hq": 32, "Hkv": 8, "D": 128, "page": 64},
        # a long prompt
        {"name": "prefill_8k", "kind": "prefill", "B": 1, "prompts": 1, "S": 8191, "start": 0, "Hq": 16, "Hkv": 4, "D": 256, "page": 64},
        # a mixed step: chunks of three prompts beside the single tokens of 29 running requests, in a padded batch
        {"name": "prefill_mixed", "kind": "prefill", "B": 32, "prompts": 3, "S": 600, "start": 3000, "Hq": 40, "Hkv": 8, "D": 128, "page": 16},
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
        if kind == "pages":
            B = _log_int(rng, 1, 400)
            case = {"kind": kind, "B": B, "page": page, "rows": _log_int(rng, 100, 16000), "ended": rng.randint(0, max(1, B // 4)),
                    "prompt": _log_int(rng, 1, 2000), "tight": rng.random() < 0.3}
        elif kind == "append":
            B = _log_int(rng, 1, 64)
            case = {"kind": kind, "B": B, "T": B if rng.random() < 0.4 else B + _log_int(rng, 1, 8000), "rows": _log_int(rng, 1, 6000), "Hq": Hq, "Hkv": Hkv,
                    "D": D, "page": page}
        elif kind == "decode":
            case = {"kind": kind, "B": _log_int(rng, 1, 100), "Hq": Hq, "Hkv": Hkv, "D": D, "len": _log_int(rng, 1, 32768), "page": page}
        else:
            B = _log_int(rng, 1, 40)
            case = {"kind": kind, "B": B, "prompts": rng.randint(1, min(B, 4)), "S": _log_int(rng, 2, 8191), "start": _log_int(rng, 1, 16000) - 1, "Hq": Hq,
                    "Hkv": Hkv, "D": D, "page": page}
            if B * case["S"] * Hq * (case["S"] + case["start"]) > 4e9:   # scores of the plain form, padded
                continue
        if _cost(case) <= limits[kind]:
            return case


# ---- lengths: ragged, of the case alone, so that work() counts them -----------------------------
def _part(b, lo=0.5):
    """1 for the first, then spread over [lo, 1]."""
    return 1.0 if b == 0 else lo + (1.0 - lo) * ((b * 0.6180339887) % 1.0)


def _page_lens(case):
    """(cached rows, new rows, whether the row's former request ended) of each request."""
    B, ended = case["B"], case["ended"]
    gone = [False] * B
    for i in range(ended):
        gone[(i * B) // max(1, ended)] = True
    cached = [max(1, int((case["rows"] - 1) * _part(b, 0.1))) for b in range(B)]
    new = [max(1, int(min(case["prompt"], case["rows"]) * _part(b, 0.25))) if gone[b] else 1 for b in range(B)]
    return cached, new, gone


def _append_lens(case):
    """(rows already there, new rows) of each request."""
    B, T = case["B"], case["T"]
    start = [int(case["rows"] * _part(b, 0.1)) for b in range(B)]
    share = [_part(b, 0.2) for b in range(B)]
    new = [1 + int((T - B) * s / sum(share)) for s in share]
    new[-1] += T - sum(new)
    return start, new


def _decode_lens(case):
    return [max(1, int(case["len"] * _part(b))) for b in range(case["B"])]


def _prefill_lens(case):
    """(new tokens, rows after them) of each request: `prompts` of them with many, the others with one."""
    B, n = case["B"], case["prompts"]
    long = {(i * B) // n for i in range(n)}
    new = [max(1, int(case["S"] * _part(b))) if b in long else 1 for b in range(B)]
    return new, [n + int(case["start"] * _part(b + 1 if B > 1 else 0)) for b, n in enumerate(new)]


def _ceil(a, b):
    return -(-a // b)


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
        e = _exponent(x.abs().amax((3, 4)))
        pages[p:p + n] = _codes(x, e[..., None, None]).view(n, Hkv, page, D)
        scale[p:p + n] = _pow2(e)
    return pages, scale


def _table(seed, rows, page, spare=3):
    """Pages of each request's rows, in shuffled order; -1 behind them. Returns the table and the pool's size."""
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


def _starts(new):
    s = [0]
    for n in new:
        s.append(s[-1] + n)
    return s


def _qkv(g, T, Hq, Hkv, D):
    """q, k and v of one fused projection's rows, as views of it."""
    x = torch.randn((T, Hq + 2 * Hkv, D), generator=g, device="cuda")
    x[:, :Hq] *= 1.2
    x[:, Hq:Hq + Hkv] *= torch.exp(0.4 * torch.randn((Hkv, D), generator=g, device="cuda"))
    x = x.to(BF)
    return x[:, :Hq], x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:]


def prepare(case, seed):
    kind, g, s = case["kind"], _gen(seed), {"case": dict(case)}
    page = case["page"]
    if kind == "pages":
        cached, new, gone = _page_lens(case)
        table, P, free = _table(seed, cached, page, 0)
        want = sum(_ceil(n if x else c + n, page) - (0 if x else _ceil(c, page)) for c, n, x in zip(cached, new, gone))
        back = sum(_ceil(c, page) for c, x in zip(cached, gone) if x)
        more = max(0, want - back)
        more = max(1, more * 2 // 3) if case["tight"] else more + 7      # pages that are free before the step
        mp = max(table.shape[1], max(_ceil(n if x else c + n, page) for c, n, x in zip(cached, new, gone)))
        s["table"] = torch.full((case["B"], mp), -1, dtype=torch.int32, device="cuda")
        s["table"][:, :table.shape[1]] = table.cuda()
        s["free"] = torch.full((P + more,), -1, dtype=torch.int32, device="cuda")
        s["free"][:more] = P + torch.randperm(more, generator=g, device="cuda").to(torch.int32)
        s["count"] = _ints([more])
        s["ended"], s["cached"], s["new"] = _ints([int(x) for x in gone]), _ints([0 if x else c for c, x in zip(cached, gone)]), _ints(new)
        # a batch may hold fewer tokens than the requests ask for
        s["slots"] = torch.zeros(max(1, sum(new) * 3 // 4) if case["tight"] else sum(new) + 13, dtype=torch.int32, device="cuda")
        s["starts"], s["lens"] = torch.empty(case["B"] + 1, dtype=torch.int32, device="cuda"), torch.empty(case["B"], dtype=torch.int32, device="cuda")
        return s
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    if kind == "append":
        start, new = _append_lens(case)
        rows, T = [a + n for a, n in zip(start, new)], case["T"]
    elif kind == "decode":
        rows, T = _decode_lens(case), case["B"]
    else:
        new, rows = _prefill_lens(case)
        T = sum(new) + (5 if case["B"] > 1 else 0)
    table, P, _ = _table(seed, rows, page)
    s["kp"], s["ks"] = _filled(g, P, Hkv, page, D, 0.4)
    s["vp"], s["vs"] = _filled(g, P, Hkv, page, D, 0.0)
    s["q"], s["k"], s["v"] = _qkv(g, T, Hq, Hkv, D)
    s["table"], s["lens"], s["max_len"] = table.cuda(), _ints(rows), max(rows)
    if kind == "append":
        tl = table.tolist()
        s["slots"] = _ints([tl[b][r // page] * page + r % page for b in range(case["B"]) for r in range(start[b], rows[b])])
        # read back: the new rows and those before them in their first block
        s["read"] = _ints([tl[b][r // page] * page + r % page for b in range(case["B"]) for r in range(start[b] // BLOCK * BLOCK, rows[b])])
        s["k_out"], s["v_out"] = (torch.empty((len(s["read"]), Hkv, D), dtype=BF, device="cuda") for _ in range(2))
        return s
    s["out"] = torch.zeros((T, Hq, D), dtype=BF, device="cuda")
    if kind == "prefill":
        s["starts"], s["S"] = _ints(_starts(new)), max(new)
    return s


# ---- the plain forms ----------------------------------------------------------------------------
def _plain_pages(s):
    page, table, free, count = s["case"]["page"], s["table"], s["free"], s["count"]
    B, mp = table.shape
    P = free.numel()
    # release
    give = (s["ended"][:, None] != 0) & (table >= 0)
    at = count + give.view(-1).cumsum(0) - 1
    at = torch.where(give.view(-1) & (at < P), at, P)
    free.copy_(torch.cat([free, free[:1]]).scatter(0, at, table.view(-1))[:P])
    count += give.sum()
    count.clamp_(max=P)
    table.masked_fill_(give, -1)
    # reserve
    c, n = s["cached"].long(), s["new"].long()
    there = (c >= 0) & (n >= 0)
    n = torch.where(there, n, 0)
    c = torch.where(there, c, 0)
    starts = torch.cat([n[:1] * 0, n.cumsum(0)])
    p = torch.arange(mp, device=table.device)
    fits = there & (c + n <= mp * page)
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
    return _pages_out(s)


def _pages_out(s):
    return {k: s[k] for k in ("table", "free", "count", "starts", "lens", "slots")}


def _plain_store(pages, scale, x, slots):
    """x [T, Hkv, D] into the rows `slots`: blocks whose scale grows are rescaled."""
    P, H, page, D = pages.shape
    keep = slots >= 0
    slot = slots.long().clamp(min=0)
    pg, blk, row = slot // page, slot % page // BLOCK, slot % BLOCK
    x = x.float()
    fine = torch.where(x.isfinite() & keep[:, None, None], x.abs(), 0.0).amax(2)                             # [T, H]
    ids = torch.where(keep, slot // BLOCK, P * (page // BLOCK))
    amax = torch.zeros((P * (page // BLOCK) + 1, H), device=x.device).index_reduce(0, ids, fine, "amax")[ids]
    first = torch.full((P * (page // BLOCK) + 1,), BLOCK, device=x.device, dtype=torch.long).index_reduce(0, ids, row, "amin")[ids]
    old = torch.frexp(scale[pg, :, blk])[1] - 1
    e = _exponent(amax)
    e = torch.where((first == 0)[:, None], e, torch.maximum(e, old))
    # the block's earlier rows at the new scale; its other rows as they are
    view = pages.view(P, H, page // BLOCK, BLOCK, D)
    held = view[pg, :, blk]                                                                                 # [T, H, 16, D]
    value = held.float() * _pow2(old)[..., None, None]
    before = (torch.arange(BLOCK, device=x.device) < first[:, None])[:, None, :, None] & (e > old)[..., None, None]
    again = torch.where(before, _codes(value, e[..., None, None]).view(torch.uint8), held.view(torch.uint8)).view(F8)
    pk, bk, rk = pg[keep], blk[keep], row[keep]
    view.view(torch.uint8)[pk, :, bk] = again[keep].view(torch.uint8)
    scale[pk, :, bk] = _pow2(e)[keep]
    view.view(torch.uint8)[pk, :, bk, rk] = _codes(x, e[..., None])[keep].view(torch.uint8)


def _plain_rows(pages, scale, slots):
    page = pages.shape[2]
    slot = slots.long()
    return (pages.view(torch.uint8)[slot // page, :, slot % page].view(F8).float() * scale[slot // page, :, slot % page // BLOCK][..., None]).to(BF)


def _plain_cache(pages, scale, table):
    """[B, Hkv, rows, D] in f32: the pages of each request, as the values they stand for."""
    B, mp = table.shape
    P, H, page, D = pages.shape
    t = table.long().clamp(min=0)
    x = pages.view(torch.uint8)[t].view(F8).float().view(B, mp, H, page // BLOCK, BLOCK, D) * scale[t][..., None, None]
    return x.transpose(1, 2).reshape(B, H, mp * page, D)


def _plain_attention(q, k, v, valid):
    """q [B, N, Hq, D], k/v [B, Hkv, L, D] in f32, valid [B, N, L] -> [B, N, Hq, D]."""
    B, N, Hq, D = q.shape
    Hkv, L = k.shape[1], k.shape[2]
    G = Hq // Hkv
    q = q.view(B, N, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B * Hkv, G * N, D) * (1.0 / math.sqrt(D))
    s = torch.bmm(q, k.reshape(B * Hkv, L, D).transpose(1, 2).contiguous()).view(B, Hkv, G, N, L)
    s.masked_fill_(~valid[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    s.sub_(m.masked_fill(m == -math.inf, 0.0)).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.bmm(s.view(B * Hkv, G * N, L), v.reshape(B * Hkv, L, D).contiguous()).view(B, Hkv, G, N, D)
    return (o / total.clamp(min=1e-38)).permute(0, 3, 1, 2, 4).reshape(B, N, Hq, D)


def _plain_decode(s):
    k, v = _plain_cache(s["kp"], s["ks"], s["table"]), _plain_cache(s["vp"], s["vs"], s["table"])
    valid = torch.arange(k.shape[2], device=k.device) < s["lens"][:, None]
    return s["out"].copy_(_plain_attention(s["q"].float()[:, None], k, v, valid[:, None])[:, 0])


def _plain_prefill(s):
    k, v = _plain_cache(s["kp"], s["ks"], s["table"]), _plain_cache(s["vp"], s["vs"], s["table"])
    start, new = s["starts"][:-1].long(), (s["starts"][1:] - s["starts"][:-1]).long()
    i = torch.arange(s["S"], device=k.device)
    there = i < new[:, None]                                                                                # [B, S]
    tok = (start[:, None] + i).clamp(max=s["q"].shape[0] - 1)
    pos = (s["lens"].long() - new)[:, None] + i
    valid = (torch.arange(k.shape[2], device=k.device) <= pos[..., None]) & there[..., None]
    s["out"][tok[there]] = _plain_attention(s["q"].float()[tok], k, v, valid)[there].to(BF)
    return s["out"]


def run(s):
    kind = s["case"]["kind"]
    if own:
        import aila_amd as A
        if kind == "pages":
            A.kv_pages_release(s["ended"], s["table"], s["free"], s["count"])
            A.kv_pages_reserve(s["cached"], s["new"], s["table"], s["free"], s["count"], s["case"]["page"], s["slots"], s["starts"], s["lens"])
            return _pages_out(s)
        cache = (s["kp"], s["vp"], s["ks"], s["vs"])
        if kind == "append":
            A.kv_append_paged_fp8(s["k"], s["v"], *cache, s["slots"])
            return A.kv_read_paged_fp8(*cache, s["read"], s["k_out"], s["v_out"])
        q = s["q"]
        if "ws" not in s:      # the workspace that a program keeps for its calls of this size
            B, (Hq, D), Hkv = s["case"]["B"], q.shape[1:], s["kp"].shape[1]
            size = A.gqa_decode_paged_fp8_workspace_size(B, Hq, Hkv, D, s["max_len"]) if kind == "decode" else \
                A.gqa_prefill_paged_fp8_workspace_size(q.shape[0], B, Hq, Hkv, D, s["max_len"])
            s["ws"] = torch.empty(size, dtype=torch.uint8, device="cuda")
        if kind == "decode":
            return A.gqa_decode_paged_fp8(q, *cache, s["table"], s["lens"], s["max_len"], out=s["out"], workspace=s["ws"])
        return A.gqa_prefill_paged_fp8(q, *cache, s["table"], s["starts"], s["lens"], s["max_len"], out=s["out"], workspace=s["ws"])
    if kind == "pages":
        return _plain_pages(s)
    if kind == "append":
        _plain_store(s["kp"], s["ks"], s["k"], s["slots"])
        _plain_store(s["vp"], s["vs"], s["v"], s["slots"])
        s["k_out"].copy_(_plain_rows(s["kp"], s["ks"], s["read"]))
        s["v_out"].copy_(_plain_rows(s["vp"], s["vs"], s["read"]))
        return s["k_out"], s["v_out"]
    return _plain_decode(s) if kind == "decode" else _plain_prefill(s)


def work(case):
    if case["kind"] == "pages":
        cached, new, gone = _page_lens(case)
        page = case["page"]
        moved = sum(_ceil(c, page) + _ceil(n, page) if x else _ceil(c + n, page) - _ceil(c, page) for c, n, x in zip(cached, new, gone))
        # lengths and flags in, starts and lengths out, slots out, the pages given and taken: table and free list
        return {"bytes": 4.0 * (5 * case["B"] + sum(new) + 2 * moved), "flops": 0.0}
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    row = Hkv * (D + 4 / BLOCK) * 2            # of the cache, K and V
    if case["kind"] == "append":
        start, new = _append_lens(case)
        T, R = case["T"], sum(a % BLOCK + n for a, n in zip(start, new))
        return {"bytes": T * (Hkv * D * 4 + row) + R * (row + Hkv * D * 4), "flops": 0.0}
    if case["kind"] == "decode":
        rows = sum(_decode_lens(case))
        return {"bytes": rows * row + case["B"] * Hq * D * 4, "flops": 4.0 * rows * Hq * D}
    new, lens = _prefill_lens(case)
    pairs = sum(n * (r - n) + n * (n + 1) // 2 for n, r in zip(new, lens))
    return {"bytes": sum(lens) * row + sum(new) * Hq * D * 4, "flops": 4.0 * pairs * Hq * D}


# ---- the definitions in 64 bits -----------------------------------------------------------------
def _step64(x):
    """Nearest e4m3 value of x (float64), ties to even."""
    a = np.abs(x)
    unit = np.exp2(np.maximum(np.floor(np.log2(np.where(a > 0, a, 1.0))), -6.0) - 3.0)
    return np.where(np.isfinite(x), np.clip(np.rint(x / unit) * unit, -LARGEST, LARGEST), np.nan)


def _exact_rows(pages, scale, x, slots, read):
    """The rows `read` after x went to `slots`, block by block of 16 rows."""
    P, H, page, D = pages.shape
    slots, read, x = slots.tolist(), read.tolist(), x.double().cpu().numpy()
    nb = page // BLOCK
    blocks = sorted({r // BLOCK for r in read} | {r // BLOCK for r in slots if r >= 0})
    at = torch.tensor(blocks, device=pages.device)
    code = pages.view(torch.uint8)[at // nb].view(len(blocks), H, nb, BLOCK, D)[torch.arange(len(blocks), device=at.device), :, at % nb].view(F8)
    old = scale[at // nb, :, at % nb].double().cpu().numpy()                                                # [n, H]
    value = code.float().double().cpu().numpy() * old[..., None, None]                                      # [n, H, 16, D]
    where = {blk: i for i, blk in enumerate(blocks)}
    runs = {}
    for t, r in enumerate(slots):
        if r >= 0:
            runs.setdefault(r // BLOCK, []).append(t)
    for blk, toks in runs.items():
        i, rows = where[blk], [slots[t] % BLOCK for t in toks]
        fresh = x[toks].transpose(1, 0, 2)                                                                  # [H, n, D]
        top = np.where(np.isfinite(fresh), np.abs(fresh), 0.0).max((1, 2))
        e = np.clip(np.ceil(np.log2(np.where(top > 0, top, 1e-300) / LARGEST)), E_MIN, E_MAX)
        s = np.exp2(e) if min(rows) == 0 else np.maximum(np.exp2(e), old[i])
        s = s[:, None, None]
        value[i][:, :min(rows)] = _step64(value[i][:, :min(rows)] / s) * s
        value[i][:, rows] = _step64(fresh / s) * s
    return np.stack([value[where[r // BLOCK]][:, r % BLOCK] for r in read])


def _exact_attention(q, kp, ks, vp, vs, table, n, rows):
    """q [N, Hq, D] of one request, its last N rows; in float64, some tokens at a time."""
    N, Hq, D = q.shape
    P, H, page, _ = kp.shape
    ids = table[:_ceil(rows, page)].long()

    def whole(pages, scale):
        x = pages.view(torch.uint8)[ids].view(F8).double() * scale[ids].double().repeat_interleave(BLOCK, 2)[..., None]
        return x.permute(1, 0, 2, 3).reshape(H, -1, D)[:, :rows].contiguous()

    k, v, out = whole(kp, ks), whole(vp, vs), torch.empty((N, Hq, D), dtype=torch.float64, device=q.device)
    kt = k.transpose(1, 2).contiguous()
    key = torch.arange(rows, device=q.device)
    step = max(1, (1 << 28) // (Hq * rows))
    for a in range(0, N, step):
        b = min(N, a + step)
        x = q[a:b].double().view(b - a, H, Hq // H, D).permute(1, 0, 2, 3).reshape(H, -1, D)
        s = (torch.bmm(x.contiguous(), kt) / math.sqrt(D)).view(H, b - a, Hq // H, rows)
        seen = key <= torch.arange(rows - N + a, rows - N + b, device=q.device)[:, None]
        w = torch.softmax(s.masked_fill(~seen[None, :, None], -math.inf), -1).view(H, -1, rows)
        out[a:b] = torch.bmm(w, v).view(H, b - a, Hq // H, D).permute(1, 0, 2, 3).reshape(b - a, Hq, D)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "pages":
        return None
    if kind == "append":
        return (_exact_rows(s["kp"], s["ks"], s["k"], s["slots"], s["read"]), _exact_rows(s["vp"], s["vs"], s["v"], s["slots"], s["read"]))
    out = s["out"].double()
    if kind == "decode":
        new, rows, at = [1] * case["B"], _decode_lens(case), list(range(case["B"] + 1))
    else:
        new, rows = _prefill_lens(case)
        at = _starts(new)
    for b in range(case["B"]):
        out[at[b]:at[b + 1]] = _exact_attention(s["q"][at[b]:at[b + 1]], s["kp"], s["ks"], s["vp"], s["vs"], s["table"][b], new[b], rows[b])
    return out
