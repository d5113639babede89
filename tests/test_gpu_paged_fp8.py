"""GPU parity of the 8-bit paged KV cache (kv_pages_*, kv_*_paged_fp8,
gqa_*_paged_fp8) against plain forms in 64 bits: tables, codes and scales bit for
bit, attention within a bound derived from its roundings."""
import os
import subprocess

import numpy as np
import pytest

import paged_fp8_ref as ref

pytestmark = pytest.mark.gpu

F8_NAN = 0x7F


@pytest.fixture(autouse=True)
def _say(request):
    print(request.node.name, flush=True)


def _cache(P, H, page, D, seed, spread=1.0):
    """A cache of random codes (all but NaN) and random scales."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes = []
    for _ in range(2):
        c = torch.randint(0, 255, (P, H, page, D), generator=g, device="cuda").to(torch.uint8)
        c[(c & 127) == F8_NAN] = 0
        c &= 0xBF          # |code| < 2: values of ordinary size
        codes.append(c.view(torch.float8_e4m3fn))
    scales = [torch.exp2(torch.randint(-2, 3, (P, H, page // 16), generator=g, device="cuda").float() * spread) for _ in range(2)]
    return (*codes, *scales)


def _table(lens, page, P, seed, extra=1):
    import torch
    mp = max(1, max(-(-n // page) for n in lens)) + extra
    perm = np.random.default_rng(seed).permutation(P)
    t = np.full((len(lens), mp), -1, np.int32)
    at = 0
    for b, n in enumerate(lens):
        k = -(-n // page)
        t[b, :k] = perm[at:at + k]
        at += k
    assert at <= P
    return torch.from_numpy(t).cuda()


def _i32(v):
    import torch
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------- rows ----
def test_read_gives_every_code_and_scale():
    import torch
    import aila_amd as A
    P, H, page, D = 14, 2, 16, 64
    codes = torch.arange(P * H * page * D, device="cuda").to(torch.uint8).view(P, H, page, D)
    exps = torch.tensor([-100, -99, -40, -10, -1, 0, 1, 9, 40, 100, 117, 118, 119, 3], device="cuda")
    scale = torch.exp2(exps.double()).float()[:, None, None].expand(P, H, 1).contiguous()
    kp, vp = codes.view(torch.float8_e4m3fn), codes.flip(3).contiguous().view(torch.float8_e4m3fn)
    slots = list(range(P * page)) + [-1, P * page, 2**31 - 1, 5]
    k, v = A.kv_read_paged_fp8(kp, vp, scale, scale, _i32(slots))
    for got, pages in ((k, kp), (v, vp)):
        want = ref.Cache(pages, scale).rows(slots)
        got = got.double().cpu().numpy()
        assert np.array_equal(got, want, equal_nan=True)


def _rows(g, T, H, D, kind):
    import torch
    x = torch.randn((T, H, D), generator=g, device="cuda", dtype=torch.float64)
    if kind == "wide":        # sizes over 60 powers of two, row by row
        x *= torch.exp2(torch.randint(-30, 31, (T, H, 1), generator=g, device="cuda").double())
    if kind == "special":
        x[0::5] = 0
        x[1::7, :, 3] = float("nan")
        x[2::6, :, 5] = float("inf")
        x[2::6, :, 6] = -float("inf")
        x[3::9] *= 1e-38
        x[4::11] *= 1e38
        x[5::13] = 3.3e38
    return x.to(torch.bfloat16)


@pytest.mark.parametrize("D,H,page,kind", [(64, 1, 16, "plain"), (128, 3, 32, "wide"), (256, 2, 48, "special"), (128, 8, 64, "special"),
                                           (64, 5, 128, "wide"), (256, 4, 16, "wide")])
def test_append_matches_the_definition(D, H, page, kind):
    """Rows arrive in pieces of all lengths, so that runs begin and end anywhere in
    a block and scales grow under rows that are there."""
    import torch
    import aila_amd as A
    g = torch.Generator(device="cuda").manual_seed(D + H + page)
    P, lens = 9, [0, 0, 0]
    kp, vp, ks, vs = _cache(P, H, page, D, 3)
    want = [ref.Cache(kp, ks), ref.Cache(vp, vs)]
    table = _table([3 * page] * 3, page, P, 7).cpu().numpy()
    for step in range(12):
        new = [[1, 16, 0], [2, 1, 5], [15, 1, 1], [1, 7, 17], [0, 1, 1], [3, 3, 3], [1, 1, 1], [1, 1, 1], [9, 0, 4], [1, 2, 1], [1, 1, 1], [5, 1, 2]][step]
        slots = []
        for b in range(3):
            for r in range(lens[b], min(lens[b] + new[b], 3 * page)):
                slots.append(int(table[b][r // page]) * page + r % page)
            lens[b] = min(lens[b] + new[b], 3 * page)
        if step % 3 == 1:
            slots = [-1] + slots + [-1, P * page, -5]
        if not slots:
            continue
        x = _rows(g, len(slots), H, 2 * D, kind)
        k, v = x[:, :, :D].contiguous(), x[:, :, D:].contiguous()
        if step % 2:
            fused = torch.cat([k, v, k], 1)
            k, v = fused[:, :H], fused[:, H:2 * H]
        A.kv_append_paged_fp8(k, v, kp, vp, ks, vs, _i32(slots))
        for c, t in zip(want, (k, v)):
            c.append(t.double().cpu().numpy(), slots)
        for c, pages, scale in zip(want, (kp, vp), (ks, vs)):
            assert np.array_equal(scale.double().cpu().numpy(), c.scale), step
            assert np.array_equal(pages.float().double().cpu().numpy(), c.val, equal_nan=True), step


def test_append_rounds_every_bf16_value():
    """All finite bf16 values, each block of 16 rows holding one power of two range."""
    import torch
    import aila_amd as A
    D, bits = 128, torch.arange(0, 0x7F80, dtype=torch.int32)
    bits = torch.cat([bits, bits | 0x8000])
    x = bits.to(torch.int16).view(torch.bfloat16)
    T = -(-len(x) // D)
    x = torch.cat([x, x.new_zeros(T * D - len(x))]).view(T, 1, D).cuda()
    P = -(-T // 16)
    kp, vp, ks, vs = A.paged_fp8_cache(P, 1, 16, D)
    slots = list(range(T))
    A.kv_append_paged_fp8(x, -x, kp, vp, ks, vs, _i32(slots))
    k, v = A.kv_read_paged_fp8(kp, vp, ks, vs, _i32(slots))
    c = ref.Cache(torch.zeros_like(kp.view(torch.uint8)), ks)
    c.append(x.double().cpu().numpy(), slots)
    assert np.array_equal(k.double().cpu().numpy(), c.rows(slots))
    assert torch.equal(v, -k)


@pytest.mark.parametrize("T", [1, 256, 257, 1023, 1025, 2047, 2049, 5003])
def test_append_of_a_long_prompt(T):
    """Above and below the batch sizes where a workgroup takes more tokens."""
    import torch
    import aila_amd as A
    H, page, D = 3, 64, 64
    g = torch.Generator(device="cuda").manual_seed(T)
    P = T // page + 2
    kp, vp, ks, vs = A.paged_fp8_cache(P, H, page, D)
    start = 37                       # the first run begins inside a block
    perm = np.random.default_rng(T).permutation(P)
    slots = [int(perm[(start + i) // page]) * page + (start + i) % page for i in range(T)]
    k, v = (torch.randn((T, H, D), generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    want = [ref.Cache(kp, ks), ref.Cache(vp, vs)]
    A.kv_append_paged_fp8(k, v, kp, vp, ks, vs, _i32(slots))
    for c, t, pages, scale in zip(want, (k, v), (kp, vp), (ks, vs)):
        c.append(t.double().cpu().numpy(), slots)
        assert np.array_equal(pages.float().double().cpu().numpy(), c.val)
        assert np.array_equal(scale.double().cpu().numpy(), c.scale)


@pytest.mark.parametrize("T", [64, 300, 1500, 2500])
def test_append_of_single_tokens_and_short_runs(T):
    """Runs of one to five tokens, so that a workgroup's tile holds many and they
    go on behind its end."""
    import torch
    import aila_amd as A
    H, page, D = 2, 16, 128
    g = torch.Generator(device="cuda").manual_seed(T)
    kp, vp, ks, vs = _cache(T, H, page, D, T)
    slots, p = [], 0
    while len(slots) < T:
        n = min(1 + p * 7 % 5, T - len(slots))
        r = p * 5 % (page - n + 1)
        slots += [p * page + r + i for i in range(n)]
        if p % 11 == 3 and len(slots) < T:
            slots.append(-1)
        p += 1
    k, v = (torch.randn((T, H, D), generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    want = [ref.Cache(kp, ks), ref.Cache(vp, vs)]
    A.kv_append_paged_fp8(k, v, kp, vp, ks, vs, _i32(slots))
    for c, t, pages, scale in zip(want, (k, v), (kp, vp), (ks, vs)):
        c.append(t.double().cpu().numpy(), slots)
        assert np.array_equal(pages.float().double().cpu().numpy(), c.val)
        assert np.array_equal(scale.double().cpu().numpy(), c.scale)


# ------------------------------------------------------------------ pages ----
def _state(rng, B, mp, page, P, most):
    """A consistent pool: lengths, table, stack of free pages."""
    cached = [int(x) for x in rng.integers(0, most + 1, B)]
    perm = [int(x) for x in rng.permutation(P)]
    table = [[-1] * mp for _ in range(B)]
    at = 0
    for b in range(B):
        k = min(-(-cached[b] // page), mp)
        if at + k > P:
            cached[b], k = 0, 0
        for p in range(k):
            table[b][p] = perm[at + p]
        at += k
    free = perm[at:] + [-7] * at
    return cached, table, free, P - at


def _reserve_both(cached, new, table, free, count, page, cap):
    import aila_amd as A
    t, f, c = _i32(table), _i32(free), _i32([count])
    slots = _i32([77] * cap)
    starts, lens, _ = A.kv_pages_reserve(_i32(cached), _i32(new), t, f, c, page, slots)
    want = ref.reserve(cached, new, table, free, count, page, cap)
    got = (t.tolist(), c.item(), starts.tolist(), lens.tolist(), slots.tolist())
    for name, a, b in zip(("table", "count", "starts", "lens", "slots"), got, want):
        assert a == b, name
    assert f.tolist() == free
    return want


@pytest.mark.parametrize("B,page,mp,P,most,new,cap", [
    (1, 16, 4, 4, 60, 1, 1), (1, 64, 2, 3, 0, 128, 128), (3, 16, 8, 20, 100, 30, 64), (32, 64, 64, 900, 3000, 3, 300),
    (257, 16, 40, 5000, 600, 20, 2700), (1024, 16, 8, 8000, 100, 1, 1024), (1025, 48, 4, 2500, 150, 5, 20000),
    (2048, 16, 6, 9000, 90, 2, 8193), (5, 128, 300, 1000, 20000, 9000, 40000), (40, 16, 30, 300, 400, 90, 2000),
    (40, 16, 1200, 30000, 19000, 100, 6000), (20, 16, 500, 9000, 7900, 3, 40)])
def test_reserve_and_release(B, page, mp, P, most, new, cap):
    """Ordinary steps, pools and batches too small for all, requests absent, rows
    that exceed the table, repeated calls and rows taken back."""
    import aila_amd as A
    rng = np.random.default_rng(B + page)
    cached, table, free, count = _state(rng, B, mp, page, P, min(most, mp * page))
    fresh = [int(x) for x in rng.integers(0, new + 1, B)]
    if B > 4:
        fresh[1], cached[2] = -3, -1 - cached[2]
        fresh[4] = mp * page
    t1, c1, _, lens, _ = _reserve_both(cached, fresh, table, free, count, page, cap)
    again = _reserve_both(cached, fresh, t1, free, c1, page, cap)       # takes pages for no request twice
    assert [x for x, n in zip(again[0], lens) if n] == [x for x, n in zip(t1, lens) if n]
    back = [max(0, n - 3) for n in lens]                                 # tokens taken back
    t2, c2, *_ = _reserve_both(back, [2 if n else 0 for n in lens], again[0], free, again[1], page, max(1, 2 * B))
    flags = [int(x) for x in rng.integers(0, 2, B)]
    t, f, c = _i32(t2), _i32(free), _i32([c2])
    A.kv_pages_release(_i32(flags), t, f, c)
    want = ref.release(flags, t2, free, c2)
    assert (t.tolist(), f.tolist(), c.item()) == want
    A.kv_pages_release(_i32(flags), t, f, c)                             # nothing left to give
    assert (t.tolist(), f.tolist(), c.item()) == want


def test_reserve_saturates_and_survives_a_bad_count():
    import aila_amd as A
    t, f = _i32([[-1, -1]] * 3), _i32([0, 1, 2, 3])
    starts, lens, slots = A.kv_pages_reserve(_i32([0, 0, 0]), _i32([2**31 - 1, 2**31 - 1, 4]), t, f, _i32([4]), 16, _i32([9] * 8))
    assert starts.tolist() == [0, 2**31 - 1, 2**31 - 1, 2**31 - 1]
    assert lens.tolist() == [0, 0, 0] and slots.tolist() == [-1] * 8 and t.tolist() == [[-1, -1]] * 3
    count = _i32([100])       # more than the stack holds: taken as the stack's size
    _, lens, _ = A.kv_pages_reserve(_i32([0, 0, 0]), _i32([1, 1, 1]), t, f, count, 16, _i32([9] * 8))
    assert lens.tolist() == [1, 1, 1] and t.tolist() == [[3, -1], [2, -1], [1, -1]] and count.item() == 1


# -------------------------------------------------------------- attention ----
def _check(got, q, cache, table, starts, lens, max_len, weight_step):
    import torch
    kp, vp, ks, vs = cache
    got = got.double()
    for b, L in enumerate(lens):
        L = min(max(L, 0), max_len)
        a, e = starts[b], starts[b + 1]
        if a == e:
            continue
        if L == 0:
            assert not got[a:e].any(), b
            continue
        k, held = ref.gather(kp, ks, table[b], L)
        v, _ = ref.gather(vp, vs, table[b], L)
        out, mag, big = ref.attention(q[a:e], k, v, held, L - (e - a) + 1)
        tol = ref.attention_tolerance(out, mag, big, L, q.shape[2], weight_step)
        nan = torch.isnan(out)
        assert torch.equal(nan, torch.isnan(got[a:e])), (b, L)
        off = ((got[a:e] - out).abs() / tol)[~nan]
        assert not len(off) or off.max() <= 1, (b, L, off.max().item())


LENS = [1, 0, 15, 16, 17, 31, 33, 127, 128, 129, 300]


@pytest.mark.parametrize("D,Hq,Hkv,page,lens", [
    (64, 2, 2, 16, LENS), (128, 3, 1, 64, LENS), (256, 4, 1, 16, LENS), (128, 10, 2, 48, [700, 5, 1025]), (256, 8, 1, 128, [2000]),
    (64, 16, 1, 16, [513, 0, 64]), (256, 32, 2, 64, [400, 90]), (128, 17, 1, 32, [600, 1]), (64, 40, 1, 16, [260]), (256, 33, 1, 16, [150, 500]),
    (128, 8, 8, 64, [4097]), (256, 6, 2, 64, [9000])])
def test_decode(D, Hq, Hkv, page, lens):
    import torch
    import aila_amd as A
    B = len(lens)
    P = sum(-(-n // page) for n in lens) + 3
    cache = _cache(P, Hkv, page, D, D + Hq)
    table = _table(lens, page, P, D + page)
    max_len = table.shape[1] * page
    g = torch.Generator(device="cuda").manual_seed(Hq)
    fused = torch.randn((B, Hq + 3, D), generator=g, device="cuda").to(torch.bfloat16)
    q = fused[:, :Hq]
    size = A.gqa_decode_paged_fp8_workspace_size(B, Hq, Hkv, D, max_len)
    full = torch.empty(size, dtype=torch.uint8, device="cuda")
    few = full[:max(1024 + 4 * 16 * (D + 4) * 4, size // 7 // 16 * 16)].contiguous()     # fewer workgroups, two at least
    for ws in (full, few, None):
        got = A.gqa_decode_paged_fp8(q, *cache, table, _i32(lens), max_len, workspace=ws)
        # P is the sum of two bf16: the second's half step is 2^-16 of it
        _check(got, q, cache, table, range(B + 1), lens, max_len, 2.0 ** -16)
    short = max(1, max(lens) // 2)        # a bound below the lengths cuts them
    got = A.gqa_decode_paged_fp8(q.contiguous(), *cache, table, _i32(lens), short, workspace=full)
    _check(got, q, cache, table, range(B + 1), lens, short, 2.0 ** -16)


@pytest.mark.parametrize("D,Hq,Hkv,page,new,lens", [
    (64, 2, 2, 16, [1, 3, 0, 16, 17], [1, 3, 9, 16, 40]), (128, 3, 1, 64, [130, 1, 1], [130, 77, 1]), (256, 4, 1, 16, [33, 2], [300, 65]),
    (128, 10, 2, 48, [50, 1, 7], [700, 5, 7]), (256, 8, 1, 128, [70], [2000]), (64, 16, 1, 16, [4, 64, 0], [513, 64, 0]),
    (256, 33, 1, 16, [6, 5], [150, 5]), (128, 8, 8, 64, [200], [200]), (64, 8, 2, 16, [5, 4, 20], [0, 2, 12]), (128, 40, 8, 16, [2, 1, 90, 1], [300, 1, 90, 257])])
def test_prefill(D, Hq, Hkv, page, new, lens):
    """Lengths below the new tokens (a request that was not admitted has 0) leave
    the first tokens without a row."""
    import torch
    import aila_amd as A
    B = len(lens)
    P = sum(-(-n // page) for n in lens) + 3
    cache = _cache(P, Hkv, page, D, D + Hq)
    table = _table(lens, page, P, D + page)
    max_len = table.shape[1] * page
    starts = [0] + [int(x) for x in np.cumsum(new)]
    T = starts[-1] + 4                       # rows behind the last request
    g = torch.Generator(device="cuda").manual_seed(Hq)
    q = torch.randn((T, Hq + 2, D), generator=g, device="cuda").to(torch.bfloat16)[:, :Hq]
    size = A.gqa_prefill_paged_fp8_workspace_size(T, B, Hq, Hkv, D, max_len)
    for ws in (torch.empty(size, dtype=torch.uint8, device="cuda"), None):
        out = torch.full((T, Hq, D), 7.0, dtype=torch.bfloat16, device="cuda")
        A.gqa_prefill_paged_fp8(q, *cache, table, _i32(starts), _i32(lens), max_len, out=out, workspace=ws)
        _check(out, q, cache, table, starts, lens, max_len, 2.0 ** -8)     # P is rounded to bf16
        assert (out[starts[-1]:] == 7).all()


@pytest.mark.parametrize("D,Hq,Hkv", [(64, 8, 2), (128, 4, 4), (256, 16, 2)])
def test_masked_rows_may_hold_anything(D, Hq, Hkv):
    """NaN codes behind the lengths and NaN and infinite scales of blocks behind
    them do not show; a NaN in an attended row shows where it is attended and
    nowhere else; rows without a page, or with one outside the pool, are masked."""
    import torch
    import aila_amd as A
    page, lens = 32, [70, 45, 33, 40]
    P = 16
    kp, vp, ks, vs = _cache(P, Hkv, page, D, 5)
    table = _table([96] * 4, page, P, 6)
    for b, L in enumerate(lens):
        for r in range(L, 96):
            p = int(table[b, r // page])
            for pages, scale in ((kp, ks), (vp, vs)):
                pages.view(torch.uint8)[p, :, r % page] = F8_NAN | (r & 1) << 7
                if r // 16 * 16 >= L:
                    scale[p, :, r % page // 16] = float("nan") if r & 16 else float("inf")
    vp.view(torch.uint8)[int(table[0, 1]), :, 4, 7] = F8_NAN        # row 36 of request 0, dim 7
    kp.view(torch.uint8)[int(table[1, 1]), :, 8, 2] = F8_NAN        # row 40 of request 1
    table[2, 0] = -1
    table[3, 1] = P                                                 # outside the pool
    g = torch.Generator(device="cuda").manual_seed(1)
    q = torch.randn((4, Hq, D), generator=g, device="cuda").to(torch.bfloat16)
    for ws in (torch.empty(A.gqa_decode_paged_fp8_workspace_size(4, Hq, Hkv, D, 96), dtype=torch.uint8, device="cuda"), None):
        got = A.gqa_decode_paged_fp8(q, kp, vp, ks, vs, table, _i32(lens), 96, workspace=ws)
        assert torch.isnan(got[0, :, 7]).all() and torch.isnan(got[1]).all()
        _check(got, q, (kp, vp, ks, vs), table, range(5), lens, 96, 2.0 ** -16)
    new = [60, 20, 3, 12]
    starts = [0] + [int(x) for x in np.cumsum(new)]
    q = torch.randn((starts[-1], Hq, D), generator=g, device="cuda").to(torch.bfloat16)
    got = A.gqa_prefill_paged_fp8(q, kp, vp, ks, vs, table, _i32(starts), _i32(lens), 96)
    _check(got, q, (kp, vp, ks, vs), table, starts, lens, 96, 2.0 ** -8)
    assert not torch.isnan(got[:26]).any()       # rows 10 .. 35 of request 0 come before its NaN


@pytest.mark.parametrize("big", [1.0, 40.0, 4000.0])
def test_large_scores(big):
    """Softmaxes that one row takes over, and maxima that keep moving."""
    import torch
    import aila_amd as A
    D, Hq, Hkv, page, L = 128, 8, 2, 16, 777
    P = L // page + 2
    kp, vp, ks, vs = _cache(P, Hkv, page, D, 9)
    table = _table([L], page, P, 2)
    ks *= torch.exp2(torch.arange(P, device="cuda") % 5.0)[:, None, None]
    q = (torch.randn((1, Hq, D), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda") * big).to(torch.bfloat16)
    ws = torch.empty(A.gqa_decode_paged_fp8_workspace_size(1, Hq, Hkv, D, L), dtype=torch.uint8, device="cuda")
    for w in (ws, None):
        got = A.gqa_decode_paged_fp8(q, kp, vp, ks, vs, table, _i32([L]), L, workspace=w)
        _check(got, q, (kp, vp, ks, vs), table, [0, 1], [L], L, 2.0 ** -16)
    got = A.gqa_prefill_paged_fp8(q.expand(5, Hq, D).contiguous(), kp, vp, ks, vs, table, _i32([0, 5]), _i32([L]), L)
    _check(got, q.expand(5, Hq, D), (kp, vp, ks, vs), table, [0, 5], [L], L, 2.0 ** -8)


def _check_tokens(got, q, cache, table, starts, lens, max_len, tokens):
    """As _check, for some of a batch's tokens: {request: its tokens}."""
    for b, some in tokens.items():
        L, a, n = min(lens[b], max_len), starts[b], starts[b + 1] - starts[b]
        k, held = ref.gather(cache[0], cache[2], table[b], L)
        v, _ = ref.gather(cache[1], cache[3], table[b], L)
        for i in sorted({x % n for x in some}):
            out, mag, big = ref.attention(q[a + i:a + i + 1], k, v, held, L - n + 1 + i)
            tol = ref.attention_tolerance(out, mag, big, L, q.shape[2], 2.0 ** -8)
            off = (got[a + i:a + i + 1].double() - out).abs() / tol
            assert off.max() <= 1, (b, i, off.max().item())


@pytest.mark.parametrize("D,Hq,Hkv,page,new,lens", [
    # one request: more keys than a workgroup looks up at once, with and without runs
    (64, 8, 2, 16, [5], [40000]), (128, 4, 1, 64, [4], [35000]), (128, 4, 4, 64, [130], [33001]), (256, 8, 2, 64, [9], [12000]),
    (256, 2, 2, 48, [200], [23077]), (64, 4, 4, 32, [700], [1500]), (128, 32, 2, 16, [150], [150]),
    # batches: runs of odd lengths, tokens beside prompts, ends of prompts with few rows
    (128, 8, 2, 64, [300, 1, 700, 2], [33000, 40000, 700, 5]), (64, 6, 2, 16, [129, 1, 1, 44], [2129, 9000, 31, 20011]),
    (256, 16, 2, 32, [17, 3, 65, 1], [11100, 4097, 65, 12000]), (128, 2, 2, 16, [129, 257, 385, 8], [129, 777, 385, 3001]),
    (64, 1, 1, 16, [128, 145, 1, 0, 16], [128, 145, 20000, 0, 16]), (256, 4, 4, 16, [130, 1, 140], [130, 7000, 6001])])
def test_prefill_of_long_requests(D, Hq, Hkv, page, new, lens):
    import torch
    import aila_amd as A
    B = len(lens)
    P = sum(-(-n // page) for n in lens) + 3
    cache = _cache(P, Hkv, page, D, D + Hq)
    table = _table(lens, page, P, D + page)
    max_len = table.shape[1] * page
    starts = [0] + [int(x) for x in np.cumsum(new)]
    T = starts[-1]
    g = torch.Generator(device="cuda").manual_seed(Hq)
    q = torch.randn((T, Hq, D), generator=g, device="cuda").to(torch.bfloat16)
    some = {b: (0, 1, new[b] // 2, -2, -1) for b in range(B) if new[b]}
    size = A.gqa_prefill_paged_fp8_workspace_size(T, B, Hq, Hkv, D, max_len)
    for ws in (torch.empty(size, dtype=torch.uint8, device="cuda"), None):
        out = A.gqa_prefill_paged_fp8(q, *cache, table, _i32(starts), _i32(lens), max_len, workspace=ws)
        _check_tokens(out, q, cache, table, starts, lens, max_len, some)


@pytest.mark.parametrize("B,D,Hq,Hkv", [(1300, 64, 2, 1), (4096, 128, 2, 2), (1100, 256, 4, 1)])
def test_prefill_of_many_requests(B, D, Hq, Hkv):
    """More tiles than the list's threads, most of them of one token; every request
    against the decode of the same rows where it has one token."""
    import torch
    import aila_amd as A
    page, rng = 16, np.random.default_rng(B)
    lens = [int(x) for x in rng.integers(0, 60, B)]
    lens[7], lens[B - 3] = 3001, 1500
    new = [min(n, int(x)) for n, x in zip(lens, rng.choice([0, 1, 1, 1, 2, 17, 40], B))]
    new[7], new[B - 3] = 1, 400
    P = sum(-(-n // page) for n in lens) + 3
    cache = _cache(P, Hkv, page, D, B)
    table = _table(lens, page, P, B, extra=0)
    max_len = table.shape[1] * page
    starts = [0] + [int(x) for x in np.cumsum(new)]
    T = starts[-1]
    q = torch.randn((T, Hq, D), generator=torch.Generator(device="cuda").manual_seed(B), device="cuda").to(torch.bfloat16)
    ws = torch.empty(A.gqa_prefill_paged_fp8_workspace_size(T, B, Hq, Hkv, D, max_len), dtype=torch.uint8, device="cuda")
    out = A.gqa_prefill_paged_fp8(q, *cache, table, _i32(starts), _i32(lens), max_len, workspace=ws)
    some = {b: (0, -1) for b in [7, B - 3] + [int(x) for x in rng.choice(B, 60)] if new[b]}
    _check_tokens(out, q, cache, table, starts, lens, max_len, some)
    ones = [b for b in range(B) if new[b] == 1]
    at = torch.tensor([starts[b] for b in ones], device="cuda")
    one = A.gqa_decode_paged_fp8(q[at], *cache, table[torch.tensor(ones, device="cuda")].contiguous(), _i32([lens[b] for b in ones]), max_len)
    # half a step of bf16 each, and weights rounded to 2^-8 at most before values below 2 * 2^2
    assert ((one.double() - out[at].double()).abs() <= 2.0 ** -7 * one.double().abs() * (1 + 2.0 ** -7) + 2.0 ** -8 * 8).all()


@pytest.mark.parametrize("D,Hq,Hkv,new,lens", [(64, 1024, 128, [100, 3], [333, 3]), (128, 768, 128, [90, 70], [517, 300]), (256, 512, 64, [60, 61, 2], [161, 460, 9])])
def test_tiles_that_end_in_one_key_tile(D, Hq, Hkv, new, lens):
    """One or two workgroups a KV head walk all tiles of a batch, many of which have
    equally many key tiles but not the same last block, in any order; the requests
    alone give the same bits."""
    import torch
    import aila_amd as A
    page, B = 16, len(lens)
    P = sum(-(-n // page) for n in lens) + 3
    cache = _cache(P, Hkv, page, D, 7)
    table = _table(lens, page, P, 8)
    max_len = table.shape[1] * page
    starts = [0] + [int(x) for x in np.cumsum(new)]
    q = torch.randn((starts[-1], Hq, D), generator=torch.Generator(device="cuda").manual_seed(2), device="cuda").to(torch.bfloat16)
    ws = torch.empty(A.gqa_prefill_paged_fp8_workspace_size(starts[-1], B, Hq, Hkv, D, max_len), dtype=torch.uint8, device="cuda")
    want = A.gqa_prefill_paged_fp8(q, *cache, table, _i32(starts), _i32(lens), max_len)
    for _ in range(10):
        got = A.gqa_prefill_paged_fp8(q, *cache, table, _i32(starts), _i32(lens), max_len, workspace=ws)
        assert torch.equal(got, want)
    few = [h for h in range(0, Hkv, Hkv // 4)]            # some heads against the definition
    g = Hq // Hkv
    heads = [h * g + i for h in few for i in range(g)]
    small = [x[:, few].contiguous() if x.dtype == torch.float32 else x.view(torch.uint8)[:, few].contiguous().view(x.dtype) for x in cache]
    _check_tokens(got[:, heads].contiguous(), q[:, heads].contiguous(), small, table, starts, lens, max_len,
                  {b: (0, n // 3, n // 2, -1) for b, n in enumerate(new)})


@pytest.mark.parametrize("B,D,Hq,Hkv,page,most,max_len", [(20, 128, 8, 4, 32, 6000, 8000), (70, 64, 16, 1, 16, 5000, 6000), (9, 256, 32, 8, 64, 3000, 5000),
                                                          (4096, 64, 2, 1, 16, 40, 48), (300, 128, 20, 1, 16, 500, 5000)])
def test_decode_of_many_sequences(B, D, Hq, Hkv, page, most, max_len):
    """Splits with few records each, and one workgroup per sequence and head."""
    import torch
    import aila_amd as A
    rng = np.random.default_rng(B)
    lens = [int(x) for x in rng.integers(0, most + 1, B)]
    lens[1], lens[B // 2] = most, 0
    P = sum(-(-n // page) for n in lens) + 3
    cache = _cache(P, Hkv, page, D, B)
    table = _table(lens, page, P, B, extra=-(-max_len // page) - -(-most // page))
    q = torch.randn((B, Hq, D), generator=torch.Generator(device="cuda").manual_seed(B), device="cuda").to(torch.bfloat16)
    size = A.gqa_decode_paged_fp8_workspace_size(B, Hq, Hkv, D, max_len)
    some = [1, B // 2, B - 1] + [int(x) for x in rng.choice(B, 12)]
    for ws in (torch.empty(size, dtype=torch.uint8, device="cuda"), None):
        got = A.gqa_decode_paged_fp8(q, *cache, table, _i32(lens), max_len, workspace=ws)
        for b in some:
            _check(got[b:b + 1], q[b:b + 1], cache, table[b:b + 1], [0, 1], lens[b:b + 1], max_len, 2.0 ** -16)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_nan_rows_of_a_long_request(D):
    """A NaN that lies behind some tokens of a chunk, far from the start: shown where
    it is attended, in its dim, and nowhere else; with the keys walked in one run
    and in several, for a tile's rows and for single rows."""
    import torch
    import aila_amd as A
    page, L, Hq, Hkv = 16, 14000, 4, 2
    P = L // page + 2
    for n in (300, 5):
        cache = _cache(P, Hkv, page, D, 5)
        table = _table([L, 1], page, P, 6)
        at = L - 1 - n // 2
        cache[1].view(torch.uint8)[int(table[0, at // page]), 1, at % page, 11] = F8_NAN
        q = torch.randn((n + 1, Hq, D), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(torch.bfloat16)
        first = n - (L - at)           # the token whose own row it is
        for B in (1, 2):
            starts, lens = [0, n, n + 1][:B + 1], [L, 1][:B]
            size = A.gqa_prefill_paged_fp8_workspace_size(n + 1, B, Hq, Hkv, D, L)
            for ws in (torch.empty(size, dtype=torch.uint8, device="cuda"), None):
                out = A.gqa_prefill_paged_fp8(q, *cache, table[:B], _i32(starts), _i32(lens), L, workspace=ws)[:n]
                want = torch.zeros((n, Hq, D), dtype=torch.bool, device="cuda")
                want[first:, 2:, 11] = True
                assert torch.equal(torch.isnan(out), want), (n, B, ws is None)


def test_two_streams_with_workspaces_of_their_own():
    """Calls that overlap in time: each has its workspace, and both give what they
    give alone."""
    import torch
    import aila_amd as A
    D, Hq, Hkv, page, lens, new = 128, 8, 2, 16, [9000, 500, 40], [300, 1, 40]
    P = sum(-(-n // page) for n in lens) + 3
    cache, table = _cache(P, Hkv, page, D, 1), _table(lens, page, P, 2)
    max_len, T = table.shape[1] * page, sum(new)
    starts, seq = _i32([0] + [int(x) for x in np.cumsum(new)]), _i32(lens)
    q = torch.randn((T, Hq, D), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(torch.bfloat16)
    sizes = (A.gqa_prefill_paged_fp8_workspace_size(T, 3, Hq, Hkv, D, max_len), A.gqa_decode_paged_fp8_workspace_size(3, Hq, Hkv, D, max_len))

    def both(stream, wp, wd):
        a = A.gqa_prefill_paged_fp8(q, *cache, table, starts, seq, max_len, workspace=wp, stream=stream)
        return a, A.gqa_decode_paged_fp8(q[:3], *cache, table, seq, max_len, workspace=wd, stream=stream)

    ws = [[torch.empty(n, dtype=torch.uint8, device="cuda") for n in sizes] for _ in range(2)]
    want = both(None, *ws[0])
    st = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in st:
        s.wait_stream(torch.cuda.current_stream())
    got = [both(s, *w) for _ in range(4) for s, w in zip(st, ws)]
    for s in st:
        s.synchronize()
    for a, d in got:
        assert torch.equal(a, want[0]) and torch.equal(d, want[1])


def test_graphs_that_share_a_workspace():
    """Two captured calls of other shapes over one workspace, replayed in turn on a
    stream, with eager calls between."""
    import torch
    import aila_amd as A
    D, Hq, Hkv, page, lens, new = 128, 8, 2, 16, [9000, 500, 40], [300, 1, 40]
    P = sum(-(-n // page) for n in lens) + 3
    cache, table = _cache(P, Hkv, page, D, 1), _table(lens, page, P, 2)
    max_len, T = table.shape[1] * page, sum(new)
    starts, seq = _i32([0] + [int(x) for x in np.cumsum(new)]), _i32(lens)
    q = torch.randn((T, Hq, D), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(torch.bfloat16)
    size = max(A.gqa_prefill_paged_fp8_workspace_size(T, 3, Hq, Hkv, D, max_len), A.gqa_decode_paged_fp8_workspace_size(3, Hq, Hkv, D, max_len))
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    qd = q[:3].contiguous()
    outs = torch.zeros_like(q), torch.zeros_like(qd)
    calls = (lambda o: A.gqa_prefill_paged_fp8(q, *cache, table, starts, seq, max_len, out=o, workspace=ws),
             lambda o: A.gqa_decode_paged_fp8(qd, *cache, table, seq, max_len, out=o, workspace=ws))
    want = [f(torch.zeros_like(o)).clone() for f, o in zip(calls, outs)]
    graphs = []
    for f, o in zip(calls, outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            f(o)
        graphs.append(g)
    for n in range(3):
        for g, f, o, w in zip(graphs, calls, outs, want):
            o.zero_()
            g.replay()
            eager = f(torch.zeros_like(o))
            torch.cuda.synchronize()
            assert torch.equal(o, w) and torch.equal(eager, w), n


# ------------------------------------------------------------- used together --
class _Server:
    """The step of a serving loop: lengths -> tables and slots -> rows -> attention."""

    def __init__(self, B, Hq, Hkv, D, page, P, mp, cap, layers=2):
        import torch
        import aila_amd as A
        self.A, self.B, self.Hq, self.Hkv, self.D, self.page, self.cap = A, B, Hq, Hkv, D, page, cap
        self.max_len = mp * page
        self.caches = [A.paged_fp8_cache(P, Hkv, page, D) for _ in range(layers)]
        self.table = torch.full((B, mp), -1, dtype=torch.int32, device="cuda")
        self.free, self.count = torch.arange(P, dtype=torch.int32, device="cuda"), _i32([P])
        self.cached, self.new, self.ended = _i32([0] * B), _i32([0] * B), _i32([0] * B)
        self.starts, self.lens, self.slots = _i32([0] * (B + 1)), _i32([0] * B), _i32([0] * cap)
        self.qkv = torch.zeros((layers, cap, Hq + 2 * Hkv, D), dtype=torch.bfloat16, device="cuda")
        self.out = torch.zeros((layers, cap, Hq, D), dtype=torch.bfloat16, device="cuda")
        self.ws = torch.empty(max(A.gqa_decode_paged_fp8_workspace_size(B, Hq, Hkv, D, self.max_len),
                                  A.gqa_prefill_paged_fp8_workspace_size(cap, B, Hq, Hkv, D, self.max_len)), dtype=torch.uint8, device="cuda")

    def step(self, decode):
        A = self.A
        A.kv_pages_release(self.ended, self.table, self.free, self.count)
        A.kv_pages_reserve(self.cached, self.new, self.table, self.free, self.count, self.page, self.slots, self.starts, self.lens)
        for i, c in enumerate(self.caches):
            q, k, v = self.qkv[i].split([self.Hq, self.Hkv, self.Hkv], 1)
            A.kv_append_paged_fp8(k, v, *c, self.slots)
            if decode:      # one token each: the batch's rows are the requests
                A.gqa_decode_paged_fp8(q[:self.B], *c, self.table, self.lens, self.max_len, out=self.out[i, :self.B], workspace=self.ws)
            else:
                A.gqa_prefill_paged_fp8(q, *c, self.table, self.starts, self.lens, self.max_len, out=self.out[i], workspace=self.ws)
        # the lengths of the next step, on the device too
        self.cached.copy_(self.lens)

    def check(self, decode):
        starts, lens = self.starts.tolist(), self.lens.tolist()
        for i, c in enumerate(self.caches):
            q = self.qkv[i, :, :self.Hq]
            rows = range(self.B + 1) if decode else starts
            _check(self.out[i], q, c, self.table, rows, lens, self.max_len, 2.0 ** -16 if decode else 2.0 ** -8)

    def fill(self, seed):
        import torch
        self.qkv.copy_(torch.randn(self.qkv.shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda"))


def test_serving_steps():
    """Prompts, decodes, an ended request whose row takes a new prompt, the whole
    cache against what was appended: the values that the bf16 entry points give
    on the rows read back are the 8-bit entry points' results."""
    import torch
    import aila_amd as A
    s = _Server(B=4, Hq=8, Hkv=2, D=128, page=16, P=60, mp=20, cap=128)
    s.new.copy_(_i32([40, 1, 0, 75]))
    s.fill(1)
    s.step(False)
    s.check(False)
    for n in range(20):
        s.new.copy_(_i32([1, 1, 1, 1]))
        s.ended.zero_()
        if n == 9:
            s.ended[1] = 1
            s.cached[1], s.new[1] = 0, 50
        s.fill(10 + n)
        s.step(n != 9)
        s.check(n != 9)
    lens, table = s.lens.tolist(), s.table.tolist()
    assert lens == [60, 60, 20, 95]
    kc = torch.zeros((4, 2, 128, 128), dtype=torch.bfloat16, device="cuda")
    vc = torch.zeros_like(kc)
    for b in range(4):
        slots = [table[b][r // 16] * 16 + r % 16 for r in range(lens[b])]
        k, v = A.kv_read_paged_fp8(*s.caches[1], _i32(slots))
        kc[b, :, :lens[b]], vc[b, :, :lens[b]] = k.transpose(0, 1), v.transpose(0, 1)
    q = s.qkv[1, :4, :8].contiguous()
    want = A.gqa_decode(q, kc, vc, 128, seq_lens=s.lens)
    # both round to bf16 what 64 bits would give within a little: two steps apart at most
    assert ((want.double() - s.out[1, :4].double()).abs() <= 2.0 ** -7 * want.double().abs() + 1e-3 * want.double().abs().max()).all()


@pytest.mark.parametrize("decode", [True, False])
def test_captured_step_replays(decode):
    """A whole step in one graph: its lengths, tables and slots live on the device,
    so each replay is the next step. Eager work runs between the replays."""
    import torch
    s, e = (_Server(B=3, Hq=8, Hkv=2, D=64, page=16, P=40, mp=12, cap=64) for _ in range(2))
    for x in (s, e):
        x.new.copy_(_i32([20, 7, 1]))
        x.fill(1)
        x.step(False)
        x.new.copy_(_i32([1, 1, 1] if decode else [2, 1, 5]))
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    saved = [t.clone() for t in (s.cached, s.table, s.free, s.count)] + [t.clone() for c in s.caches for t in (c[0].view(torch.uint8), c[1].view(torch.uint8), c[2], c[3])]
    with torch.cuda.graph(g):
        s.step(decode)
    for t, x in zip([s.cached, s.table, s.free, s.count] + [t for c in s.caches for t in (c[0].view(torch.uint8), c[1].view(torch.uint8), c[2], c[3])], saved):
        t.copy_(x)
    for n in range(5):
        for x in (s, e):
            x.fill(40 + n)
        g.replay()
        e.step(decode)
        torch.cuda.synchronize()
        s.check(decode)
        assert torch.equal(s.out, e.out) and torch.equal(s.table, e.table) and torch.equal(s.lens, e.lens) and torch.equal(s.count, e.count), n


def test_on_another_stream():
    import torch
    import aila_amd as A
    kp, vp, ks, vs = _cache(20, 2, 16, 64, 3)
    table, lens = _table([200, 31], 16, 20, 4), [200, 31]
    q = torch.randn((2, 4, 64), device="cuda").to(torch.bfloat16)
    seq = _i32(lens)
    want = A.gqa_decode_paged_fp8(q, kp, vp, ks, vs, table, seq, 208)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    got = A.gqa_decode_paged_fp8(q, kp, vp, ks, vs, table, seq, 208, stream=st)
    k, v = A.kv_read_paged_fp8(kp, vp, ks, vs, seq, stream=st)
    st.synchronize()
    assert torch.equal(got, want)
    k2, v2 = A.kv_read_paged_fp8(kp, vp, ks, vs, seq)
    assert torch.equal(k, k2) and torch.equal(v, v2)


def test_offsets_beyond_32_bits():
    """Pages past 2^32 codes: appended, read back and attended there."""
    import torch
    import aila_amd as A
    H, page, D = 8, 128, 256
    P = (1 << 32) // (H * page * D) + 40
    cache = A.paged_fp8_cache(P, H, page, D)
    L = 300
    table = _i32([[P - 1, 3, P - 2], [P - 9, P - 5, 0]])
    tl = table.tolist()
    slots = [tl[b][r // page] * page + r % page for b in range(2) for r in range(L)]
    g = torch.Generator(device="cuda").manual_seed(8)
    qkv = torch.randn((2 * L, 16 + 2 * H, D), generator=g, device="cuda").to(torch.bfloat16)
    q, k, v = qkv.split([16, H, H], 1)
    A.kv_append_paged_fp8(k, v, *cache, _i32(slots))
    rk, rv = A.kv_read_paged_fp8(*cache, _i32(slots))
    # a code is within half a step (2^-4 of the value; at the block's bottom 2^-10 of the scale, at most amax / 224)
    for got, x in ((rk, k), (rv, v)):
        x = x.double()
        assert ((got.double() - x).abs() <= 2.0 ** -4 * x.abs() + 2.0 ** -10 / 224 * x.abs().max()).all()
    ws = torch.empty(A.gqa_decode_paged_fp8_workspace_size(2, 16, H, D, L), dtype=torch.uint8, device="cuda")
    rows = [L - 1, 2 * L - 1]
    small = [t[[P - 1, 3, P - 2, P - 9, P - 5, 0]] if t.dtype == torch.float32 else t.view(torch.uint8)[[P - 1, 3, P - 2, P - 9, P - 5, 0]].view(t.dtype) for t in cache]
    there = _i32([[0, 1, 2], [3, 4, 5]])
    got = A.gqa_decode_paged_fp8(q[rows].contiguous(), *cache, table, _i32([L, L]), L, workspace=ws)
    assert torch.equal(got, A.gqa_decode_paged_fp8(q[rows].contiguous(), *small, there, _i32([L, L]), L, workspace=ws))
    got = A.gqa_prefill_paged_fp8(q, *cache, table, _i32([0, L, 2 * L]), _i32([L, L]), L)
    assert torch.equal(got, A.gqa_prefill_paged_fp8(q, *small, there, _i32([0, L, 2 * L]), _i32([L, L]), L))
    _check(got[rows], q[rows], tuple(small), there, range(3), [L, L], L, 2.0 ** -8)


def test_cpp_ops():
    """The C++ forms (tests/cpp/test_paged_fp8.cpp)."""
    exe = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "test_paged_fp8")
    assert os.path.exists(exe), "build first: python -c 'import __graft_entry__ as g; g.build()'"
    r = subprocess.run([exe], capture_output=True, text=True, timeout=100)
    print(r.stdout)
    assert r.returncode == 0 and "ALL OK" in r.stdout, r.stdout + r.stderr
