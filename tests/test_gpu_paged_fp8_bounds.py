"""The 8-bit paged cache under a length bound far above the lengths, as a captured
step of a server has it: decode then splits and joins records whatever the
lengths are, prefill's key runs are mostly empty. And page tables of more entries
than the planning workgroup keeps on the chip."""
import numpy as np
import pytest

import paged_fp8_ref as ref
from test_gpu_paged_fp8 import F8_NAN, LENS, _cache, _check, _i32, _reserve_both, _table

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _say(request):
    print(request.node.name, flush=True)


def _split_decode(q, cache, table, lens, max_len, ws):
    """A decode that has to have split: its unit counts stand in the workspace."""
    import torch
    import aila_amd as A
    ws.fill_(0xEE)
    got = A.gqa_decode_paged_fp8(q, *cache, table, _i32(lens), max_len, workspace=ws)
    units = [max(1, -(-min(max(n, 0), max_len) // 128)) for n in lens]
    assert ws[:4 * (len(lens) + 1)].view(torch.int32).tolist() == [0] + [int(x) for x in np.cumsum(units)]
    return got


def _workspaces(B, Hq, Hkv, D, max_len):
    """All the bytes that help, a seventh of them, and the least."""
    import torch
    import aila_amd as A
    size = A.gqa_decode_paged_fp8_workspace_size(B, Hq, Hkv, D, max_len)
    G = Hq // Hkv
    chunks = -(-G // 16)
    least = -(-4 * (B + 1) // 256) * 256 + 2 * 2 * -(-G // chunks) * (D + 4) * 4
    full = torch.empty(size, dtype=torch.uint8, device="cuda")
    return full, full[:max(least, size // 7 // 16 * 16)], full[:least]


@pytest.mark.parametrize("D,Hq,Hkv,page,lens", [
    (64, 2, 2, 16, LENS), (128, 3, 1, 64, LENS), (256, 4, 1, 16, LENS), (64, 16, 1, 16, [513, 0, 64]), (256, 32, 2, 64, [400, 90]),
    (128, 17, 1, 32, [600, 1]), (64, 40, 1, 16, [260]), (256, 33, 1, 16, [150, 500]), (64, 10, 2, 48, [1290, 3, 0, 4096]), (256, 8, 4, 32, [2049, 0, 700])])
def test_split_decode_of_short_sequences(D, Hq, Hkv, page, lens):
    import torch
    B = len(lens)
    P = sum(-(-n // page) for n in lens) + 3
    cache = _cache(P, Hkv, page, D, D + Hq)
    max_len = 9000 // page * page
    table = _table(lens, page, P, D + page, extra=max_len // page - -(-max(lens) // page))
    g = torch.Generator(device="cuda").manual_seed(Hq)
    q = torch.randn((B, Hq + 3, D), generator=g, device="cuda").to(torch.bfloat16)[:, :Hq]
    for ws in _workspaces(B, Hq, Hkv, D, max_len):
        _check(_split_decode(q, cache, table, lens, max_len, ws), q, cache, table, range(B + 1), lens, max_len, 2.0 ** -16)


@pytest.mark.parametrize("B,D,Hq,Hkv", [(130, 64, 6, 2), (87, 128, 12, 3), (66, 256, 8, 4), (9, 256, 33 * 29, 29)])
def test_split_decode_of_many_heads(B, D, Hq, Hkv):
    """256 (sequence, head)s and more: the other merge kernel."""
    import torch
    page, rng = 16, np.random.default_rng(B)
    lens = [int(x) for x in rng.integers(0, 500, B)]
    lens[1], lens[B // 2], lens[B - 1] = 1500, 0, 129
    P = sum(-(-n // page) for n in lens) + 3
    cache = _cache(P, Hkv, page, D, B)
    max_len = 4800
    table = _table(lens, page, P, B, extra=max_len // page - -(-max(lens) // page))
    q = torch.randn((B, Hq, D), generator=torch.Generator(device="cuda").manual_seed(B), device="cuda").to(torch.bfloat16)
    some = sorted({0, 1, 2, B // 2, B - 2, B - 1} | {int(x) for x in rng.choice(B, 6)})
    for ws in _workspaces(B, Hq, Hkv, D, max_len)[:2]:
        got = _split_decode(q, cache, table, lens, max_len, ws)
        for b in some:
            _check(got[b:b + 1], q[b:b + 1], cache, table[b:b + 1], [0, 1], lens[b:b + 1], max_len, 2.0 ** -16)


@pytest.mark.parametrize("D,Hq,Hkv", [(64, 8, 2), (128, 4, 4), (256, 16, 2)])
def test_split_decode_masks_what_is_not_held(D, Hq, Hkv):
    """NaN codes and NaN or infinite scales behind the lengths, NaN in attended rows,
    rows without a page or with one outside the pool, in sequences that several
    workgroups walk."""
    import torch
    page, lens = 32, [700, 1045, 33, 40, 1300]
    P = 110
    kp, vp, ks, vs = _cache(P, Hkv, page, D, 5)
    held = [-(-n // page) * page for n in lens]
    max_len = 5024
    table = _table(held, page, P, 6, extra=max_len // page - max(held) // page)
    for b, L in enumerate(lens):
        for r in range(L, held[b]):
            p = int(table[b, r // page])
            for pages, scale in ((kp, ks), (vp, vs)):
                pages.view(torch.uint8)[p, :, r % page] = F8_NAN | (r & 1) << 7
                if r // 16 * 16 >= L:
                    scale[p, :, r % page // 16] = float("nan") if r & 16 else float("inf")
    vp.view(torch.uint8)[int(table[0, 20]), :, 4, 7] = F8_NAN        # row 644 of request 0, dim 7
    vp.view(torch.uint8)[int(table[0, 0]), 1, 9, D - 1] = F8_NAN     # row 9, head 1 alone, the last dim
    kp.view(torch.uint8)[int(table[1, 1]), :, 8, 2] = F8_NAN         # row 40 of request 1
    table[2, 0] = -1
    table[3, 1] = P                                                  # outside the pool
    table[4, 3:9] = -1
    table[4, 31] = 2**31 - 1
    table[3, 2:], table[2, 2:] = P + 9, -2**31                       # behind the lengths
    q = torch.randn((5, Hq, D), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(torch.bfloat16)
    for ws in _workspaces(5, Hq, Hkv, D, max_len):
        got = _split_decode(q, (kp, vp, ks, vs), table, lens, max_len, ws)
        assert torch.isnan(got[0, :, 7]).all() and torch.isnan(got[1]).all() and not torch.isnan(got[2:]).any()
        _check(got, q, (kp, vp, ks, vs), table, range(6), lens, max_len, 2.0 ** -16)


def test_split_decode_beyond_32_bits():
    """Pages past 2^32 codes, walked by several workgroups: the same rows in a small
    pool give the same bits."""
    import torch
    import aila_amd as A
    H, page, D, L = 8, 128, 256, 700
    P = (1 << 32) // (H * page * D) + 40
    cache = A.paged_fp8_cache(P, H, page, D)
    own = [[P - 1, 3, P - 2, P - 7, P - 3, 1], [P - 9, P - 5, 0, P - 11, 2, P - 4]]
    max_len = 20 * page
    table = _i32([x + [-1] * 14 for x in own])
    slots = _i32([own[b][r // page] * page + r % page for b in range(2) for r in range(L)])
    g = torch.Generator(device="cuda").manual_seed(8)
    k, v = torch.randn((2 * L, 2 * H, D), generator=g, device="cuda").to(torch.bfloat16).split([H, H], 1)
    A.kv_append_paged_fp8(k, v, *cache, slots)
    ids = own[0] + own[1]
    small = [t[ids] if t.dtype == torch.float32 else t.view(torch.uint8)[ids].view(t.dtype) for t in cache]
    there = _i32([[0, 1, 2, 3, 4, 5] + [-1] * 14, [6, 7, 8, 9, 10, 11] + [-1] * 14])
    q = torch.randn((2, 16, D), generator=g, device="cuda").to(torch.bfloat16)
    ws = _workspaces(2, 16, H, D, max_len)[0]
    got = _split_decode(q, cache, table, [L, L], max_len, ws)
    assert torch.equal(got, _split_decode(q, small, there, [L, L], max_len, ws))
    _check(got, q, tuple(small), there, range(3), [L, L], max_len, 2.0 ** -16)


@pytest.mark.parametrize("D,Hq,Hkv,new,lens", [
    (64, 8, 2, [3], [3]), (128, 4, 4, [1], [300]), (256, 8, 2, [40], [60]), (128, 16, 2, [40], [700]), (256, 4, 1, [7], [0]),
    (128, 8, 2, [5, 1, 0, 70], [5, 400, 9, 70]), (256, 16, 4, [1, 33, 2], [90, 33, 600]), (64, 4, 1, [2, 20], [0, 257])])
def test_prefill_under_a_loose_bound(D, Hq, Hkv, new, lens):
    """Lengths far below the bound and fewer tokens than rows of q, as a captured
    step has them: runs without a key and tiles without a row."""
    import torch
    import aila_amd as A
    page, B = 16, len(lens)
    P = sum(-(-n // page) for n in lens) + 3
    cache = _cache(P, Hkv, page, D, D + Hq)
    max_len = 30000 // page * page
    table = _table(lens, page, P, D, extra=max_len // page - -(-max(lens) // page))
    starts = [0] + [int(x) for x in np.cumsum(new)]
    T = starts[-1] + 60
    q = torch.randn((T, Hq, D), generator=torch.Generator(device="cuda").manual_seed(Hq), device="cuda").to(torch.bfloat16)
    size = A.gqa_prefill_paged_fp8_workspace_size(T, B, Hq, Hkv, D, max_len)
    for ws in (torch.full((size,), 0xEE, dtype=torch.uint8, device="cuda"), None):
        out = torch.full((T, Hq, D), 7.0, dtype=torch.bfloat16, device="cuda")
        A.gqa_prefill_paged_fp8(q, *cache, table, _i32(starts), _i32(lens), max_len, out=out, workspace=ws)
        _check(out, q, cache, table, starts, lens, max_len, 2.0 ** -8)
        assert (out[starts[-1]:] == 7).all()


@pytest.mark.parametrize("B,new,cap,P", [(70, 1024, 80000, 5000), (70, 1024, 80000, 2000), (70, 1024, 2048, 5000), (70, 1024, 512, 5000),
                                         (900, 100, 100000, 7000)])
def test_reserve_of_more_entries_than_fit_the_chip(B, new, cap, P):
    """More than 4096 table entries to look at, and more pages to take than are
    fetched beforehand; some requests hold pages, some are refused."""
    import aila_amd as A
    page, mp = 16, 70
    rng = np.random.default_rng(B + cap)
    perm = [int(x) for x in rng.permutation(P)]
    cached = [int(x) if b % 3 == 0 else 0 for b, x in enumerate(rng.integers(0, 90, B))]
    fresh = [new - int(x) for x in rng.integers(0, 9, B)]
    fresh[0], fresh[5], cached[7] = 40, -1, -2
    fresh[11] = mp * page + 1                                           # more than its table row
    table, at = [[-1] * mp for _ in range(B)], 0
    for b in range(B):
        for p in range(-(-max(cached[b], 0) // page)):
            table[b][p] = perm[at]
            at += 1
    free, count = perm[at:] + [-9] * at, P - at
    entries = sum(-(-(c + n) // page) - c // page for c, n in zip(cached, fresh) if c >= 0 and n >= 0 and c + n <= mp * page)
    assert entries > 4096
    t1, c1, _, lens, _ = _reserve_both(cached, fresh, table, free, count, page, cap)
    assert cap < 80000 or count - c1 > 1024
    again = _reserve_both(cached, fresh, t1, free, c1, page, cap)
    assert [x for x, n in zip(again[0], lens) if n] == [x for x, n in zip(t1, lens) if n]
    flags = [int(x) for x in rng.integers(0, 2, B)]
    t, f, c = _i32(again[0]), _i32(free), _i32([again[1]])
    A.kv_pages_release(_i32(flags), t, f, c)
    assert (t.tolist(), f.tolist(), c.item()) == ref.release(flags, again[0], free, again[1])


def test_reserve_of_two_pages_each_by_the_small_plan():
    """512 pages to take for 256 requests and 512 tokens: twice the pages that the
    plan of 256 threads fetches beforehand."""
    B, page, P = 256, 16, 600
    perm = [int(x) for x in np.random.default_rng(3).permutation(P)]
    t, count, _, lens, slots = _reserve_both([15] * B, [2] * B, [[-1] * 3 for _ in range(B)], perm, P, page, 512)
    assert count == P - 512 and lens == [17] * B and min(slots) >= 0
