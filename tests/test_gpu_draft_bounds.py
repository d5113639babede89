"""Drafted trees on the 8-bit paged cache where their kernels can go wrong: blocks that
nobody attends, values that are not finite, each walk at its borders, roundings."""
import numpy as np
import pytest

import draft_ref as dref
import paged_fp8_ref as ref
from test_gpu_drafts import _np, _prepare_inputs, _prepare_slack, _tree_case, _tree_check
from test_gpu_paged_fp8 import _cache, _i32, _table

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _say(request):
    print(request.node.name, flush=True)


def _workspace(q, cache, new, max_len, mask):
    import torch
    import aila_amd as A
    size = A.gqa_tree_paged_fp8_workspace_size(q.shape[0], len(new), q.shape[1], cache[0].shape[1], q.shape[2], max_len, mask.shape[1])
    return torch.full((size,), 0xff, dtype=torch.uint8, device="cuda")


def _walked_as_prompt(ws, new, rows, group, D, words, max_len=1 << 30):
    """Whether the call that used `ws` took the wide walk: it leaves there the key tiles of each
    request's tiles of 128 query rows, 8 more each, summed up."""
    import torch
    keys, units = 32 if D == 256 else 64, [0]
    for n, r in zip(new, rows):
        tiles = -(-min(n, 64 * words) * group // 128)
        units.append(units[-1] + tiles * (8 + max(1, -(-min(r, max_len) // keys))))
    return ws[:4 * len(units)].view(torch.int32).tolist() == units


# ---------------------------------------------------- blocks that nobody attends ----
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("D,Hq,Hkv", [(64, 16, 2), (128, 16, 2), (256, 16, 2)])
def test_blocks_that_nobody_attends_may_have_any_scale(D, Hq, Hkv, wide):
    """A block of drafted rows that all masks leave out: no scale of it, as of a pool that was filled
    with zeros or not at all, reaches an output."""
    import torch
    import aila_amd as A
    page, new, before = 32, [60, 3], [36, 1000]
    q, cache, table, starts, lens, mask, seen, rows = _tree_case(D, Hq, Hkv, page, new, before, 31)
    # rows 48 .. 63 and 64 .. 79 of request 0, its drafted tokens 12 .. 27 and 28 .. 43
    for i in range(60):
        seen[i] = [j for j in seen[i] if not 12 <= j < 44]
    mask = dref.mask_words(seen + [[]] * 3, 1).cuda()
    kp, vp, ks, vs = cache
    ws = _workspace(q, cache, new, max(rows), mask) if wide else None
    want = A.gqa_tree_paged_fp8(q, *cache, table, starts, lens, mask, max(rows), workspace=ws)[:63].clone()
    assert not wide or _walked_as_prompt(ws, new, rows, Hq // Hkv, D, 1)
    _tree_check(want, q, cache, table, new, before, seen, pick={0, 11, 30, 59})
    t = table.tolist()[0]
    for k_bad, v_bad in ((0.0, 1.0), (1.0, 0.0), (0.0, 0.0), (float("nan"), 1.0), (1.0, float("nan")), (float("inf"), float("inf")), (-1.0, -4.0), (1e-45, 3e38)):
        for p, blk in ((t[1], 1), (t[2], 0)):
            ks[p, :, blk], vs[p, :, blk] = k_bad, v_bad
        out = A.gqa_tree_paged_fp8(q, kp, vp, ks, vs, table, starts, lens, mask, max(rows), workspace=ws)
        assert torch.equal(out[:63], want), (k_bad, v_bad)


# ------------------------------------------------------------- prepare's roundings ----
def test_prepare_divides_as_the_definition():
    """Rows of +-s, whose root is s: x / root is +-1, and times a weight it is a tie between two codes. A
    product with the rounded reciprocal falls short of it for these s."""
    import torch
    import aila_amd as A
    s = [x for x in range(1, 257) if np.float32(x) * (np.float32(1) / np.float32(x)) != 1]
    assert len(s) > 10
    for D in (64, 128, 256):
        page, H = 16, 2
        P = -(-len(s) // page)
        sign = 1 - 2 * torch.randint(0, 2, (len(s), H, D), generator=torch.Generator().manual_seed(D)).double()
        k = (torch.tensor(s).double()[:, None, None] * sign).to(torch.bfloat16).cuda()
        w = (1 + (2 * (torch.arange(D) % 8) + 1) / 16).double()
        cache = A.paged_fp8_cache(P, H, page, D)
        q = A.prepare_qkv_paged_fp8(k, k, k, *cache, torch.arange(len(s), dtype=torch.int32, device="cuda"), None, q_norm=w.to(torch.bfloat16).cuda(),
                                    k_norm=w.to(torch.bfloat16).cuda(), rotary_dim=0, eps=0.0)
        y = (sign * w).numpy()
        assert np.array_equal(q.double().cpu().numpy(), y)
        got = ref.Cache(cache[0], cache[2])
        e = ref.scale_exp(float(np.abs(y).max()))
        assert np.all(got.scale.reshape(P, H)[:len(s) // page] == 2.0 ** e)
        rows = got.val.transpose(0, 2, 1, 3).reshape(P * page, H, D)[:len(s)]
        assert np.array_equal(rows, ref.e4m3(y * 2.0 ** -e)), D


def test_prepare_turns_as_the_definition():
    """Rows of ones turned by angles at which cos - sin or sin + cos comes closest to a border between two
    codes, but no closer than cosine, sine and their sum, each rounded to fp32, can cross: half a unit of
    each, and what the angle (2^20 radians in fp64) and the series leave, 2e-9."""
    import torch
    import aila_amd as A
    D, theta = 128, 1e6
    f = theta ** (-2.0 * np.arange(D // 2) / D)

    def values(pos, freq, m):
        """y, and the distance to the next border less what the roundings may take."""
        a = pos * freq
        c, s = m.cos(a), m.sin(a)
        out = []
        for y in (c - s, s + c):
            v = y.abs() if m is torch else np.abs(y)
            half = [m.exp2(m.floor(m.log2(x)) - 24) for x in (c.abs(), s.abs(), v)] if m is torch else [
                np.exp2(np.floor(np.log2(x)) - 24) for x in (np.abs(c), np.abs(s), v)]
            unit = m.exp2(m.floor(m.log2(v * 256)) - 3) / 256
            part = v / unit
            slack = half[0] + half[1] + half[2] + 2e-9
            out.append((y, (part - m.floor(part) - 0.5) * unit, slack))
        return out

    hits = []
    for j in range(0, D // 2):
        pos = torch.arange(1, 1 << 20, dtype=torch.float64, device="cuda")
        for which, (y, d, slack) in enumerate(values(pos, float(f[j]), torch)):
            near = ((d.abs() > slack * 1.01) & (d.abs() < slack * 1.35) & (y.abs() > 2.0 ** -6)).nonzero().view(-1)
            hits += [(int(pos[i]), j, which) for i in near.tolist()]
    hits = [h for h in hits if (lambda x: abs(x[1]) > x[2])(values(float(h[0]), f[h[1]], np)[h[2]])]
    assert len(hits) > 60
    n = len(hits)
    page, P = 16, -(-n // 16)
    cache = A.paged_fp8_cache(P, 1, page, D)
    one = torch.ones((n, 1, D), dtype=torch.bfloat16, device="cuda")
    pos = torch.tensor([h[0] for h in hits], dtype=torch.int32, device="cuda")
    A.prepare_qkv_paged_fp8(one, one, one, *cache, torch.arange(n, dtype=torch.int32, device="cuda"), pos, theta=theta, eps=0.0)
    got = ref.Cache(cache[0], cache[2])
    assert np.all(got.scale == 2.0 ** -8)
    rows = got.val.transpose(0, 2, 1, 3).reshape(P * page, D)
    wrong = [(p, j, which) for i, (p, j, which) in enumerate(hits)
             if rows[i, j + which * (D // 2)] != ref.e4m3(np.float64(values(float(p), f[j], np)[which][0] * 256))]
    assert not wrong, (len(wrong), n, wrong[:5])


@pytest.mark.parametrize("D,Hq,Hkv,page,T,rot", [(64, 32, 8, 16, 11400, 32), (128, 32, 8, 64, 5700, 128), (256, 16, 4, 32, 5650, 64), (128, 40, 3, 48, 7000, 64)])
def test_prepare_of_long_prompts_is_that_of_their_parts(D, Hq, Hkv, page, T, rot):
    """Above 120 MiB rows and queries are a launch each: bit for bit what calls of fewer tokens give, cut
    where a block of 16 ends. Gates between the queries, three streams of positions, skipped tokens."""
    import torch
    import aila_amd as A
    assert T * D * (4 * Hq + 6 * Hkv) > 120 << 20
    q, k, v, qw, kw = _prepare_inputs(T, Hq, Hkv, D, 50, True)
    assert q.stride(1) == 2 * D
    rng = np.random.default_rng(T)
    P = -(-T // page) + 4
    caches = [_cache(P, Hkv, page, D, 51) for _ in range(2)]
    # three requests, whose rows begin inside a block; some tokens of no row; a last block alone
    slots = np.concatenate([np.arange(5, 1000), [-1] * 7, np.arange(1013, T - 40), [-1] * 40, [T + page + 3]])[:T]
    slots = np.concatenate([slots, np.full(T - len(slots), -1)])
    slots[[300, 2000, 2001]] = -1                       # and holes in a run
    slots[301:304] = -1                                 # up to the next block: two runs may not meet in one
    for i in (300, 2000):
        j = i
        while slots[j] < 0 or slots[j] % 16:
            slots[j] = -1
            j += 1
    pos = torch.tensor(rng.integers(0, 1 << 20, (3, T)), dtype=torch.int32, device="cuda")
    sections = (rot // 2 - 2 * (rot // 6), rot // 6, rot // 6)
    st = torch.tensor(slots, dtype=torch.int32, device="cuda")

    def run(cache, a, z):
        return A.prepare_qkv_paged_fp8(q[a:z], k[a:z], v[a:z], *cache, st[a:z].contiguous(), pos[:, a:z].contiguous(), q_norm=qw, k_norm=kw, rotary_dim=rot,
                                       theta=1e6, eps=1e-6, sections=sections)
    whole = run(caches[0], 0, T)
    cuts, at = [0], 0
    for size in (1, 200, 700, 1500):                    # all four lengths of a workgroup's tile
        at += size
        while slots[at] >= 0 and slots[at] % 16:
            at += 1
        cuts.append(at)
    while cuts[-1] < T:
        at = min(cuts[-1] + 3000, T)
        while at < T and slots[at] >= 0 and slots[at] % 16:
            at += 1
        cuts.append(at)
    assert max(z - a for a, z in zip(cuts, cuts[1:])) * D * (4 * Hq + 6 * Hkv) < 120 << 20
    parts = torch.cat([run(caches[1], a, z) for a, z in zip(cuts, cuts[1:])])
    assert torch.equal(whole, parts)
    for x, y in zip(*caches):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    used = torch.tensor(sorted({int(s) // 16 for s in slots if s >= 0}), device="cuda")
    fresh = _cache(P, Hkv, page, D, 51)
    blocks = [x.view(torch.uint8).view(P, Hkv, page // 16, 16 * D).transpose(1, 2).reshape(-1, Hkv * 16 * D) for x in (caches[0][0], fresh[0])]
    changed = (blocks[0] != blocks[1]).any(1).nonzero().view(-1)
    assert torch.equal(changed, used)


def test_prepare_is_the_calls_that_it_stands_for():
    """Against head_rms_norm, apply_rope and the append, each value within their roundings: the single calls
    round the normalised value to bf16 and the turned one again, 2^-8 of each term and of the sum, and
    their angle is a product in fp32; then both round to codes, half a step of their scale each."""
    import torch
    import aila_amd as A
    T, Hq, Hkv, page, first = 45, 6, 3, 32, 300
    for D, rot in ((64, 64), (128, 128), (256, 64)):
        q, k, v, qw, kw = _prepare_inputs(T, Hq, Hkv, D, 12, False)
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
        a, b = ([x.clone() for x in _cache(4, Hkv, page, D, 2)] for _ in range(2))
        at = list(range(16, 16 + T))
        slots, pos = _i32(at), _i32(list(range(first, first + T)))
        out = A.prepare_qkv_paged_fp8(q, k, v, *a, slots, pos, q_norm=qw, k_norm=kw, rotary_dim=rot, theta=1e6, eps=1e-6)
        q2, k2 = q.clone(), k.clone()
        A.head_rms_norm(q2, qw, 1e-6)
        A.head_rms_norm(k2, kw, 1e-6)
        A.apply_rope(q2, k2, first, rot, 1e6)
        A.kv_append_paged_fp8(k2, v, *b, slots)
        assert torch.equal(a[1].view(torch.uint8), b[1].view(torch.uint8)) and torch.equal(a[3], b[3])

        def bound(x, w):
            """The definition, and how far the single calls may be from it."""
            y, size = dref.norm_rotate(_np(x), _np(w), np.arange(first, first + T)[:, None], rot, 1e6, 1e-6)
            half = 2.0 ** -8
            far = half * size + (first + T) * 2.0 ** -22 * size + 2 * _prepare_slack(size, D)
            return y, far + half * (np.abs(y) + far)
        y, far = bound(q, qw)
        assert np.all(np.abs(_np(q2) - y) <= far)
        assert np.all(np.abs(_np(out) - y) <= 2.0 ** -8 * np.abs(y) + _prepare_slack(np.abs(y) + far, D))
        assert np.all(np.abs(_np(out) - _np(q2)) <= far + 2.0 ** -8 * np.abs(y) + _prepare_slack(np.abs(y) + far, D))
        y, far = bound(k, kw)
        rows = [ref.Cache(c[0], c[2]).rows(at) for c in (a, b)]
        scales = [ref.Cache(c[0], c[2]).scale.transpose(0, 2, 1).reshape(-1, Hkv)[[s // 16 for s in at]][:, :, None] for c in (a, b)]
        assert np.all(np.abs(np.log2(scales[0] / scales[1])) <= 1)
        near = [np.maximum(np.abs(x) * 2.0 ** -4, s * 2.0 ** -10) * (1 + 2.0 ** -3) for x, s in zip(rows, scales)]
        assert np.all(np.abs(rows[0] - rows[1]) <= far + near[0] + near[1])
        assert np.all(np.abs(rows[0] - y) <= near[0] + _prepare_slack(np.abs(y) + far, D))


# -------------------------------------------------------------------------- trees ----
def test_tree_merge_of_more_columns_than_a_launch_has_threads():
    """4096 requests of whom one may have 16384 query rows a KV head: a thread for each would be 2^33."""
    import torch
    import aila_amd as A
    B, D, Hq, Hkv, page, words = 4096, 64, 32, 8, 16, 64
    rng = np.random.default_rng(2)
    new, before = rng.integers(0, 3, B).tolist(), rng.integers(0, 20, B).tolist()
    new[7], before[7], new[B - 1], before[B - 1] = 300, 900, 70, 8100
    q, cache, table, starts, lens, mask, seen, rows = _tree_case(D, Hq, Hkv, page, new, before, 3, words=words)
    max_len = table.shape[1] * page                    # above 4096: not a workgroup for each request
    assert max_len > 4096 and q.shape[0] > 4096 and B * Hkv * 4 * 64 * words * D // 4 >= 1 << 32
    ws = _workspace(q, cache, new, max_len, mask)
    out = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device="cuda")
    A.gqa_tree_paged_fp8(q, *cache, table, starts, lens, mask, max_len, out=out, workspace=ws)
    assert not _walked_as_prompt(ws, new, rows, Hq // Hkv, D, words)
    assert bool(out.isfinite().all()) and bool((out[sum(new):] == 7.0).all())
    at = np.concatenate([[0], np.cumsum(new)])
    for b in [7, B - 1] + rng.choice(B, 20, replace=False).tolist():
        a, z = int(at[b]), int(at[b + 1])
        _tree_check(out[a:z], q[a:z], cache, table[b:b + 1], [new[b]], [before[b]], seen[a:z], pick={0, 1, 63, 64, 255, 299}, words=words)


def _pages(table, page, rows):
    """A wider table: its bound on the lengths is what the choice of the walk sees."""
    import torch
    more = -(-rows // page) - table.shape[1]
    return table if more <= 0 else torch.cat([table, torch.full((table.shape[0], more), -1, dtype=torch.int32, device="cuda")], 1).contiguous()


@pytest.mark.parametrize("D,Hq,Hkv,page,B", [(128, 40, 8, 16, 64), (64, 32, 8, 64, 64), (256, 24, 8, 32, 48), (128, 33, 3, 16, 40)])
def test_wide_trees_whose_tiles_stand_in_a_row(D, Hq, Hkv, page, B):
    """Some hundred tiles of query rows, ten and more a workgroup: whole requests one after the other, tiles
    that reuse the keys looked up and loaded for the one before, and their borders."""
    import torch
    import aila_amd as A
    rng = np.random.default_rng(D + B)
    new, before = (120 + rng.integers(0, 9, B)).tolist(), rng.integers(0, 260, B).tolist()
    q, cache, table, starts, lens, mask, seen, rows = _tree_case(D, Hq, Hkv, page, new, before, 40, words=3, extra=0.1)
    table = _pages(table, page, 1200)
    max_len = table.shape[1] * page
    outs = []
    for _ in range(2):
        ws = _workspace(q, cache, new, max_len, mask)
        outs.append(torch.full(q.shape, 7.0, dtype=torch.bfloat16, device="cuda"))
        A.gqa_tree_paged_fp8(q, *cache, table, starts, lens, mask, max_len, out=outs[-1], workspace=ws)
        assert _walked_as_prompt(ws, new, rows, Hq // Hkv, D, 3)
    assert torch.equal(*outs) and bool((outs[0][sum(new):] == 7.0).all())
    tile = 128 // (Hq // Hkv)        # tokens of a tile, the last shared with the next
    at = np.concatenate([[0], np.cumsum(new)])
    for b in rng.choice(B, 12, replace=False):
        a, z = int(at[b]), int(at[b + 1])
        pick = {x for i in range(0, 129, max(1, tile)) for x in (i - 1, i, i + 1)} if tile > 8 else set(range(0, 129, 9))
        _tree_check(outs[0][a:z], q[a:z], cache, table[b:b + 1], [new[b]], [before[b]], seen[a:z], pick=pick, words=3)


@pytest.mark.parametrize("D,Hq,Hkv,page,B", [(128, 32, 8, 64, 100), (64, 16, 2, 16, 150), (256, 16, 4, 32, 70)])
def test_wide_trees_of_many_requests(D, Hq, Hkv, page, B):
    """More requests than a wave has lanes, some without tokens, some without rows before them, some refused."""
    import torch
    import aila_amd as A
    rng = np.random.default_rng(D)
    new, before = rng.integers(30, 100, B), rng.integers(0, 500, B)
    new[rng.random(B) < 0.3] = 0
    new[[0, 1, 63, 64, B - 1]] = [0, 40, 0, 0, 0]
    before[[1, 5, 66]] = 0
    new, before = new.tolist(), before.tolist()
    q, cache, table, starts, lens, mask, seen, rows = _tree_case(D, Hq, Hkv, page, new, before, 41, words=2, extra=0.1)
    table = _pages(table, page, 8000)
    refused = next(b for b in range(10, B) if new[b])
    lens[refused], rows[refused] = 0, 0
    max_len = table.shape[1] * page
    ws = _workspace(q, cache, new, max_len, mask)
    out = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device="cuda")
    A.gqa_tree_paged_fp8(q, *cache, table, starts, lens, mask, max_len, out=out, workspace=ws)
    assert _walked_as_prompt(ws, new, rows, Hq // Hkv, D, 2)
    at = np.concatenate([[0], np.cumsum(new)])
    assert bool(out.isfinite().all()) and bool((out[sum(new):] == 7.0).all())
    assert bool((out[at[refused]:at[refused + 1]] == 0).all())
    for b in {1, 5, 65, 66, B - 2, *rng.choice(B, 12, replace=False).tolist()} - {refused}:
        a, z = int(at[b]), int(at[b + 1])
        _tree_check(out[a:z], q[a:z], cache, table[b:b + 1], [new[b]], [before[b]], seen[a:z], pick={0, 15, 16, 31, 32, 63, 64}, words=2)


@pytest.mark.parametrize("D,Hkv,n,before", [(256, 128, 150, 12000), (256, 128, 120, 30000), (128, 256, 120, 33000), (64, 256, 150, 33000), (256, 256, 240, 11000)])
def test_wide_trees_over_more_keys_than_are_looked_up_at_once(D, Hkv, n, before):
    """One or two workgroups a KV head: a piece of the line spans segments of 11008 rows (D = 256) or 32256,
    the drafts in the last; whole tiles, and one tile cut in two."""
    import torch
    import aila_amd as A
    page = 64
    q, cache, table, starts, lens, mask, seen, rows = _tree_case(D, Hkv, Hkv, page, [n], [before], 42, words=4, extra=0.1)
    ws = _workspace(q, cache, [n], rows[0], mask)
    out = A.gqa_tree_paged_fp8(q, *cache, table, starts, lens, mask, rows[0], workspace=ws)
    assert _walked_as_prompt(ws, [n], rows, 1, D, 4)
    heads = [0, 37, Hkv - 1]
    some = [x[:, heads].contiguous() for x in cache]
    _tree_check(out[:, heads], q[:, heads], some, table, [n], [before], seen, pick={0, 5, 31, 64, 100, 127, 128, 200}, words=4)


@pytest.mark.parametrize("D,Hq,Hkv", [(64, 4, 1), (128, 4, 2), (256, 2, 1)])
@pytest.mark.parametrize("workspace", [False, True])
def test_tree_of_4096_tokens(D, Hq, Hkv, workspace):
    """The widest masks, 64 words, and a request with more tokens than they have bits."""
    import torch
    import aila_amd as A
    new, before = [4096, 4100, 5], [100, 7, 60]
    q, cache, table, starts, lens, mask, seen, rows = _tree_case(D, Hq, Hkv, 64, new, before, 43, words=64, extra=0.002)
    ws = _workspace(q, cache, new, max(rows), mask) if workspace else None
    out = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device="cuda")
    A.gqa_tree_paged_fp8(q, *cache, table, starts, lens, mask, max(rows), out=out, workspace=ws)
    assert not workspace or _walked_as_prompt(ws, new, rows, Hq // Hkv, D, 64)
    _tree_check(out, q, cache, table, new, before, seen, pick={0, 1, 63, 64, 2047, 2048, 4032, 4094, 4095}, words=64)
    assert bool((out[4096 * 2:4096 * 2 + 4] == 7.0).all()) and bool((out[sum(new):] == 7.0).all())


@pytest.mark.parametrize("D,Hq,Hkv", [(64, 16, 2), (128, 16, 2), (256, 16, 2)])
@pytest.mark.parametrize("wide", [False, True])
def test_tree_of_nan_keys_and_queries(D, Hq, Hkv, wide):
    """NaN in a drafted key reaches the tokens that attend it, of its KV head; NaN and infinity in a query
    its own output; a NaN key before the draft all of that head."""
    import torch
    import aila_amd as A
    page, new, before, G = 32, [60, 3], [36, 1000], Hq // Hkv
    q, cache, table, starts, lens, mask, seen, rows = _tree_case(D, Hq, Hkv, page, new, before, 44, extra=0.3)
    kp = cache[0]
    ws = _workspace(q, cache, new, max(rows), mask) if wide else None

    def run(x):
        return A.gqa_tree_paged_fp8(x, *cache, table, starts, lens, mask, max(rows), workspace=ws)[:63].clone()
    want = run(q)
    assert not wide or _walked_as_prompt(ws, new, rows, G, D, 1)
    t = table.tolist()
    bad = q.clone()
    bad[3, 2, 5], bad[30, Hq - 1, D - 1], bad[61, 0, 0] = float("nan"), float("inf"), float("-inf")
    got = run(bad)
    nan = torch.zeros((63, Hq), dtype=torch.bool, device="cuda")
    nan[3, 2] = nan[30, Hq - 1] = nan[61, 0] = True
    assert torch.equal(got.isnan(), nan[:, :, None].expand(got.shape)) and torch.equal(got[~nan], want[~nan])
    row = before[0] + 7
    held = kp.view(torch.uint8)[t[0][row // page], 1, row % page, 9].clone()
    kp.view(torch.uint8)[t[0][row // page], 1, row % page, 9] = 0x7f
    got = run(q)
    nan = torch.zeros((63, Hq), dtype=torch.bool, device="cuda")
    nan[:60, G:] = torch.tensor([7 in s for s in seen[:60]], device="cuda")[:, None]
    assert 0 < int(nan.sum()) < 60 * G
    assert torch.equal(got.isnan(), nan[:, :, None].expand(got.shape)) and torch.equal(got[~nan], want[~nan])
    kp.view(torch.uint8)[t[0][row // page], 1, row % page, 9] = held
    kp.view(torch.uint8)[t[1][500 // page], 0, 500 % page, 0] = 0xff
    got = run(q)
    nan = torch.zeros((63, Hq), dtype=torch.bool, device="cuda")
    nan[60:, :G] = True
    assert torch.equal(got.isnan(), nan[:, :, None].expand(got.shape)) and torch.equal(got[~nan], want[~nan])


# --------------------------------------------------------------------------- keep ----
@pytest.mark.parametrize("D,H,page,B,layers", [(64, 13, 16, 40, 5), (128, 11, 32, 40, 10), (256, 9, 16, 50, 5), (128, 1, 16, 300, 8), (256, 16, 64, 20, 8)])
def test_keep_of_many_is_that_of_each_layer(D, H, page, B, layers):
    """Many requests and layers, where a wave of D = 64 or 128 takes four heads (the last of them doubled where
    the heads are no multiple), against a call for each layer, where it takes one."""
    import torch
    import aila_amd as A
    assert B * layers * (-(-H // 2)) > (2000 if D == 128 else 1000) >= B * (-(-H // 2))
    rng = np.random.default_rng(D + H)
    cached, new = rng.integers(0, 70, B).tolist(), rng.integers(1, 60, B).tolist()
    cached[3], new[4] = -1, 1
    kept = [dref.paths(dref.parents(n, rng))[int(rng.integers(0, n))] if rng.random() < 0.7 else sorted(rng.choice(n, int(rng.integers(0, n + 1)), replace=False).tolist())
            for n in new]
    counts, most = [len(x) for x in kept], max(len(x) for x in kept) + 1
    rows = [max(c, 0) + n for c, n in zip(cached, new)]
    P = sum(-(-r // page) for r in rows) + 2
    table = _table(rows, page, P, 3)
    caches = [_cache(P, H, page, D, 60 + i) for i in range(layers)]
    single = [[x.clone() for x in c] for c in caches]
    arr = _i32([x + [-1] * (most - len(x)) for x in kept])
    lens = A.kv_keep_paged_fp8(caches, table, _i32(cached), arr, _i32(counts))
    for c in single:
        assert torch.equal(lens, A.kv_keep_paged_fp8(c, table, _i32(cached), arr, _i32(counts)))
    assert lens.tolist() == [c + n if c >= 0 else c for c, n in zip(cached, counts)]
    for c, s, i in zip(caches, single, range(layers)):
        for x, y in zip(c, s):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8)), i
    was = _cache(P, H, page, D, 60)
    assert not torch.equal(was[0].view(torch.uint8), caches[0][0].view(torch.uint8))
    # and the first layer against the plain form, some of its requests
    want = ref.Cache(was[0], was[2])
    some = [b for b in range(B) if b % 7 == 0]
    t = table.cpu().tolist()
    dref.keep(want, [t[b] for b in some], [cached[b] for b in some], [arr.cpu().tolist()[b] for b in some], [counts[b] for b in some], page)
    got = ref.Cache(caches[0][0], caches[0][2])
    pages = [p for b in some for p in t[b] if p >= 0]
    assert np.array_equal(got.val[pages], want.val[pages], equal_nan=True) and np.array_equal(got.scale[pages], want.scale[pages])
