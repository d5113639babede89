"""GPU parity of what a step with drafted trees adds to the 8-bit paged cache
(prepare_qkv_paged_fp8, gqa_tree_paged_fp8, kv_keep_paged_fp8, kv_pages_trim,
kv_copy_paged_fp8) against plain forms in 64 bits: rows, scales and tables bit for
bit where nothing is computed, else within bounds derived from the roundings."""
import numpy as np
import pytest

import draft_ref as dref
import paged_fp8_ref as ref
from test_gpu_paged_fp8 import _cache, _i32, _table

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _say(request):
    print(request.node.name, flush=True)


def _np(t):
    return t.double().cpu().numpy()


# ---------------------------------------------------------------- prepare ----
# A value is a sum of products of normalised values with a cosine and a sine, `size`
# the sum of their sizes. In fp32: the mean of D squares is off by (D + 2) 2^-24 of
# itself (half of that in the root), root, reciprocal and the two products of a
# normalised value by 5 2^-24, an angle of up to pi by 2^-25 of a turn twice (its
# rounding, times 2 pi), sine and cosine by 2^-22, product and sum by 2 2^-24.
def _prepare_slack(size, D):
    return size * ((D / 2 + 10) * 2.0 ** -24 + 2.0 ** -22 + 2 * np.pi * 2.0 ** -24) + 1e-30


def _check_rows(got, scale, y, slack, slots, page, before):
    """Codes' values `got` [P, H, page, D] and scales after y [T, H, D] went to slots: each value
    lies between the roundings of y - slack and y + slack, under the scale that the largest of
    them asks for. before: a ref.Cache of what was there."""
    t = 0
    while t < len(slots):
        s = slots[t]
        if s < 0:
            t += 1
            continue
        r0, n = s % 16, 1
        while t + n < len(slots) and r0 + n < 16 and slots[t + n] == s + n:
            n += 1
        p, r, blk = s // page, s % page, s % page // 16
        for h in range(got.shape[1]):
            rows, d = y[t:t + n, h], slack[t:t + n, h]
            fine = np.isfinite(rows)
            lo, hi = (ref.scale_exp(float(np.max(np.where(fine, np.maximum(np.abs(rows) + x * d, 0), 0.0)))) for x in (-1, 1))
            if r0:
                old = min(max(int(np.log2(before.scale[p, h, blk])), -100), 119)
                lo, hi = max(lo, old), max(hi, old)
            e = int(np.log2(scale[p, h, blk]))
            assert lo <= e <= hi, (t, h, lo, e, hi)
            with np.errstate(invalid="ignore", over="ignore"):
                low, high = ref.e4m3((rows - d) * 2.0 ** -e), ref.e4m3((rows + d) * 2.0 ** -e)
            g = got[p, h, r:r + n]
            assert np.array_equal(np.isnan(g), ~fine), (t, h)
            assert np.all((g >= low) & (g <= high) | ~fine), (t, h)
            if r0:
                assert np.array_equal(got[p, h, r - r0:r], ref.e4m3(before.val[p, h, r - r0:r] * 2.0 ** (old - e)), equal_nan=True)
        t += n


def _prepare_inputs(T, Hq, Hkv, D, seed, packed, kind="plain"):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    wide = 2 if packed else 1
    x = torch.randn((T, (wide * Hq + 2 * Hkv) * D + 8), generator=g, device="cuda")
    if kind == "wide":
        x *= torch.exp2(torch.randint(-20, 20, (T, 1), generator=g, device="cuda").float())
    if kind == "special":
        x[0::5] = 0
        x[1::7, 5::97] = float("nan")
        x[2::6, 3::61] = float("inf")
    x = x.to(torch.bfloat16)
    q = x[:, :wide * Hq * D].view(T, Hq, wide * D)[..., :D] if not packed else x[:, :2 * Hq * D].unflatten(1, (Hq, 2 * D))[..., :D]
    k, v = (x[:, (wide * Hq + i * Hkv) * D:(wide * Hq + (i + 1) * Hkv) * D].unflatten(1, (Hkv, D)) for i in range(2))
    w = [(1 + 0.3 * torch.randn(D, generator=g, device="cuda")).to(torch.bfloat16) for _ in range(2)]
    return q, k, v, *w


def _runs(T, P, page, seed):
    """Slots of T tokens: runs of several lengths that begin anywhere, some tokens skipped, two runs never in one block."""
    rng = np.random.default_rng(seed)
    slots, blocks = [], list(rng.permutation(P * page // 16))
    while len(slots) < T:
        if rng.random() < 0.15:
            slots.append(-1)
            continue
        n = int(rng.choice([1, 1, 2, 5, 16, 16, 16]))
        r0 = 0 if n == 16 else int(rng.integers(0, 17 - n))
        s = int(blocks.pop()) * 16 + r0
        slots += range(s, s + n)
    return slots[:T]


@pytest.mark.parametrize("D,Hq,Hkv,page,T,rot,packed,kind", [
    (128, 8, 2, 32, 1, 128, False, "plain"), (128, 40, 8, 64, 77, 128, False, "wide"), (256, 16, 4, 16, 130, 64, True, "plain"),
    (64, 32, 8, 16, 41, 16, False, "special"), (64, 3, 1, 48, 300, 64, True, "wide"), (256, 5, 5, 32, 1100, 256, False, "special"),
    (128, 4, 1, 128, 2100, 8, True, "plain"), (128, 9, 3, 16, 33, 0, False, "plain"), (256, 2, 2, 64, 259, 248, False, "wide")])
def test_prepare_matches_the_definition(D, Hq, Hkv, page, T, rot, packed, kind):
    import torch
    import aila_amd as A
    P = -(-3 * T // page) * 3 + 8
    q, k, v, qw, kw = _prepare_inputs(T, Hq, Hkv, D, 7 + T, packed, kind)
    kp, vp, ks, vs = _cache(P, Hkv, page, D, T)
    was_k, was_v = ref.Cache(kp, ks), ref.Cache(vp, vs)
    slots = _runs(T, P, page, T)
    pos = np.random.default_rng(T).integers(0, 1 << 20, T)
    out = A.prepare_qkv_paged_fp8(q, k, v, kp, vp, ks, vs, _i32(slots), _i32(pos.tolist()) if rot else None, q_norm=qw, k_norm=kw if kind != "wide" else None,
                                  rotary_dim=rot, theta=1e6, eps=1e-6)
    y, size = dref.norm_rotate(_np(q), _np(qw), pos[:, None], rot, 1e6, 1e-6)
    tol = 2.0 ** -8 * np.abs(y) + _prepare_slack(size, D) * (1 + 2.0 ** -8)
    got = _np(out)
    fine = np.isfinite(y)
    assert np.array_equal(fine, np.isfinite(got))
    assert np.all(np.abs(got - y)[fine] <= tol[fine])
    y, size = dref.norm_rotate(_np(k), _np(kw) if kind != "wide" else None, pos[:, None], rot, 1e6, 1e-6)
    _check_rows(ref.Cache(kp, ks).val, _np(ks), y, _prepare_slack(size, D), slots, page, was_k)
    was_v.append(_np(v), slots)
    now = ref.Cache(vp, vs)
    used = sorted({s // 16 for s in slots if s >= 0})
    assert np.array_equal(now.scale, was_v.scale)
    # rows behind a run stay as they were, like all else
    assert np.array_equal(now.val, was_v.val, equal_nan=True)
    others = np.ones(P * page // 16, bool)
    others[used] = False
    blocks = others.reshape(P, page // 16)
    same = ref.Cache(kp, ks)
    assert np.array_equal(same.scale[:, 0][blocks], was_k.scale[:, 0][blocks])
    assert np.array_equal(same.val.reshape(P, Hkv, page // 16, 16, D).transpose(0, 2, 1, 3, 4)[blocks],
                          was_k.val.reshape(P, Hkv, page // 16, 16, D).transpose(0, 2, 1, 3, 4)[blocks], equal_nan=True)


def test_prepare_with_streams_and_a_table_of_frequencies():
    import torch
    import aila_amd as A
    T, Hq, Hkv, D, page, rot = 37, 6, 2, 128, 32, 64
    q, k, v, qw, kw = _prepare_inputs(T, Hq, Hkv, D, 3, False)
    cache = _cache(8, Hkv, page, D, 1)
    was = ref.Cache(cache[0], cache[2])
    pos = np.random.default_rng(0).integers(0, 4000, (3, T))
    slots = list(range(16, 16 + T))
    sections = (12, 10, 10)
    for inv in (None, 1.0 / 1e4 ** (np.arange(rot // 2) * 2 / rot)):
        inv32 = None if inv is None else torch.tensor(inv, dtype=torch.float32, device="cuda")
        out = A.prepare_qkv_paged_fp8(q, k, v, *cache, _i32(slots), torch.tensor(pos, dtype=torch.int32, device="cuda"), q_norm=qw, k_norm=kw, rotary_dim=rot,
                                      theta=5e5, eps=1e-5, sections=sections, inv_freq=inv32)
        y, size = dref.norm_rotate(_np(q), _np(qw), dref.streams(pos, sections, rot), rot, 5e5, 1e-5, None if inv is None else _np(inv32))
        assert np.all(np.abs(_np(out) - y) <= 2.0 ** -8 * np.abs(y) + _prepare_slack(size, D) * (1 + 2.0 ** -8))
        y, size = dref.norm_rotate(_np(k), _np(kw), dref.streams(pos, sections, rot), rot, 5e5, 1e-5, None if inv is None else _np(inv32))
        _check_rows(ref.Cache(cache[0], cache[2]).val, _np(cache[2]), y, _prepare_slack(size, D), slots, page, was)


def test_prepare_in_place_and_after_the_reference_calls():
    """q_out may be q; and a step's result is that of the calls it stands for, but for their roundings."""
    import torch
    import aila_amd as A
    T, Hq, Hkv, D, page = 40, 8, 2, 128, 64
    q, k, v, qw, kw = _prepare_inputs(T, Hq, Hkv, D, 11, False)
    q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    a, b = _cache(4, Hkv, page, D, 2), _cache(4, Hkv, page, D, 2)
    slots, pos = _i32(list(range(64, 64 + T))), _i32(list(range(300, 300 + T)))
    want = A.prepare_qkv_paged_fp8(q, k, v, *a, slots, pos, q_norm=qw, k_norm=kw)
    q2, k2 = q.clone(), k.clone()
    A.head_rms_norm(q2, qw, 1e-6)
    A.head_rms_norm(k2, kw, 1e-6)
    A.apply_rope(q2, k2, 300, 128, 1e6)
    A.kv_append_paged_fp8(k2, v, *b, slots)
    assert torch.equal(a[1].view(torch.uint8), b[1].view(torch.uint8)) and torch.equal(a[3], b[3])
    # bf16 rounded twice there (2 half steps of the sizes) and once here
    d = (q2.double() - want.double()).abs()
    size = q.double().abs().amax() * 2
    assert float(d.max()) <= float(want.double().abs().max()) * 4 * 2.0 ** -8 and size > 0
    mine = q.clone()
    assert A.prepare_qkv_paged_fp8(mine, k, v, *a, slots, pos, q_norm=qw, k_norm=kw, q_out=mine) is mine
    assert torch.equal(mine, want)


# ------------------------------------------------------------------- tree ----
def _tree_case(D, Hq, Hkv, page, new, before, seed, words=None, pad=3, extra=0.0):
    """Requests of new[b] drafted tokens behind before[b] rows. extra: share of random bits in place of ancestors."""
    import torch
    rng = np.random.default_rng(seed)
    rows = [c + n for c, n in zip(before, new)]
    P = sum(-(-r // page) for r in rows) + 3
    cache = _cache(P, Hkv, page, D, seed)
    T = sum(new) + pad
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = torch.randn((T, Hq, D), generator=g, device="cuda").to(torch.bfloat16)
    seen = []
    for n in new:
        for path in dref.paths(dref.parents(n, rng)) if n else []:
            seen.append([j for j in range(n) if rng.random() < 0.5] if rng.random() < extra else path)
    W = words or max(1, -(-max(new) // 64))
    mask = dref.mask_words(seen + [[]] * pad, W).cuda()
    starts = np.concatenate([[0], np.cumsum(new)]).tolist()
    return q, cache, _table(rows, page, P, seed), _i32(starts), _i32(rows), mask, seen, rows


def _tree_check(out, q, cache, table, new, before, seen, max_len=None, pick=None, words=10**6):
    """Compares the tokens of the requests (all, or some of each) with the plain form."""
    at = 0
    for b, (n, c) in enumerate(zip(new, before)):
        L = c + n if max_len is None else min(c + n, max_len)
        toks = [i for i in range(n) if (pick is None or i in pick or i == n - 1) and i < 64 * words]
        if toks:
            k, held = ref.gather(cache[0], cache[2], table[b].cpu(), max(L, 1))
            v, _ = ref.gather(cache[1], cache[3], table[b].cpu(), max(L, 1))
            k, v, held = k[:, :L], v[:, :L], held[:L]
            want, mag, big = dref.tree_attention(q[[at + i for i in toks]], k, v, held, L - n, n, [seen[at + i] for i in toks])
            tol = ref.attention_tolerance(want, mag, big, L, q.shape[2], 2.0 ** -8)
            got = out[[at + i for i in toks]].double()
            bad = ~((got - want).abs() <= tol)
            assert not bool(bad.any()), (b, int(bad.sum()), float((got - want).abs().max()))
        at += n


@pytest.mark.parametrize("D,Hq,Hkv,page,new,before", [
    (128, 8, 8, 16, [1], [0]), (128, 8, 2, 32, [1], [37]), (64, 4, 2, 16, [5], [0]), (256, 16, 4, 64, [7], [100]),
    (128, 40, 8, 16, [26, 1, 13], [300, 0, 511]), (64, 32, 8, 48, [17, 64, 3], [95, 1000, 16]), (256, 16, 4, 16, [60, 9], [700, 31]),
    (128, 32, 8, 64, [120, 65], [200, 1500]), (256, 24, 1, 128, [33, 2], [257, 64]), (64, 6, 6, 16, [130], [333]), (128, 5, 1, 32, [63, 64, 65], [31, 32, 33]),
    (128, 64, 1, 16, [40, 7], [90, 400]), (256, 8, 8, 32, [0, 4, 0, 9], [50, 20, 0, 33])])
@pytest.mark.parametrize("workspace", [True, False])
def test_tree(D, Hq, Hkv, page, new, before, workspace):
    import torch
    import aila_amd as A
    q, cache, table, starts, lens, mask, seen, rows = _tree_case(D, Hq, Hkv, page, new, before, len(new) + D + sum(new), extra=0.3)
    ws = torch.empty(A.gqa_tree_paged_fp8_workspace_size(q.shape[0], len(new), Hq, Hkv, D, max(rows), mask.shape[1]), dtype=torch.uint8, device="cuda")
    out = torch.full((q.shape[0], Hq, D), 7.0, dtype=torch.bfloat16, device="cuda")
    A.gqa_tree_paged_fp8(q, *cache, table, starts, lens, mask, max(rows), out=out, workspace=ws if workspace else None)
    _tree_check(out, q, cache, table, new, before, seen)
    assert bool((out[sum(new):] == 7.0).all())      # behind the last token


@pytest.mark.parametrize("D,Hq,Hkv,page,new,before", [(128, 40, 8, 16, [26] * 3 + [5] * 9 + [1] * 8, [1200, 3000, 17] + [900 + 53 * i for i in range(17)]),
                                                     (256, 16, 4, 64, [60], [9000]), (64, 32, 8, 128, [100, 3], [5000, 8000]),
                                                     (128, 16, 8, 64, [128, 128], [4000, 2500])])
def test_tree_over_long_contexts(D, Hq, Hkv, page, new, before):
    import torch
    import aila_amd as A
    q, cache, table, starts, lens, mask, seen, rows = _tree_case(D, Hq, Hkv, page, new, before, 5)
    size = A.gqa_tree_paged_fp8_workspace_size(q.shape[0], len(new), Hq, Hkv, D, max(rows), mask.shape[1])
    outs = []
    for ws_bytes in (size, size // 3):
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device="cuda")
        outs.append(A.gqa_tree_paged_fp8(q, *cache, table, starts, lens, mask, max(rows), workspace=ws))
        _tree_check(outs[-1], q, cache, table, new, before, seen, pick={0, 1, 4, 25, 40})


@pytest.mark.parametrize("D,Hq,Hkv,page,new,before", [
    (128, 16, 8, 16, [12, 3, 0, 20], [3000, 5000, 10, 2500]),                     # a split with several requests
    (64, 32, 8, 64, [9], [4000]), (256, 16, 4, 32, [6], [3000]), (128, 5, 1, 16, [7], [1500]),
    (128, 16, 8, 32, [90] + [1] * 7, [5000, 30] + [700 * i for i in range(1, 7)]),   # one wide tree among single tokens: several items
    (256, 16, 4, 64, [70] + [1] * 15, [2500, 0] + [150 * i for i in range(1, 15)]),  # the same, and the merge of many requests
    (64, 64, 2, 16, [3, 4], [9000, 2])])
def test_tree_split_over_workgroups(D, Hq, Hkv, page, new, before):
    """Few columns after long contexts: the items' line, both merges, any workspace; twice the same bits."""
    import torch
    import aila_amd as A
    q, cache, table, starts, lens, mask, seen, rows = _tree_case(D, Hq, Hkv, page, new, before, 7)
    size = A.gqa_tree_paged_fp8_workspace_size(q.shape[0], len(new), Hq, Hkv, D, max(rows), mask.shape[1])
    whole = A.gqa_tree_paged_fp8(q, *cache, table, starts, lens, mask, max(rows))
    _tree_check(whole, q, cache, table, new, before, seen, pick={0, 2, 11, 40})
    for n in (size, size // 2, size // 5):
        ws = torch.full((n,), 0xff, dtype=torch.uint8, device="cuda")        # NaN records where none is written
        a = A.gqa_tree_paged_fp8(q, *cache, table, starts, lens, mask, max(rows), workspace=ws)
        _tree_check(a, q, cache, table, new, before, seen, pick={0, 2, 11, 40})
        b = A.gqa_tree_paged_fp8(q, *cache, table, starts, lens, mask, max(rows), workspace=ws)
        assert torch.equal(a[:sum(new)], b[:sum(new)])


@pytest.mark.parametrize("D,Hq,Hkv,page,new,before", [
    (128, 32, 8, 64, [33], [7000]), (256, 16, 4, 16, [120, 120, 60], [3000, 1000, 2000]), (64, 32, 8, 32, [100, 100, 60], [4000, 100, 900]),   # wide: few tiles, many
    (64, 32, 8, 16, [3] * 6, [5000 - 700 * i for i in range(6)]), (256, 16, 4, 32, [64], [16000]), (64, 8, 2, 64, [1], [60000]),             # narrow: few columns, many
    (128, 16, 8, 16, [64, 0, 1], [9000, 7, 0]), (256, 8, 8, 64, [2, 2], [12000, 0])])
def test_tree_joins(D, Hq, Hkv, page, new, before):
    """Joins of few and of many records of both walks, over records that hold NaN where none is written; masks that leave nothing; twice the same bits."""
    import torch
    import aila_amd as A
    q, cache, table, starts, lens, mask, seen, rows = _tree_case(D, Hq, Hkv, page, new, before, 13)
    mask[sum(new) - 1] = 0          # the last token attends no drafted row, and nothing at all where none is before them
    seen[sum(new) - 1] = []
    size = A.gqa_tree_paged_fp8_workspace_size(q.shape[0], len(new), Hq, Hkv, D, max(rows), mask.shape[1])
    ws = torch.full((size,), 0xff, dtype=torch.uint8, device="cuda")
    outs = [torch.full((q.shape[0], Hq, D), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    for out in outs:
        A.gqa_tree_paged_fp8(q, *cache, table, starts, lens, mask, max(rows), out=out, workspace=ws)
    assert torch.equal(*outs) and bool((outs[0][sum(new):] == 7.0).all())
    _tree_check(outs[0], q, cache, table, new, before, seen, pick={0, 1, 31, 32, 63, 64, 99})


@pytest.mark.parametrize("B,D,Hq,Hkv,most,long", [(1300, 128, 4, 2, 3, 40), (4096, 64, 2, 2, 2, 20), (600, 256, 8, 1, 9, 300), (700, 128, 16, 1, 12, 30)])
def test_trees_of_many_requests(B, D, Hq, Hkv, most, long):
    import torch
    import aila_amd as A
    rng = np.random.default_rng(B)
    new, before = rng.integers(0, most + 1, B).tolist(), rng.integers(0, long, B).tolist()
    q, cache, table, starts, lens, mask, seen, rows = _tree_case(D, Hq, Hkv, 16, new, before, 3)
    ws = torch.empty(A.gqa_tree_paged_fp8_workspace_size(q.shape[0], B, Hq, Hkv, D, max(rows), 1), dtype=torch.uint8, device="cuda")
    out = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device="cuda")
    A.gqa_tree_paged_fp8(q, *cache, table, starts, lens, mask, max(rows), out=out, workspace=ws)
    assert bool(out.isfinite().all()) and bool((out[sum(new):] == 7.0).all())
    at = np.concatenate([[0], np.cumsum(new)])
    for b in rng.choice(B, 40, replace=False):
        a, z = int(at[b]), int(at[b + 1])
        _tree_check(out[a:z], q[a:z], cache, table[b:b + 1], [new[b]], [before[b]], seen[a:z])


def test_tree_that_is_a_chain_is_the_prefill():
    import torch
    import aila_amd as A
    new, before = [9, 1, 30], [70, 200, 0]
    q, cache, table, starts, lens, mask, seen, rows = _tree_case(128, 8, 2, 32, new, before, 3, pad=0)
    chain = dref.mask_words([list(range(i + 1)) for n in new for i in range(n)], 1).cuda()
    a = A.gqa_tree_paged_fp8(q, *cache, table, starts, lens, chain, max(rows))
    b = A.gqa_prefill_paged_fp8(q, *cache, table, starts, lens, max(rows))
    # both round the weights (2^-8) and the output (2^-8 of it)
    assert float((a.double() - b.double()).abs().max()) <= 4 * 2.0 ** -8 * float(b.double().abs().max())


@pytest.mark.parametrize("D,Hq,Hkv,n", [(64, 8, 2, 40), (128, 4, 4, 40), (256, 16, 2, 40), (64, 8, 1, 150), (128, 16, 2, 70), (256, 4, 1, 40)])
def test_masked_drafts_may_hold_anything(D, Hq, Hkv, n):
    """NaN codes in drafted rows reach the tokens that attend them and no others; rows behind the
    last and of pages that are not there reach none; a token that attends nothing gives 0."""
    import torch
    import aila_amd as A
    page, new, before = 16, [n, 6], [50, 0]
    q, cache, table, starts, lens, mask, seen, rows = _tree_case(D, Hq, Hkv, page, new, before, 9, extra=0.2)
    kp, vp, ks, vs = cache
    seen[n] = []                                    # request 1 has no rows before its draft
    seen[n + 1] = [1]
    words = -(-n // 64)
    mask = dref.mask_words(seen + [[]] * 3, words).cuda()
    t = table.cpu().numpy()
    nan_tok = 7
    row = before[0] + nan_tok
    vp.view(torch.uint8)[t[0, row // page], :, row % page, 3] = 0x7f
    vp.view(torch.uint8)[t[0, row // page], 0, row % page, D - 1] = 0xff
    end = rows[0]
    vp.view(torch.uint8)[t[0, end // page], :, end % page:] = 0x7f          # behind the last row
    kp.view(torch.uint8)[t[0, end // page], :, end % page:] = 0x7f
    table[0, 1] = -1                                 # a page that is not there
    table[0, 2] = 10**6
    for ws in (None, torch.empty(A.gqa_tree_paged_fp8_workspace_size(q.shape[0], 2, Hq, Hkv, D, max(rows), words), dtype=torch.uint8, device="cuda")):
        out = A.gqa_tree_paged_fp8(q, *cache, table, starts, lens, mask, max(rows), workspace=ws).double().cpu()
        sees = torch.tensor([nan_tok in s for s in seen[:n]])
        assert 0 < int(sees.sum()) < n
        want = torch.zeros((n, Hq, D), dtype=torch.bool)
        want[sees, :, 3] = True
        want[sees, :Hq // Hkv, D - 1] = True
        assert torch.equal(out[:n].isnan(), want)
        assert bool((out[n] == 0).all()) and bool(out[n + 1:n + 6].isfinite().all())
        clean = vp.clone()
        clean.view(torch.uint8)[t[0, row // page], :, row % page] = 0
        full = A.gqa_tree_paged_fp8(q, kp, clean, ks, vs, table, starts, lens, mask, max(rows), workspace=ws)
        assert torch.equal(full[:n].double().cpu()[~sees], out[:n][~sees])
        _tree_check(full, q, (kp, clean, ks, vs), table, new, before, seen)
        k, held = ref.gather(kp, ks, table[0].cpu(), rows[0])
        assert int((~held).sum()) == 2 * page


def test_tree_of_refused_requests_and_loose_bounds():
    import torch
    import aila_amd as A
    D, Hq, Hkv, page, new, before = 128, 8, 2, 16, [5, 6, 70, 2], [40, 0, 99, 300]
    q, cache, table, starts, lens, mask, seen, rows = _tree_case(D, Hq, Hkv, page, new, before, 21, words=1)
    mp = table.shape[1]
    lens[1] = 0                                      # refused: no rows, its output is 0
    out = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device="cuda")
    size = A.gqa_tree_paged_fp8_workspace_size(q.shape[0], 4, Hq, Hkv, D, mp * page, 1)
    for ws in (None, torch.empty(size, dtype=torch.uint8, device="cuda")):
        out.fill_(7.0)
        A.gqa_tree_paged_fp8(q, *cache, table, starts, lens, mask, mp * page, out=out, workspace=ws)
        assert bool((out[5:11] == 0).all())
        # request 2 has more tokens than its mask has bits: those behind are not computed
        assert bool((out[11 + 64:11 + 70] == 7.0).all()) and bool((out[83:] == 7.0).all())
        keep = [0, 2, 3]
        s = [seen[a:a + n] for a, n in zip((0, 5, 11, 81), new)]
        for b in keep:
            a = (0, 5, 11, 81)[b]
            _tree_check(out[a:a + new[b]], q[a:a + new[b]], cache, table[b:b + 1], [new[b]], [before[b]], s[b], words=1)
    # a bound below the lengths cuts them, and moves the draft with it
    out = A.gqa_tree_paged_fp8(q, *cache, table, starts, lens, mask, 90)
    _tree_check(out[81:83], q[81:83], cache, table[3:4], [2], [300], seen[81:83], max_len=90)


@pytest.mark.parametrize("big", [40.0, 4000.0])
def test_tree_of_large_scores(big):
    import torch
    import aila_amd as A
    new, before = [20, 3], [200, 65]
    q, cache, table, starts, lens, mask, seen, rows = _tree_case(128, 8, 2, 16, new, before, 2)
    q = (q.float() * big).to(torch.bfloat16)
    out = A.gqa_tree_paged_fp8(q, *cache, table, starts, lens, mask, max(rows))
    _tree_check(out, q, cache, table, new, before, seen)


def test_tree_scales_over_the_whole_range():
    """Blocks of V from 2^-100 to 2^90 beside each other, blocks of K from 2^-20 to 2^5."""
    import torch
    import aila_amd as A
    new, before = [12], [500]
    q, (kp, vp, ks, vs), table, starts, lens, mask, seen, rows = _tree_case(128, 8, 2, 16, new, before, 4)
    g = torch.Generator(device="cuda").manual_seed(1)
    ks = torch.exp2(torch.randint(-20, 5, ks.shape, generator=g, device="cuda").float())
    for lo, hi in ((-100, -90), (80, 91), (-100, 91)):
        vs = torch.exp2(torch.randint(lo, hi, vs.shape, generator=g, device="cuda").double()).float()
        out = A.gqa_tree_paged_fp8(q, kp, vp, ks, vs, table, starts, lens, mask, max(rows))
        if lo == -100 and hi == -90:
            # the outputs are normal bf16, but a weight times such a scale is flushed below 2^-126: 2^-26 of each
            k, held = ref.gather(kp, ks, table[0].cpu(), rows[0])
            v, _ = ref.gather(vp, vs, table[0].cpu(), rows[0])
            want, mag, big = dref.tree_attention(q[:12], k, v, held, 500, 12, seen)
            tol = ref.attention_tolerance(want, mag, big, rows[0], 128, 2.0 ** -8) + rows[0] * 2.0 ** -26 * (v.abs().max() + want.abs())
            assert bool(((out[:12].double() - want).abs() <= tol).all())
        else:
            _tree_check(out, q, (kp, vp, ks, vs), table, new, before, seen)


# ------------------------------------------------------------------- keep ----
def _same_cache(cache, want_k, want_v, rows=None):
    for pages, scale, want in ((cache[0], cache[2], want_k), (cache[1], cache[3], want_v)):
        got = ref.Cache(pages, scale)
        assert np.array_equal(got.scale, want.scale)
        assert np.array_equal(got.val, want.val, equal_nan=True)


@pytest.mark.parametrize("D,H,page,layers", [(64, 1, 16, 1), (128, 3, 32, 2), (256, 2, 48, 1), (128, 8, 16, 3), (64, 5, 64, 66)])
def test_keep(D, H, page, layers):
    import aila_amd as A
    rng = np.random.default_rng(D + H)
    cached = [0, 5, 16, 31, 33, -1, 47, 60, 7, 100]
    new = [1, 9, 20, 2, 40, 4, 17, 64, 130, 3]
    kept = [dref.paths(dref.parents(n, rng))[-1] for n in new]
    kept[2] = list(range(20))                        # all of them: nothing moves
    kept[7] = list(range(3, 64))                     # a long run, over many blocks
    kept[8] = [0, 1, 2] + list(range(9, 130, 3))
    kept[3] = []
    kept[9] = [0, 1]
    most = max(len(k) for k in kept) + 2
    counts = [len(k) for k in kept]
    rows = [max(c, 0) + n for c, n in zip(cached, new)]
    P = sum(-(-r // page) for r in rows) + 2
    table = _table(rows, page, P, 3)
    caches = [_cache(P, H, page, D, 10 + i) for i in range(layers)]
    want = [(ref.Cache(c[0], c[2]), ref.Cache(c[1], c[3])) for c in caches]
    arr = _i32([k + [-7] * (most - len(k)) for k in kept])
    lens = A.kv_keep_paged_fp8(caches if layers > 1 else caches[0], table, _i32(cached), arr, _i32(counts))
    t = table.cpu().tolist()
    for (wk, wv), c in zip(want, caches):
        w = dref.keep(wk, t, cached, arr.cpu().tolist(), counts, page)
        assert dref.keep(wv, t, cached, arr.cpu().tolist(), counts, page) == w == lens.tolist()
        _same_cache(c, wk, wv)


def test_keep_of_bad_rows():
    """Counts beyond the list and the table, pages and indices out of range: left as they were."""
    import aila_amd as A
    D, H, page, P = 64, 2, 16, 12
    cache = _cache(P, H, page, D, 1)
    wk, wv = ref.Cache(cache[0], cache[2]), ref.Cache(cache[1], cache[3])
    t = [[0, 1, -1], [2, 99, 3], [4, 5, 6], [7, 8, 9], [10, 11, -5]]
    cached, counts = [10, 14, 40, 0, 2**30], [9, 4, 100, 3, 4]
    kept = [[1, 2, 8, 20, 21, 22, 23, 24, 25], [1, 5, 6, 25] + [0] * 5, [1, 2, 3, 4, 5, 6, 7, 9, 11], [2, 50, 2**31 - 1] + [0] * 6, [1] * 9]
    lens = A.kv_keep_paged_fp8([cache], _i32(t), _i32(cached), _i32(kept), _i32(counts))
    want = dref.keep(wk, t, cached, kept, counts, page)
    dref.keep(wv, t, cached, kept, counts, page)
    assert lens.tolist() == want
    _same_cache(cache, wk, wv)


def test_keep_loses_only_to_underflow():
    import torch
    import aila_amd as A
    D, H, page = 128, 1, 16
    kp, vp, ks, vs = _cache(2, H, page, D, 8)
    for s in (ks, vs):
        s[0], s[1] = 2.0 ** -100, 2.0 ** 119
    vp.view(torch.uint8)[1, 0, 3, 5] = 0x7f
    wk, wv = ref.Cache(kp, ks), ref.Cache(vp, vs)
    args = (_i32([[0, 1]]), _i32([4]), _i32([[0, 3, 15]]), _i32([3]))
    A.kv_keep_paged_fp8((kp, vp, ks, vs), *args)
    for w in (wk, wv):
        dref.keep(w, [[0, 1]], [4], [[0, 3, 15]], [3], page)
    _same_cache((kp, vp, ks, vs), wk, wv)
    assert float(ks[0, 0, 0]) == 2.0 ** 119 and bool(vp[0, 0, 6, 5].float().isnan())


# ------------------------------------------------------------------- trim ----
@pytest.mark.parametrize("B,mp,page,seed", [(1, 1, 16, 0), (3, 5, 32, 1), (40, 9, 16, 2), (300, 70, 64, 3), (2048, 3, 16, 4), (5, 1200, 16, 5), (33, 600, 128, 6)])
def test_trim(B, mp, page, seed):
    import aila_amd as A
    rng = np.random.default_rng(seed)
    P = B * mp + 4
    perm = rng.permutation(P).tolist()
    table = np.full((B, mp), -1, np.int32)
    held = rng.random((B, mp)) < rng.choice([0.1, 0.9, 1.0], (B, 1))
    n = int(held.sum())
    table[held] = perm[:n]
    free, count = perm[n:] + [-1] * n, P - n
    lens = [int(rng.choice([-1, 0, 1, page, mp * page, 2**31 - 1, int(rng.integers(0, mp * page + 1))])) for _ in range(B)]
    dt, df, dc = _i32(table.tolist()), _i32(free), _i32([count])
    A.kv_pages_trim(_i32(lens), dt, df, dc, page)
    want = dref.trim(lens, table.tolist(), free, count, page)
    assert dt.cpu().tolist() == want[0] and int(dc) == want[2] and df.tolist()[:want[2]] == want[1][:want[2]]
    A.kv_pages_trim(_i32(lens), dt, df, dc, page)        # again: nothing is left to give
    assert int(dc) == want[2]


def test_trim_with_a_bad_count():
    import aila_amd as A
    t, f, c = _i32([[0, 1, 2], [3, 4, 5]]), _i32([9, 9, 9, 9]), _i32([3])
    A.kv_pages_trim(_i32([16, 0]), t, f, c, 16)
    assert int(c) == 4 and f.tolist() == [9, 9, 9, 1] and t.tolist() == [[0, -1, -1], [-1, -1, -1]]
    t, f, c = _i32([[0, 1, 2]]), _i32([9, 9, 9, 9]), _i32([-5])
    A.kv_pages_trim(_i32([1]), t, f, c, 16)
    assert int(c) == 2 and f.tolist()[:2] == [1, 2]


# ------------------------------------------------------------------- copy ----
@pytest.mark.parametrize("D,H,page,layers", [(64, 1, 16, 1), (128, 3, 32, 2), (256, 4, 64, 1), (128, 8, 128, 3), (64, 2, 48, 65)])
def test_copy(D, H, page, layers):
    import aila_amd as A
    rows = [200, 200, 200, 17, 64, 1, 5, 100, 100]
    P = sum(-(-r // page) for r in rows) + 2
    table = _table(rows, page, P, 3)
    table[8, 0] = P                                   # a page out of range: skipped
    src, dst, lens = [0, 0, 3, 5, 7, -1, 4, 0, 4], [1, 2, 4, 6, 8, 3, 9, 99, 4], [200, 129, 17, 1, 100, 5, 5, 5, 60]
    caches = [_cache(P, H, page, D, 20 + i) for i in range(layers)]
    want = [(ref.Cache(c[0], c[2]), ref.Cache(c[1], c[3])) for c in caches]
    A.kv_copy_paged_fp8(caches if layers > 1 else caches[0], table, _i32(src), _i32(dst), _i32(lens), 190)
    t = table.cpu().tolist()
    for (wk, wv), c in zip(want, caches):
        for w in (wk, wv):
            dref.copy(w, t, src, dst, lens, 190, page)
        _same_cache(c, wk, wv)
