"""Drafted trees on the 8-bit paged cache where their kernels can go wrong: blocks that
nobody attends, values that are not finite, each walk at its borders, roundings."""
import numpy as np
import pytest

import draft_ref as dref
import paged_fp8_ref as ref
from test_gpu_drafts import _tree_case, _tree_check

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
