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
