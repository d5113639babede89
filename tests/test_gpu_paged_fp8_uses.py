"""Uses of the 8-bit paged cache that are not a server's ordinary step: nothing to
do, queries that are not numbers, many KV heads, many query heads of one, lengths
above the bound."""
import numpy as np
import pytest

from test_gpu_paged_fp8 import _cache, _check, _i32, _table

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _say(request):
    print(request.node.name, flush=True)


def _attention_ws(A, T, B, Hq, Hkv, D, max_len):
    import torch
    return torch.empty(max(16, A.gqa_prefill_paged_fp8_workspace_size(T, B, Hq, Hkv, D, max_len),
                           A.gqa_decode_paged_fp8_workspace_size(B, Hq, Hkv, D, max_len)), dtype=torch.uint8, device="cuda")


@pytest.mark.parametrize("max_len", [64, 5008])
def test_a_step_without_tokens(max_len):
    """All requests absent or without a new token: nothing is written but the lists
    and, by the decode, the outputs of empty sequences."""
    import torch
    import aila_amd as A
    B, Hq, Hkv, D, page, T = 5, 8, 2, 128, 16, 40
    cache = _cache(9, Hkv, page, D, 1)
    before = [x.clone() for x in cache]
    table = torch.full((B, max_len // page), -1, dtype=torch.int32, device="cuda")
    free, count, slots = _i32(range(9)), _i32([9]), _i32([5] * T)
    starts, lens, _ = A.kv_pages_reserve(_i32([-1, 0, -7, 0, -1]), _i32([1, 0, 0, -1, 0]), table, free, count, page, slots)
    assert starts.tolist() == [0] * 6 and lens.tolist() == [0] * 5 and slots.tolist() == [-1] * T
    assert count.item() == 9 and (table == -1).all()
    qkv = torch.randn((T, Hq + 2 * Hkv, D), device="cuda").to(torch.bfloat16)
    q, k, v = qkv.split([Hq, Hkv, Hkv], 1)
    A.kv_append_paged_fp8(k, v, *cache, slots)
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(cache, before))
    ws = _attention_ws(A, T, B, Hq, Hkv, D, max_len)
    for w in (ws, None):
        out = torch.full((T, Hq, D), 7.0, dtype=torch.bfloat16, device="cuda")
        A.gqa_prefill_paged_fp8(q, *cache, table, starts, lens, max_len, out=out, workspace=w)
        assert (out == 7).all()
        assert not A.gqa_decode_paged_fp8(q[:B], *cache, table, lens, max_len, workspace=w).any()


@pytest.mark.parametrize("D,Hq,Hkv", [(64, 8, 2), (128, 6, 2), (256, 4, 1)])
def test_queries_that_are_not_numbers(D, Hq, Hkv):
    """A query of NaN gives NaN in its own token and head; its neighbours in the
    tile, the wave and the records keep their values."""
    import torch
    import aila_amd as A
    page, lens, new = 16, [700, 90, 40], [45, 1, 2]
    P = sum(-(-n // page) for n in lens) + 1
    cache = _cache(P, Hkv, page, D, 2)
    max_len = 4800
    table = _table(lens, page, P, 3, extra=max_len // page - -(-max(lens) // page))
    starts = [0] + [int(x) for x in np.cumsum(new)]
    q = torch.randn((starts[-1], Hq, D), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(torch.bfloat16)
    q[3, 1, 5], q[44, Hq - 1, 0], q[45, 0, D - 1], q[47, 2] = (float("nan"),) * 4
    want = torch.isnan(q).any(2)
    ws = _attention_ws(A, starts[-1], 3, Hq, Hkv, D, max_len)
    for w in (ws, None):
        got = A.gqa_prefill_paged_fp8(q, *cache, table, _i32(starts), _i32(lens), max_len, workspace=w)
        assert torch.equal(torch.isnan(got).any(2), want) and torch.equal(torch.isnan(got).all(2), want)
        _check(got, q, cache, table, starts, lens, max_len, 2.0 ** -8)
    rows = q[[3, 20, 45]].contiguous()
    rows[1, 0, 0] = float("inf")
    for w in (ws, None):
        for bound in (max_len, 720):      # split, and one workgroup each
            got = A.gqa_decode_paged_fp8(rows, *cache, table, _i32(lens), bound, workspace=w)
            _check(got, rows, cache, table, range(4), lens, bound, 2.0 ** -16)
            assert torch.isnan(got[0, 1]).all() and torch.isnan(got[1, 0]).all() and torch.isnan(got[2, 0]).all()


@pytest.mark.parametrize("D,Hq,Hkv,new,lens", [(64, 300, 300, [3, 1, 40], [3, 50, 300]), (128, 514, 257, [20], [33]), (64, 200, 1, [2, 1, 5], [90, 300, 5]),
                                               (128, 333, 1, [3], [700]), (256, 130, 1, [1, 4], [40, 200])])
def test_many_heads(D, Hq, Hkv, new, lens):
    """More KV heads than CUs, and more query heads of one than a tile has rows;
    rows appended first."""
    import torch
    import aila_amd as A
    page, B, max_len = 16, len(lens), 5008
    P = sum(-(-n // page) for n in lens) + 1
    cache = _cache(P, Hkv, page, D, 2)
    table = _table(lens, page, P, 3, extra=max_len // page - -(-max(lens) // page))
    starts = [0] + [int(x) for x in np.cumsum(new)]
    T, tl = starts[-1], table.tolist()
    qkv = torch.randn((T, Hq + 2 * Hkv, D), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(torch.bfloat16)
    q, k, v = qkv.split([Hq, Hkv, Hkv], 1)
    slots = [tl[b][r // page] * page + r % page for b in range(B) for r in range(lens[b] - new[b], lens[b])]
    A.kv_append_paged_fp8(k, v, *cache, _i32(slots))
    for x, got in zip((k, v), A.kv_read_paged_fp8(*cache, _i32(slots))):
        # the scales of the rows before are at most 2^2: half a step is 2^-4 of a value, or 2^-10 of 2^2
        assert ((got.double() - x.double()).abs() <= 2.0 ** -4 * x.double().abs() + 2.0 ** -8).all()
    ws = _attention_ws(A, T, B, Hq, Hkv, D, max_len)
    last = q[[s - 1 for s in starts[1:]]]
    for w in (ws, None):
        got = A.gqa_prefill_paged_fp8(q, *cache, table, _i32(starts), _i32(lens), max_len, workspace=w)
        _check(got, q, cache, table, starts, lens, max_len, 2.0 ** -8)
        got = A.gqa_decode_paged_fp8(last, *cache, table, _i32(lens), max_len, workspace=w)
        _check(got, last, cache, table, range(B + 1), lens, max_len, 2.0 ** -16)


@pytest.mark.parametrize("D,Hq,Hkv", [(64, 4, 2), (128, 8, 1), (256, 4, 4)])
def test_prefill_of_lengths_above_the_bound(D, Hq, Hkv):
    """A length above max_len counts as max_len, which may end inside a block."""
    import torch
    import aila_amd as A
    page, lens, new = 16, [300, 90, 217], [30, 1, 5]
    P = sum(-(-n // page) for n in lens) + 1
    cache, table = _cache(P, Hkv, page, D, 2), _table(lens, page, P, 3)
    for B in (1, 3):
        starts = [0] + [int(x) for x in np.cumsum(new[:B])]
        q = torch.randn((starts[-1], Hq, D), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(torch.bfloat16)
        for bound in (16, 85, 216, 301):
            for w in (_attention_ws(A, starts[-1], B, Hq, Hkv, D, bound), None):
                got = A.gqa_prefill_paged_fp8(q, *cache, table[:B], _i32(starts), _i32(lens[:B]), bound, workspace=w)
                _check(got, q, cache, table, starts, lens[:B], bound, 2.0 ** -8)
