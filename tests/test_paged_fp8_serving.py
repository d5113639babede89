"""The serving loop over the 8-bit paged cache when its pool runs out: a request
that is refused a page keeps its rows and goes on behind them later."""
import pytest

import paged_fp8_ref as ref


def next_cached(cached, lens):
    """The lengths of the next step, as kv_pages_reserve documents them."""
    return [n if n > 0 else c for c, n in zip(cached, lens)]


def test_lengths_of_a_refused_request():
    """Request 1 fills its pages while none is free, is refused, and is asked for
    again after request 0 has ended: its tokens go behind its rows."""
    page, table, free, count = 16, [[4, -1, -1], [0, 1, -1], [-1, -1, -1]], [9, 9, 9, 9, 9], 0
    cached, new = [15, 32, -1], [1, 1, 1]
    table, count, _, lens, slots = ref.reserve(cached, new, table, free, count, page, 4)
    assert lens == [16, 0, 0] and slots == [4 * 16 + 15, -1, -1, -1]
    # a copy of the lengths would start request 1 again on the page of its first row
    assert ref.reserve(lens, new, table, free, count, page, 4)[4][1] == 0 * 16
    cached = next_cached(cached, lens)
    assert cached == [16, 32, -1]
    assert ref.reserve(cached, [0, 1, 0], table, free, count, page, 4)[3] == [16, 0, 0]       # still no page
    table, free, count = ref.release([1, 0, 0], table, free, count)
    cached[0] = 0
    table, count, _, lens, slots = ref.reserve(cached, [0, 1, 0], table, free, count, page, 4)
    assert lens == [0, 33, 0] and slots == [4 * 16, -1, -1, -1] and table[1] == [0, 1, 4]
    assert next_cached(cached, lens) == [0, 33, -1]


@pytest.mark.gpu
@pytest.mark.parametrize("decode", [False, True])
def test_a_running_request_without_a_page(decode):
    """The whole loop on the device: pages run out under two running requests, which
    are refused for some steps, lose no row, and go on when a third has ended. The
    absent request stays absent."""
    import torch
    import aila_amd as A
    from test_gpu_paged_fp8 import _Server, _check, _i32

    class Tight(_Server):
        def step(self, decode):
            before = self.cached.clone()
            super().step(decode)
            torch.where(self.lens > 0, self.lens, before, out=self.cached)

        def held(self, b, n):
            """Rows [0, n) of request b, K and V of each layer."""
            t = self.table[b].tolist()
            slots = _i32([t[r // self.page] * self.page + r % self.page for r in range(n)])
            return [x for c in self.caches for x in A.kv_read_paged_fp8(*c, slots)]

    # three of 30, 32 and 31 rows hold all six pages
    s = Tight(B=4, Hq=8, Hkv=2, D=64, page=16, P=6, mp=8, cap=128)
    s.cached.copy_(_i32([0, 0, 0, -1]))
    s.new.copy_(_i32([30, 32, 31, 1]))
    s.fill(1)
    s.step(False)
    assert s.cached.tolist() == [30, 32, 31, -1] and s.count.item() == 0
    want = [30, 32, 31]
    seen = 0
    for n in range(6):
        s.ended.zero_()
        if n == 4:         # request 0 ends: its two pages go to the others
            s.ended[0], s.cached[0], want[0] = 1, -1, -1
        s.new.copy_(_i32([1, 1, 1, 1]))
        rows = [s.held(b, want[b]) if want[b] > 0 else None for b in range(3)]
        s.fill(10 + n)
        # one token each where all requests are there: row b of the batch is request b
        one = decode and n < 4
        s.step(one)
        ok = [n < 2, n >= 4, n < 1 or n >= 4]      # 30 + 2, 32 + 0, 31 + 1 rows fit; then a page for each of the two
        want = [w + o if w > 0 else w for w, o in zip(want, ok)]
        assert s.cached.tolist() == want + [-1], n
        assert s.lens.tolist() == [w if o else 0 for w, o in zip(want, ok)] + [0], n
        if one:
            lens = s.lens.tolist()[:3]
            for i, c in enumerate(s.caches):
                _check(s.out[i], s.qkv[i, :, :8], c, s.table, range(4), lens, s.max_len, 2.0 ** -16)
        else:
            s.check(False)
        for b in range(3):
            if rows[b] is None:
                continue
            # a token may raise its block's scale, and the block's rows are rounded again; all others stay
            k = (want[b] - 1) // 16 * 16 if ok[b] else want[b]
            assert all(torch.equal(x[:k], y[:k]) for x, y in zip(rows[b], s.held(b, want[b]))), (n, b)
            seen += k
    assert want == [-1, 34, 34] and seen > 0


@pytest.mark.gpu
@pytest.mark.parametrize("D,max_len", [(64, 96), (128, 4800), (256, 96)])
def test_a_batch_with_idle_requests(D, max_len):
    """Absent and idle requests have no token in the batch, a refused one keeps its
    place: prefill takes the batch as it is, decode its rows gathered by the starts."""
    import torch
    import aila_amd as A
    from test_gpu_paged_fp8 import _cache, _check, _i32, _table
    B, Hq, Hkv, page, P = 8, 8, 2, 16, 40
    held = [50, 33, 20, 16, 0, 45, 31, 12]       # the last idle one's start is the batch's end
    cache = _cache(P, Hkv, page, D, 4)
    table = _table(held, page, P, 5, extra=max_len // page - 4)
    cached, new = _i32([50, -33, 20, 16, 0, 45, 31, 12]), _i32([1, 1, 0, 1, 0, 1, 1, 0])
    count, slots = _i32([0]), _i32([9] * 4)
    starts, lens, _ = A.kv_pages_reserve(cached, new, table, _i32([0] * P), count, page, slots)
    assert starts.tolist() == [0, 1, 1, 1, 2, 2, 3, 4, 4] and lens.tolist() == [51, 0, 20, 0, 0, 46, 32, 12]       # request 3 finds no page
    qkv = torch.randn((4, Hq + 2 * Hkv, D), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(torch.bfloat16)
    q, k, v = qkv.split([Hq, Hkv, Hkv], 1)
    A.kv_append_paged_fp8(k, v, *cache, slots)
    ws = torch.empty(max(A.gqa_decode_paged_fp8_workspace_size(B, Hq, Hkv, D, max_len), A.gqa_prefill_paged_fp8_workspace_size(4, B, Hq, Hkv, D, max_len)),
                     dtype=torch.uint8, device="cuda")
    got = A.gqa_prefill_paged_fp8(q, *cache, table, starts, lens, max_len, workspace=ws)
    _check(got, q, cache, table, starts.tolist(), lens.tolist(), max_len, 2.0 ** -8)
    rows = q[starts[:B].long().clamp(max=3)]
    got = A.gqa_decode_paged_fp8(rows, *cache, table, lens, max_len, workspace=ws)
    _check(got, rows, cache, table, range(B + 1), lens.tolist(), max_len, 2.0 ** -16)
    for b, n in ((0, 51), (5, 46), (6, 32)):      # the rows that the gathered tokens wrote
        at = int(table[b, (n - 1) // page]) * page + (n - 1) % page
        assert slots[starts[b]].item() == at
