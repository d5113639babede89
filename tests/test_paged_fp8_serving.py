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
