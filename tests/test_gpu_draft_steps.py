"""A step with drafted trees as a serving engine runs it: pages -> rows -> attention ->
the accepted path kept -> pages back; forks; captured, on other streams, past 2^32."""
import os
import subprocess

import numpy as np
import pytest

import draft_ref as dref
import paged_fp8_ref as ref
from test_gpu_drafts import _tree_check
from test_gpu_paged_fp8 import _cache, _i32, _table

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _say(request):
    print(request.node.name, flush=True)


class _Engine:
    """Requests that verify a tree each step; what the sampler accepts is an input."""

    def __init__(self, B, Hq, Hkv, D, page, P, mp, cap, most, layers=3, rot=None):
        import torch
        import aila_amd as A
        self.A, self.B, self.Hq, self.Hkv, self.D, self.page, self.P, self.cap, self.most, self.rot = A, B, Hq, Hkv, D, page, P, cap, most, rot
        self.max_len = mp * page
        self.caches = [A.paged_fp8_cache(P, Hkv, page, D) for _ in range(layers)]
        self.table = torch.full((B, mp), -1, dtype=torch.int32, device="cuda")
        self.free, self.count = torch.arange(P, dtype=torch.int32, device="cuda"), _i32([P])
        self.cached, self.new = _i32([0] * B), _i32([0] * B)
        self.starts, self.rows, self.slots, self.pos = _i32([0] * (B + 1)), _i32([0] * B), _i32([0] * cap), _i32([0] * cap)
        self.kept, self.kept_lens, self.lens = _i32([[0] * most] * B), _i32([0] * B), _i32([0] * B)
        self.mask = torch.zeros((cap, 1), dtype=torch.int64, device="cuda")
        self.qkv = torch.zeros((layers, cap, Hq + 2 * Hkv, D), dtype=torch.bfloat16, device="cuda")
        self.norm = [(1 + 0.1 * torch.randn(D, generator=torch.Generator(device="cuda").manual_seed(i), device="cuda")).to(torch.bfloat16) for i in range(2)]
        self.q = torch.zeros((layers, cap, Hq, D), dtype=torch.bfloat16, device="cuda")
        self.out = torch.zeros_like(self.q)
        self.ws = torch.empty(A.gqa_tree_paged_fp8_workspace_size(cap, B, Hq, Hkv, D, self.max_len, 1), dtype=torch.uint8, device="cuda")

    def state(self):
        import torch
        return [self.cached, self.table, self.free, self.count, self.rows, self.lens] + [
            t.view(torch.uint8) if t.dtype != torch.float32 else t for c in self.caches for t in c]

    def draft(self, par, accepted, seed):
        """par: a tree for each request ([]: idle); accepted: the node whose path is kept (-1: none)."""
        import torch
        seen, pos, kept = [], [], []
        cached = self.cached.tolist()
        for b, p in enumerate(par):
            paths = dref.paths(p)
            seen += paths
            pos += [max(cached[b], 0) + len(x) - 1 for x in paths]
            kept.append(paths[accepted[b]] if p and accepted[b] >= 0 else [])
        self.seen = seen
        pad = self.cap - len(seen)
        self.new.copy_(_i32([len(p) for p in par]))
        self.pos.copy_(_i32(pos + [0] * pad))
        self.mask.copy_(dref.mask_words(seen + [[]] * pad, 1))
        self.kept.copy_(_i32([k + [-1] * (self.most - len(k)) for k in kept]))
        self.kept_lens.copy_(_i32([len(k) for k in kept]))
        self.qkv.copy_(torch.randn(self.qkv.shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda"))

    def attend(self):
        A = self.A
        A.kv_pages_reserve(self.cached, self.new, self.table, self.free, self.count, self.page, self.slots, self.starts, self.rows)
        for i, c in enumerate(self.caches):
            q, k, v = self.qkv[i].split([self.Hq, self.Hkv, self.Hkv], 1)
            A.prepare_qkv_paged_fp8(q, k, v, *c, self.slots, self.pos, q_norm=self.norm[0], k_norm=self.norm[1], rotary_dim=self.rot, q_out=self.q[i])
            A.gqa_tree_paged_fp8(self.q[i], *c, self.table, self.starts, self.rows, self.mask, self.max_len, out=self.out[i], workspace=self.ws)

    def commit(self):
        import torch
        A = self.A
        n = torch.where(self.rows > 0, self.kept_lens, torch.zeros_like(self.kept_lens))     # a refused request keeps nothing
        A.kv_keep_paged_fp8(self.caches, self.table, self.cached, self.kept, n, lens=self.lens)
        A.kv_pages_trim(self.lens, self.table, self.free, self.count, self.page)
        self.cached.copy_(self.lens)

    def slots_of(self, b, rows):
        t = self.table.tolist()
        return [t[b][r // self.page] * self.page + r % self.page for r in rows]


def _trees(rng, B, most):
    return [dref.parents(int(rng.integers(1, most + 1)), rng) for _ in range(B)]


@pytest.mark.parametrize("D,Hq,Hkv,page,rot", [(128, 8, 2, 16, 128), (256, 16, 4, 32, 64), (64, 8, 8, 16, 64)])
def test_speculative_steps(D, Hq, Hkv, page, rot):
    """Attention over what the steps before kept, the rows kept, and the pages: nothing lost, nothing held twice."""
    import torch
    B, P, most = 4, 60, 20
    e = _Engine(B, Hq, Hkv, D, page, P, mp=12, cap=90, most=most, rot=rot)
    rng = np.random.default_rng(D)
    for step in range(12):
        par = _trees(rng, B, most)
        if step == 3:
            par[1] = []
        acc = [int(rng.integers(-1 if step % 4 == 2 else 0, len(p))) if p else -1 for p in par]
        e.draft(par, acc, 100 + step)
        before = e.cached.tolist()
        e.attend()
        new = [len(p) for p in par]
        for i, c in enumerate(e.caches):
            _tree_check(e.out[i], e.q[i], c, e.table, new, before, e.seen, pick={0, 1, 5, 13})
        # what the rows stand for before they move
        was = [[e.A.kv_read_paged_fp8(*c, _i32(e.slots_of(b, list(range(before[b])) + [before[b] + k for k in e.kept[b].tolist()[:int(e.kept_lens[b])]]) or [-1]))
                for b in range(B)] for c in e.caches]
        e.commit()
        lens = e.lens.tolist()
        assert lens == [x + int(n) for x, n in zip(before, e.kept_lens.tolist())]
        for c, w in zip(e.caches, was):
            for b in range(B):
                got = e.A.kv_read_paged_fp8(*c, _i32(e.slots_of(b, range(lens[b])) or [-1]))
                for g, x, s in zip(got, w[b], c[2:]):
                    # the same but for what a larger scale of the block flushes: half its smallest step
                    assert float((g.double() - x.double()).abs().max()) <= 2.0 ** -10 * float(s.max())
                    assert float((g != x).double().mean()) < 0.02
        held = sum(-(-n // page) for n in lens)
        t = e.table
        assert int((t >= 0).sum()) == held and int(e.count) == P - held
        pages = torch.cat([t[t >= 0], e.free[:int(e.count)]]).tolist()
        assert sorted(pages) == list(range(P))


def test_a_refused_request_keeps_its_rows():
    B, page = 3, 16
    e = _Engine(B, 4, 2, 64, page, P=6, mp=6, cap=60, most=20)
    rng = np.random.default_rng(5)
    e.draft([dref.parents(18, rng), dref.parents(16, rng), dref.parents(3, rng)], [17, 15, 2], 1)
    e.kept.copy_(_i32([list(range(18)) + [-1] * 2, list(range(16)) + [-1] * 4, [0, 1, 2] + [-1] * 17]))
    e.kept_lens.copy_(_i32([18, 16, 3]))
    e.attend()
    e.commit()
    assert e.lens.tolist() == [18, 16, 3]                            # 2 + 1 + 1 pages of 6
    e.draft([dref.parents(20, rng), dref.parents(20, rng), dref.parents(20, rng)], [19, 19, 19], 2)
    kept = [int(x) for x in e.kept_lens.tolist()]
    e.attend()
    rows = e.rows.tolist()
    assert rows[0] == 38 and rows[1] == 0                            # one page more for the first, two are not there for the second
    e.commit()
    assert e.lens.tolist() == [18 + kept[0], 16, 3 + (kept[2] if rows[2] else 0)]
    assert bool((e.out[0, 20:40] == 0).all())


def test_captured_steps_replay():
    """A whole step in one graph, each replay the next step, with eager steps between."""
    import torch
    g_, e = (_Engine(3, 8, 2, 128, 16, P=50, mp=10, cap=64, most=20, layers=2) for _ in range(2))
    rng = np.random.default_rng(1)
    for x in (g_, e):
        x.draft([dref.parents(9, np.random.default_rng(2))] * 3, [8, 3, 0], 3)
        x.attend()
        x.commit()
    torch.cuda.synchronize()
    saved = [t.clone() for t in g_.state()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        g_.attend()
        g_.commit()
    for t, x in zip(g_.state(), saved):
        t.copy_(x)
    for n in range(5):
        par = _trees(rng, 3, 20)
        acc = [int(rng.integers(0, len(p))) for p in par]
        for x in (g_, e):
            x.draft(par, acc, 50 + n)
        graph.replay()
        e.attend()
        e.commit()
        torch.cuda.synchronize()
        live = sum(len(p) for p in par)
        assert torch.equal(g_.out[:, :live], e.out[:, :live]), n
        for a, b in zip(g_.state(), e.state()):
            assert torch.equal(a, b), n


@pytest.mark.parametrize("D,Hq,Hkv,new,before", [(128, 8, 2, [30, 1, 40], [9000, 500, 40]), (128, 16, 8, [4, 2, 7], [9000, 500, 40]), (256, 8, 2, [60, 2], [3000, 40])])
def test_graphs_that_share_a_workspace_and_streams_that_do_not(D, Hq, Hkv, new, before):
    import torch
    import aila_amd as A
    rng = np.random.default_rng(3)
    rows = [a + b for a, b in zip(new, before)]
    P, B, T = sum(-(-r // 16) for r in rows) + 3, len(new), sum(new)
    cache, table = _cache(P, Hkv, 16, D, 1), _table(rows, 16, P, 2)
    max_len, starts, seq = table.shape[1] * 16, _i32([0] + [int(x) for x in np.cumsum(new)]), _i32(rows)
    q = torch.randn((T, Hq, D), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(torch.bfloat16)
    mask = dref.mask_words([p for n in new for p in dref.paths(dref.parents(n, rng))], 1).cuda()
    one = [_i32([0, new[0]]), _i32([rows[0]]), table[:1].contiguous()]
    size = max(A.gqa_tree_paged_fp8_workspace_size(T, B, Hq, Hkv, D, max_len, 1), A.gqa_tree_paged_fp8_workspace_size(new[0], 1, Hq, Hkv, D, max_len, 1))

    def both(ws, stream=None, out=(None, None)):
        return (A.gqa_tree_paged_fp8(q, *cache, table, starts, seq, mask, max_len, out=out[0], workspace=ws, stream=stream),
                A.gqa_tree_paged_fp8(q[:new[0]], *cache, one[2], one[0], one[1], mask[:new[0]], max_len, out=out[1], workspace=ws, stream=stream))

    ws = [torch.empty(size, dtype=torch.uint8, device="cuda") for _ in range(2)]
    want = [x.clone() for x in both(ws[0])]
    st = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in st:
        s.wait_stream(torch.cuda.current_stream())
    got = [both(w, s) for _ in range(4) for s, w in zip(st, ws)]
    for s in st:
        s.synchronize()
    for a in got:
        assert torch.equal(a[0], want[0]) and torch.equal(a[1], want[1])
    outs = [torch.zeros_like(x) for x in want]
    graphs = []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            if i:
                A.gqa_tree_paged_fp8(q[:new[0]], *cache, one[2], one[0], one[1], mask[:new[0]], max_len, out=outs[1], workspace=ws[0])
            else:
                A.gqa_tree_paged_fp8(q, *cache, table, starts, seq, mask, max_len, out=outs[0], workspace=ws[0])
        graphs.append(g)
    for n in range(3):
        for g, o, w in zip(graphs, outs, want):
            o.zero_()
            g.replay()
            eager = both(ws[0])
            torch.cuda.synchronize()
            assert torch.equal(o, w) and torch.equal(eager[0], want[0]) and torch.equal(eager[1], want[1]), n


def test_forks_decode_as_their_source():
    """A prompt's rows copied to two more requests, whose next tokens then differ."""
    import torch
    import aila_amd as A
    Hq, Hkv, D, page, P, B, L = 8, 2, 128, 16, 40, 4, 75
    caches = [A.paged_fp8_cache(P, Hkv, page, D) for _ in range(2)]
    table = torch.full((B, 8), -1, dtype=torch.int32, device="cuda")
    free, count, slots = torch.arange(P, dtype=torch.int32, device="cuda"), _i32([P]), _i32([0] * 256)
    g = torch.Generator(device="cuda").manual_seed(4)
    k, v = (torch.randn((256, Hkv, D), generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    A.kv_pages_reserve(_i32([0, -1, -1, -1]), _i32([L, 0, 0, 0]), table, free, count, page, slots)
    for c in caches:
        A.kv_append_paged_fp8(k, v, *c, slots)
    A.kv_pages_reserve(_i32([L, 0, -1, 0]), _i32([0, L, 0, L]), table, free, count, page, slots)
    A.kv_copy_paged_fp8(caches, table, _i32([0, 0]), _i32([1, 3]), _i32([L, L]), L)
    q = torch.randn((1, Hq, D), generator=g, device="cuda").to(torch.bfloat16).expand(B, Hq, D).contiguous()
    for c in caches:
        out = A.gqa_decode_paged_fp8(q, *c, table, _i32([L, L, 0, L]), 128)
        assert torch.equal(out[0], out[1]) and torch.equal(out[0], out[3]) and bool((out[2] == 0).all())
    before = [x.clone() for x in A.kv_read_paged_fp8(*caches[0], slots_of(table, 0, L, page))]
    A.kv_pages_reserve(_i32([L, L, -1, L]), _i32([1, 1, 0, 1]), table, free, count, page, slots)
    A.kv_append_paged_fp8(k[100:] * 8, v[100:] * 8, *caches[0], slots[:156].contiguous())
    after = A.kv_read_paged_fp8(*caches[0], slots_of(table, 3, L, page))
    # each has its own pages; the last block took a larger scale, which flushes half its smallest step at most
    for a, b in zip(before, after):
        assert float((a.double() - b.double()).abs().max()) <= 2.0 ** -10 * float(caches[0][2].max())
    assert len({int(x) for x in table[table >= 0].tolist()}) == int((table >= 0).sum())


def slots_of(table, b, n, page):
    t = table.tolist()[b]
    return _i32([t[r // page] * page + r % page for r in range(n)])


def test_on_another_stream():
    import torch
    import aila_amd as A
    a, b = ([_cache(20, 2, 16, 64, 3 + i) for i in range(2)] for _ in range(2))
    table = _table([200, 31, 40], 16, 20, 4)
    g = torch.Generator(device="cuda").manual_seed(4)
    qkv = torch.randn((9, 8, 64), generator=g, device="cuda").to(torch.bfloat16)
    q, k, v = qkv.split([4, 2, 2], 1)
    tl = table.tolist()
    slots, pos = _i32([tl[0][r // 16] * 16 + r % 16 for r in range(191, 200)]), _i32(list(range(9)))
    mask = dref.mask_words([list(range(i + 1)) for i in range(9)], 1).cuda()
    starts, rows, free, count = _i32([0, 9, 9, 9]), _i32([200, 31, 40]), _i32([-1] * 20), [_i32([0]), _i32([0])]

    def step(c, stream, table, count):
        o = A.prepare_qkv_paged_fp8(q, k, v, *c[0], slots, pos, stream=stream)
        t = A.gqa_tree_paged_fp8(o, *c[0], table, starts, rows, mask, 208, stream=stream)
        n = A.kv_keep_paged_fp8(c, table, _i32([191, 31, 40]), _i32([[0, 3, 7], [0, 0, 0], [0, 0, 0]]), _i32([3, 0, 0]), stream=stream)
        A.kv_copy_paged_fp8(c, table, _i32([1]), _i32([2]), _i32([31]), 48, stream=stream)
        A.kv_pages_trim(n, table, free.clone(), count, 16, stream=stream)
        return o, t, n

    t1, t2 = table.clone(), table.clone()
    want = step(a, None, t1, count[0])
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        inside = step(b, None, t2, count[1])
    st.synchronize()
    for x, y in zip(want, inside):
        assert torch.equal(x, y)
    c = [_cache(20, 2, 16, 64, 3 + i) for i in range(2)]
    t3, n3 = table.clone(), _i32([0])
    torch.cuda.synchronize()
    given = step(c, st, t3, n3)
    st.synchronize()
    for x, y in zip(want, given):
        assert torch.equal(x, y)
    assert torch.equal(t1, t2) and torch.equal(t1, t3) and int(count[0]) == int(count[1]) == int(n3)
    for x, y, z in zip(a, b, c):
        for i in range(4):
            assert torch.equal(x[i].view(torch.uint8), y[i].view(torch.uint8)) and torch.equal(x[i].view(torch.uint8), z[i].view(torch.uint8))


def test_offsets_beyond_32_bits():
    import torch
    import aila_amd as A
    H, page, D = 8, 128, 256
    P = (1 << 32) // (H * page * D) + 40
    cache = A.paged_fp8_cache(P, H, page, D)
    L, n = 300, 40
    table = _i32([[P - 1, 3, P - 2], [P - 9, P - 5, 0], [P - 11, P - 12, P - 13]])
    use = [P - 1, 3, P - 2, P - 9, P - 5, 0, P - 11, P - 12, P - 13]
    tl = table.tolist()
    slots = [tl[b][r // page] * page + r % page for b in range(2) for r in range(L)]
    g = torch.Generator(device="cuda").manual_seed(8)
    qkv = torch.randn((2 * L, 16 + 2 * H, D), generator=g, device="cuda").to(torch.bfloat16)
    q, k, v = qkv.split([16, H, H], 1)
    pos = _i32(list(range(L)) * 2)
    small = [t[use].clone() if t.dtype == torch.float32 else t.view(torch.uint8)[use].view(t.dtype) for t in cache]
    there = _i32([[0, 1, 2], [3, 4, 5], [6, 7, 8]])
    near = [there.tolist()[b][r // page] * page + r % page for b in range(2) for r in range(L)]
    a = A.prepare_qkv_paged_fp8(q, k, v, *cache, _i32(slots), pos, rotary_dim=64)
    b = A.prepare_qkv_paged_fp8(q, k, v, *small, _i32(near), pos, rotary_dim=64)
    assert torch.equal(a, b)
    rows = list(range(L - n, L)) + list(range(2 * L - 2, 2 * L))
    rng = np.random.default_rng(1)
    mask = dref.mask_words([p for m in (n, 2) for p in dref.paths(dref.parents(m, rng))], 1).cuda()
    starts, lens = _i32([0, n, n + 2, n + 2]), _i32([L, L, 0])
    for ws in (0, 1):
        w = torch.empty(A.gqa_tree_paged_fp8_workspace_size(n + 2, 3, 16, H, D, L, 1), dtype=torch.uint8, device="cuda") if ws else None
        x = A.gqa_tree_paged_fp8(a[rows].contiguous(), *cache, table, starts, lens, mask, L, workspace=w)
        y = A.gqa_tree_paged_fp8(a[rows].contiguous(), *small, there, starts, lens, mask, L, workspace=w)
        assert torch.equal(x, y)
    kept, counts = _i32([[0, 3, 9, 30], [1, 1, 1, 1], [0, 0, 0, 0]]), _i32([4, 1, 0])
    for c, t in ((cache, table), (small, there)):
        A.kv_keep_paged_fp8([c], t, _i32([L - n, L - 2, -1]), kept, counts)
        A.kv_copy_paged_fp8([c], t, _i32([0]), _i32([2]), _i32([L]), L)
    for big, little in zip(cache, small):
        assert torch.equal((big.view(torch.uint8) if big.dtype != torch.float32 else big)[use], little.view(torch.uint8) if big.dtype != torch.float32 else little)


def test_cpp_ops():
    """The C++ forms (tests/cpp/test_drafts.cpp)."""
    exe = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "test_drafts")
    assert os.path.exists(exe), "build first: python -c 'import __graft_entry__ as g; g.build()'"
    r = subprocess.run([exe], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stdout + r.stderr
