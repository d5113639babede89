"""CPU checks of the entry points for drafts, forks and trims over the 8-bit paged
cache: every refusal comes before any device work, and their plain forms hold on
hand-made cases."""
import ctypes

import numpy as np
import pytest
import torch

import aila_amd
import draft_ref as dref
import paged_fp8_ref as ref
from test_paged_fp8_args import P16, PAGES, _Fake, _rc

PREPARE = dict(q=P16, qs=512, qh=128, k=P16, kst=256, v=P16, vst=256, qo=P16, qn=P16, kn=P16, kp=P16, vp=P16, ks=P16, vs=P16, slots=P16, pos=P16, ph=None,
               pw=None, sh=0, sw=0, T=3, Hq=4, H=2, D=128, page=16, P=10, rot=128, theta=ctypes.c_float(1e6), inv=None, eps=ctypes.c_float(1e-6))
TREE = dict(q=P16, stride=512, kp=P16, vp=P16, ks=P16, vs=P16, out=P16, ws=P16, ws_bytes=1 << 30, T=9, B=2, Hq=4, H=2, D=128, page=16, P=10, table=P16,
            mp=20, max_len=300, starts=P16, lens=P16, mask=P16, words=1)
TRIM = dict(lens=P16, table=P16, free=P16, count=P16, B=4, mp=8, page=16, P=40)


def _arr(*v):
    return (ctypes.c_void_p * len(v))(*v)


def _keep(**bad):
    a = dict(kp=P16, vp=P16, ks=P16, vs=P16)
    a.update({k: bad.pop(k) for k in list(bad) if k in a})
    b = dict(layers=1, table=P16, cached=P16, kept=P16, counts=P16 + 64, lens=P16 + 128, B=3, most=5, H=2, D=128, page=16, P=10, mp=8)
    arrays = {k: _arr(x) for k, x in a.items()}
    arrays.update({k: None for k in bad.pop("none", ())})
    b.update(bad)
    return _rc("kv_keep_paged_fp8", {**arrays, **b})


def _copy(**bad):
    a = dict(kp=P16, vp=P16, ks=P16, vs=P16)
    a.update({k: bad.pop(k) for k in list(bad) if k in a})
    b = dict(layers=1, table=P16, src=P16, dst=P16, lens=P16, n=2, max_len=100, B=3, H=2, D=128, page=16, P=10, mp=8)
    arrays = {k: _arr(x) for k, x in a.items()}
    arrays.update({k: None for k in bad.pop("none", ())})
    b.update(bad)
    return _rc("kv_copy_paged_fp8", {**arrays, **b})


@pytest.mark.parametrize("name,args,bad", [("prepare_qkv_paged_fp8", PREPARE, b) for b in (
    *PAGES, *({k: None} for k in ("q", "k", "v", "qo", "slots", "pos")), dict(Hq=0), dict(Hq=65536), dict(T=0), dict(T=-3), dict(T=1 << 30), dict(rot=-8), dict(rot=136),
    dict(rot=4), dict(rot=12), dict(ph=P16), dict(pw=P16), dict(sh=-1), dict(sw=-1), dict(theta=ctypes.c_float(0)), dict(qh=120), dict(qh=132), dict(qs=504),
    dict(qs=516), dict(qh=136, qs=528), dict(kst=248), dict(kst=260), dict(vst=248), dict(vst=260), dict(q=P16 + 8), dict(k=P16 + 8), dict(v=P16 + 2), dict(qo=P16 + 8),
    dict(qn=P16 + 4), dict(kn=P16 + 8))]
    + [("gqa_tree_paged_fp8", TREE, b) for b in (
        *PAGES, *({k: None} for k in ("q", "out", "table", "lens", "starts", "mask")), dict(T=0), dict(T=1 << 30), dict(B=0), dict(B=4097), dict(Hq=0), dict(Hq=5),
        dict(stride=504), dict(stride=516), dict(q=P16 + 8), dict(out=P16 + 8), dict(ws=P16 + 8), dict(mp=0), dict(mp=1 << 27), dict(max_len=-1), dict(max_len=321),
        dict(mask=P16 + 4), dict(words=0), dict(words=65), dict(ws_bytes=100))]
    + [("kv_pages_trim", TRIM, b) for b in (*({k: None} for k in ("lens", "table", "free", "count")), dict(B=0), dict(B=2049), dict(mp=0), dict(page=0), dict(page=24),
                                            dict(P=0), dict(mp=1 << 21, B=1024))])
def test_refusals(name, args, bad):
    rc, msg = _rc(name, args, **bad)
    want = -2 if bad.get("D", 128) != 128 else -4 if "ws_bytes" in bad else -1
    assert rc == want, (rc, msg)
    assert msg.startswith(name + ":"), msg


@pytest.mark.parametrize("bad", [*PAGES, dict(none=("kp",)), dict(none=("vs",)), dict(layers=0), dict(table=None), dict(cached=None), dict(kept=None), dict(counts=None),
                                 dict(lens=None), dict(B=0), dict(B=65536), dict(most=0), dict(most=65537), dict(mp=0), dict(mp=1 << 27), dict(lens=P16),
                                 dict(lens=P16 + 64)])
def test_keep_refusals(bad):
    rc, msg = _keep(**bad)
    assert rc == (-2 if bad.get("D", 128) != 128 else -1) and msg.startswith("kv_keep_paged_fp8:"), (rc, msg)


@pytest.mark.parametrize("bad", [*PAGES, dict(none=("vp",)), dict(none=("ks",)), dict(layers=-1), dict(table=None), dict(src=None), dict(dst=None), dict(lens=None),
                                 dict(B=0), dict(n=0), dict(n=65536), dict(mp=0), dict(mp=1 << 27), dict(max_len=-1), dict(max_len=129),
                                 dict(n=65535, max_len=1 << 20, mp=1 << 20)])
def test_copy_refusals(bad):
    rc, msg = _copy(**bad)
    assert rc == (-2 if bad.get("D", 128) != 128 else -1) and msg.startswith("kv_copy_paged_fp8:"), (rc, msg)


def test_every_layer_is_checked():
    a = [_arr(P16, P16), _arr(P16, P16), _arr(P16, P16), _arr(P16, P16 + 2)]
    rc = aila_amd.lib().aila_hip_kv_keep_paged_fp8(*a, 2, P16, P16, P16, P16 + 64, P16 + 128, 3, 5, 2, 128, 16, 10, 8, None)
    assert rc == -1


@pytest.mark.parametrize("bad", [dict(lens=P16 + 4), dict(lens=P16 + 56), dict(counts=P16 + 136), dict(cached=P16 + 124), dict(table=P16 + 48)])
def test_keep_lengths_over_what_comes_in(bad):
    """kept is 15 ints from P16 on, the table 24, the lengths going out 3 from P16 + 128 on."""
    rc, msg = _keep(**bad)
    assert rc == -1 and "comes in" in msg, (rc, msg)


def test_keep_of_the_same_pages_twice():
    for k, v in (((P16, P16 + 4096), (P16 + 64, P16)), ((P16, P16), (P16 + 64, P16 + 128)), ((P16, P16 + 64), (P16 + 128, P16 + 128)), ((P16,), (P16,))):
        a = [_arr(*k), _arr(*v), _arr(*[P16] * len(k)), _arr(*[P16] * len(k))]
        rc = aila_amd.lib().aila_hip_kv_keep_paged_fp8(*a, len(k), P16, P16, P16, P16 + 128, P16 + 256, 3, 5, 2, 128, 16, 10, 8, None)
        assert rc == -1 and b"twice" in aila_amd.lib().aila_hip_last_error()


@pytest.mark.parametrize("bad", [dict(qs=1024), dict(qh=256, qs=1024), dict(qh=256, qs=1024, T=1)])
def test_prepare_of_strided_queries_in_place(bad):
    rc, msg = _rc("prepare_qkv_paged_fp8", PREPARE, **bad)
    assert rc == -1 and "q_out may be q" in msg, (rc, msg)


def test_a_copy_of_no_rows_does_nothing():
    assert _copy(max_len=0)[0] == 0


def test_tree_workspace_sizes():
    f = aila_amd.gqa_tree_paged_fp8_workspace_size
    assert f(0, 1, 16, 8, 128, 100, 1) == f(9, 1, 16, 8, 96, 100, 1) == f(9, 0, 16, 8, 128, 100, 1) == f(9, 1, 16, 8, 128, -1, 1) == f(9, 1, 15, 8, 128, 100, 1) == 0
    assert f(9, 1, 16, 8, 128, 100, 0) == 0
    assert f(9, 1, 16, 8, 128, 100, 1) > 0


# ---- the binding's own checks, with stand-ins for device tensors -----------------------------
def _fakes():
    i32, f8, f32, bf = torch.int32, torch.float8_e4m3fn, torch.float32, torch.bfloat16
    return dict(q=_Fake((5, 4, 64), bf), k=_Fake((5, 2, 64), bf), v=_Fake((5, 2, 64), bf), kp=_Fake((4, 2, 32, 64), f8), vp=_Fake((4, 2, 32, 64), f8),
                ks=_Fake((4, 2, 2), f32), vs=_Fake((4, 2, 2), f32), slots=_Fake((5,), i32), pos=_Fake((5,), i32), qn=_Fake((64,), bf), kn=_Fake((64,), bf),
                out=_Fake((5, 4, 64), bf), table=_Fake((3, 2), i32), lens=_Fake((3,), i32), starts=_Fake((4,), i32), mask=_Fake((5, 1), torch.int64),
                cached=_Fake((3,), i32), kept=_Fake((3, 6), i32), counts=_Fake((3,), i32), free=_Fake((9,), i32), count=_Fake((1,), i32), src=_Fake((2,), i32),
                dst=_Fake((2,), i32), rows=_Fake((2,), i32), inv=_Fake((32,), f32))


BF, I32 = torch.bfloat16, torch.int32


@pytest.mark.parametrize("bad", [
    dict(q=_Fake((5, 4, 64), torch.float16)), dict(q=_Fake((5, 4, 64), BF, stride=(256, 64, 2))), dict(q=_Fake((5, 4, 64), BF, stride=(256, 60, 1))),
    dict(q=_Fake((5, 4, 64), BF, stride=(200, 64, 1))), dict(q=_Fake((5, 4, 64), BF, stride=(516, 128, 1))), dict(q=_Fake((5, 4, 64), BF, stride=(512, 132, 1))),
    dict(q=_Fake((5, 4, 64), BF, ptr=4104)), dict(q=_Fake((5, 4, 128), BF)), dict(k=_Fake((5, 2, 64), BF, stride=(256, 128, 1))), dict(k=_Fake((4, 2, 64), BF)),
    dict(v=_Fake((5, 2, 64), torch.float32)), dict(v=_Fake((5, 2, 64), BF, device=1)), dict(k=None), dict(slots=_Fake((5,), torch.int64)), dict(slots=_Fake((4,), I32)),
    dict(pos=_Fake((5,), torch.int64)), dict(pos=_Fake((4,), I32)), dict(pos=_Fake((3, 4), I32)), dict(pos=_Fake((3, 5), I32, stride=(1, 3))), dict(pos=_Fake((3, 5), I32)),
    dict(qn=_Fake((32,), BF)), dict(kn=_Fake((64,), torch.float32)), dict(kn=_Fake((64,), BF, device=1)), dict(out=_Fake((5, 4, 64), BF, stride=(512, 64, 1))),
    dict(out=_Fake((5, 4, 64), torch.float32)), dict(inv=_Fake((31,), torch.float32)), dict(inv=_Fake((32,), torch.float64)), dict(kp=_Fake((4, 2, 32, 64), torch.uint8))])
def test_prepare_checks_its_tensors(monkeypatch, bad):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    f = {**_fakes(), **bad}
    with pytest.raises(ValueError):
        aila_amd.prepare_qkv_paged_fp8(*(f[x] for x in ("q", "k", "v", "kp", "vp", "ks", "vs", "slots", "pos")), q_norm=f["qn"], k_norm=f["kn"], q_out=f["out"],
                                       inv_freq=f["inv"] if "inv" in bad else None)


@pytest.mark.parametrize("bad", [
    dict(mask=_Fake((5, 1), torch.int32)), dict(mask=_Fake((4, 1), torch.int64)), dict(mask=_Fake((5,), torch.int64)), dict(mask=_Fake((5, 2), torch.int64, stride=(4, 1))),
    dict(mask=_Fake((5, 1), torch.int64, device=1)), dict(mask=None), dict(starts=None), dict(starts=_Fake((3,), I32)), dict(lens=_Fake((4,), I32)),
    dict(table=_Fake((3, 2), torch.int64)), dict(q=_Fake((5, 4, 64), BF, stride=(512, 128, 1))), dict(out=_Fake((5, 4, 64), BF, device=1))])
def test_tree_checks_its_tensors(monkeypatch, bad):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    f = {**_fakes(), **bad}
    with pytest.raises(ValueError):
        aila_amd.gqa_tree_paged_fp8(f["q"], f["kp"], f["vp"], f["ks"], f["vs"], f["table"], f["starts"], f["lens"], f["mask"], 64, out=f["out"])


@pytest.mark.parametrize("bad", [
    dict(kept=_Fake((3,), I32)), dict(kept=_Fake((4, 6), I32)), dict(kept=_Fake((3, 6), torch.int64)), dict(counts=_Fake((4,), I32)), dict(cached=_Fake((3,), torch.int64)),
    dict(lens=_Fake((3,), I32, device=1)), dict(table=_Fake((3, 2), I32, stride=(4, 1))), dict(vp=_Fake((4, 2, 16, 64), torch.float8_e4m3fn)), dict(caches=[]),
    dict(second=(4, 2, 16, 64)), dict(ks=_Fake((4, 2, 2), torch.float32, device=1))])
def test_keep_checks_its_tensors(monkeypatch, bad):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    f = {**_fakes(), **bad}
    caches = [tuple(f[x] for x in ("kp", "vp", "ks", "vs"))]
    if "second" in bad:
        f8, n = torch.float8_e4m3fn, bad["second"]
        caches.append((_Fake(n, f8), _Fake(n, f8), _Fake((4, 2, 1), torch.float32), _Fake((4, 2, 1), torch.float32)))
    with pytest.raises(ValueError):
        aila_amd.kv_keep_paged_fp8(bad.get("caches", caches), f["table"], f["cached"], f["kept"], f["counts"], lens=f["lens"])


@pytest.mark.parametrize("bad", [
    dict(src=_Fake((3,), I32)), dict(dst=_Fake((2,), torch.int64)), dict(rows=_Fake((2,), I32, device=1)), dict(table=_Fake((3, 2), torch.int64)),
    dict(kp=_Fake((4, 2, 32, 64), torch.float8_e5m2)), dict(rows=_Fake((2,), I32, stride=(2,)))])
def test_copy_checks_its_tensors(monkeypatch, bad):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    f = {**_fakes(), **bad}
    with pytest.raises(ValueError):
        aila_amd.kv_copy_paged_fp8([tuple(f[x] for x in ("kp", "vp", "ks", "vs"))], f["table"], f["src"], f["dst"], f["rows"], 64)


@pytest.mark.parametrize("bad", [dict(lens=_Fake((4,), I32)), dict(lens=_Fake((3,), torch.int64)), dict(count=_Fake((2,), I32)), dict(free=_Fake((9,), I32, device=1)),
                                 dict(table=_Fake((3, 2), I32, stride=(1, 3)))])
def test_trim_checks_its_tensors(monkeypatch, bad):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    f = {**_fakes(), **bad}
    with pytest.raises(ValueError):
        aila_amd.kv_pages_trim(f["lens"], f["table"], f["free"], f["count"], 32)


# ---- the plain forms ---------------------------------------------------------------------------
def test_plain_keep_moves_rows_and_scales():
    c = ref.Cache(torch.zeros((3, 1, 16, 64), dtype=torch.uint8), torch.ones((3, 1, 1)))
    c.scale[0], c.scale[2] = 0.25, 1.0
    for r in range(16):
        c.val[0, 0, r], c.val[2, 0, r] = 8 + r % 8, 64 + 8 * (r % 8)      # 14 rows of page 0, then a draft that ends in page 2
    # draft rows 14.. : tokens 0, 1 in page 0 (rows 14, 15), 2.. in page 2 (rows 0..); tokens 0 and 3 stay
    lens = dref.keep(c, [[0, 2]], [14], [[0, 3, -1]], [2], 16)
    assert lens == [16] and c.scale[0, 0, 0] == 1.0
    assert c.val[0, 0, 15, 0] == 72 and c.val[0, 0, 14, 0] == 3.5 and c.val[0, 0, 0, 0] == 2.0
    assert dref.keep(c, [[0, 2]], [-1], [[0, 3, -1]], [2], 16) == [-1]
    assert dref.trim([16, -1], [[0, 2], [1, -1]], [0, 0, 0], 0, 16) == ([[0, -1], [1, -1]], [2, 0, 0], 1)


def test_plain_norm_and_rotation():
    x = np.zeros((2, 1, 64))
    x[:, 0, 0], x[:, 0, 40] = 3.0, 4.0
    y, size = dref.norm_rotate(x, None, [[0], [1]], 32, 1e4, 0.0)
    r = np.sqrt(25 / 64)
    assert np.allclose(y[0, 0, [0, 40]], [3 / r, 4 / r]) and np.allclose(y[1, 0, [0, 16, 40]], [3 / r * np.cos(1), 3 / r * np.sin(1), 4 / r])
    assert np.allclose(size[1, 0, [0, 16, 40]], [3 / r, 3 / r, 4 / r])
    assert dref.streams([[0, 1], [10, 11], [20, 21]], (1, 1, 1), 12).tolist() == [[0, 10, 20, 0, 0, 0], [1, 11, 21, 1, 1, 1]]
    assert dref.mask_words([[0, 64], [63]], 2).tolist() == [[1, 1], [-2**63, 0]]
