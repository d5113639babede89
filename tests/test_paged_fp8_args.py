"""CPU checks of the 8-bit paged cache's entry points: every refusal comes before
any device work, and the plain forms that the GPU tests compare with hold
against torch's own conversion and hand-made cases."""
import ctypes

import numpy as np
import pytest
import torch

import aila_amd
import paged_fp8_ref as ref

P16 = 4096           # an aligned address that is never dereferenced


def _rc(name, args, **bad):
    a = dict(args)
    a.update(bad)
    rc = getattr(aila_amd.lib(), "aila_hip_" + name)(*a.values(), None)
    return rc, aila_amd.lib().aila_hip_last_error().decode()


RESERVE = dict(cached=P16, new=P16 + 64, table=P16, free=P16, count=P16, starts=P16 + 128, lens=P16 + 192, slots=P16, B=4, mp=8, page=16, P=40, T=9)
RELEASE = dict(flags=P16, table=P16, free=P16, count=P16, B=4, mp=8, P=40)
APPEND = dict(k=P16, v=P16, stride=256, kp=P16, vp=P16, ks=P16, vs=P16, slots=P16, T=3, H=2, D=128, page=16, P=10)
READ = dict(kp=P16, vp=P16, ks=P16, vs=P16, slots=P16, ko=P16, vo=P16, T=3, H=2, D=128, page=16, P=10)
DECODE = dict(q=P16, stride=512, kp=P16, vp=P16, ks=P16, vs=P16, out=P16, ws=P16, ws_bytes=1 << 30, B=2, Hq=4, H=2, D=128, page=16, P=10, table=P16,
              mp=20, max_len=300, lens=P16)
PREFILL = dict(q=P16, stride=512, kp=P16, vp=P16, ks=P16, vs=P16, out=P16, ws=P16, ws_bytes=1 << 30, T=9, B=2, Hq=4, H=2, D=128, page=16, P=10, table=P16,
               mp=20, max_len=300, starts=P16, lens=P16)
PAGES = [dict(H=0), dict(H=-1), dict(page=0), dict(page=24), dict(page=-16), dict(P=0), dict(P=1 << 28), dict(kp=P16 + 8), dict(vp=P16 + 4), dict(ks=P16 + 2),
         dict(vs=P16 + 1), dict(kp=None), dict(vp=None), dict(ks=None), dict(vs=None), dict(D=96), dict(D=512), dict(D=0)]


@pytest.mark.parametrize("name,args,bad", [("kv_pages_reserve", RESERVE, b) for b in (
    *({k: None} for k in ("cached", "new", "table", "free", "count", "starts", "lens", "slots")), dict(lens=P16), dict(lens=P16 + 64), dict(starts=P16),
    dict(B=0), dict(B=2049), dict(mp=0), dict(mp=1 << 27), dict(page=0), dict(page=8), dict(P=0), dict(P=1 << 27), dict(T=0), dict(T=-1),
    dict(mp=1 << 21, B=1024))]
    + [("kv_pages_release", RELEASE, b) for b in (*({k: None} for k in ("flags", "table", "free", "count")), dict(B=0), dict(B=2049), dict(mp=0), dict(P=0),
                                                  dict(mp=1 << 21, B=1024))]
    + [("kv_append_paged_fp8", APPEND, b) for b in (*PAGES, dict(k=None), dict(v=None), dict(slots=None), dict(T=0), dict(stride=255), dict(stride=248),
                                                    dict(stride=260), dict(k=P16 + 8), dict(v=P16 + 2))]
    + [("kv_read_paged_fp8", READ, b) for b in (*PAGES, dict(slots=None), dict(ko=None), dict(vo=None), dict(T=0), dict(T=1 << 30), dict(ko=P16 + 8), dict(vo=P16 + 8))]
    + [("gqa_decode_paged_fp8", DECODE, b) for b in (
        *PAGES, dict(q=None), dict(out=None), dict(table=None), dict(lens=None), dict(B=0), dict(B=4097), dict(Hq=0), dict(Hq=5), dict(stride=504),
        dict(stride=516), dict(q=P16 + 8), dict(out=P16 + 8), dict(mp=0), dict(mp=1 << 27), dict(max_len=-1), dict(max_len=321), dict(ws=P16 + 8),
        dict(ws_bytes=100), dict(B=4096, H=64, Hq=64, stride=8192, mp=1 << 20, max_len=1 << 24))]
    + [("gqa_prefill_paged_fp8", PREFILL, b) for b in (
        *PAGES, dict(q=None), dict(out=None), dict(table=None), dict(lens=None), dict(starts=None), dict(T=0), dict(T=1 << 30), dict(B=0), dict(B=4097),
        dict(Hq=0), dict(Hq=5), dict(stride=504), dict(stride=516), dict(q=P16 + 8), dict(out=P16 + 8), dict(mp=0), dict(mp=1 << 27), dict(max_len=-1),
        dict(max_len=321))])
def test_refusals(name, args, bad):
    rc, msg = _rc(name, args, **bad)
    want = -2 if bad.get("D", 128) != 128 else -4 if "ws_bytes" in bad else -1
    assert rc == want, (rc, msg)
    assert msg.startswith(name + ":"), msg


def test_workspace_sizes():
    f = aila_amd.gqa_decode_paged_fp8_workspace_size
    assert f(1, 16, 8, 128, 612) == 256 + 8 * 5 * 2 * 2 * 132 * 4  # a record pair for each 128 rows of each KV head, and the counts
    assert f(64, 40, 8, 128, 4000) == f(64, 40, 8, 128, 32768)     # as many as the device holds
    assert f(0, 16, 8, 128, 612) == f(1, 16, 0, 128, 612) == f(1, 15, 8, 128, 612) == f(1, 16, 8, 128, -1) == 0
    f = aila_amd.gqa_prefill_paged_fp8_workspace_size
    assert f(0, 1, 16, 8, 128, 100) == f(9, 1, 16, 8, 96, 100) == f(9, 0, 16, 8, 128, 100) == f(9, 1, 16, 8, 128, -1) == 0
    assert f(5000, 1, 16, 8, 128, 9000) == 0                       # tiles enough: no runs
    assert f(128, 1, 16, 8, 128, 9000) == 2 * 16 * 8 * 128 * 130 * 4    # 2 tiles a head, 16 runs each
    assert f(9, 2, 16, 8, 128, 9000) > 2 * 32 * 8 * 128 * 130 * 4  # a list, and the runs of 32 workgroups a head


def test_a_batch_needs_its_whole_workspace():
    need = aila_amd.gqa_prefill_paged_fp8_workspace_size(9, 2, 4, 2, 128, 300)
    rc, msg = _rc("gqa_prefill_paged_fp8", PREFILL, ws_bytes=need - 1)
    assert rc == -4 and str(need) in msg


# ---- the binding's own checks, with stand-ins for device tensors -----------------------------
class _Fake:
    """What the checks look at of a device tensor."""

    def __init__(self, shape, dtype, stride=None, ptr=4096, device=0):
        self.shape, self.dtype, self.is_cuda, self._ptr, self._dev = torch.Size(shape), dtype, True, ptr, device
        full = []
        n = 1
        for s in reversed(shape):
            full.insert(0, n)
            n *= s
        self._stride = tuple(stride or full)
        self._contig = self._stride == tuple(full)
        self.device = torch.device("cuda", device)

    def is_contiguous(self):
        return self._contig

    def stride(self, d=None):
        return self._stride if d is None else self._stride[d]

    def data_ptr(self):
        return self._ptr

    def dim(self):
        return len(self.shape)

    def numel(self):
        return int(np.prod(self.shape))

    def get_device(self):
        return self._dev


def _fakes():
    i32, f8, f32, bf = torch.int32, torch.float8_e4m3fn, torch.float32, torch.bfloat16
    return dict(k=_Fake((5, 2, 64), bf), v=_Fake((5, 2, 64), bf), kp=_Fake((4, 2, 32, 64), f8), vp=_Fake((4, 2, 32, 64), f8), ks=_Fake((4, 2, 2), f32),
                vs=_Fake((4, 2, 2), f32), slots=_Fake((5,), i32), q=_Fake((3, 4, 64), bf), table=_Fake((3, 2), i32), lens=_Fake((3,), i32),
                starts=_Fake((4,), i32), out=_Fake((3, 4, 64), bf))


@pytest.mark.parametrize("bad", [
    dict(k=_Fake((5, 2, 64), torch.float16)), dict(k=_Fake((5, 2, 64), torch.bfloat16, stride=(128, 64, 2))), dict(k=_Fake((5, 2, 64), torch.bfloat16, stride=(64, 64, 1))),
    dict(k=_Fake((5, 2, 64), torch.bfloat16, stride=(132, 64, 1))), dict(k=_Fake((5, 2, 64), torch.bfloat16, stride=(256, 128, 1))),
    dict(k=_Fake((5, 2, 64), torch.bfloat16, stride=(256, 64, 1))), dict(k=_Fake((4, 2, 64), torch.bfloat16)), dict(k=_Fake((5, 2, 64), torch.bfloat16, ptr=4100)),
    dict(k=None), dict(kp=_Fake((4, 2, 32, 64), torch.uint8)), dict(vp=_Fake((4, 2, 16, 64), torch.float8_e4m3fn)), dict(kp=_Fake((4, 2, 32), torch.float8_e4m3fn)),
    dict(ks=_Fake((4, 2, 1), torch.float32)), dict(vs=_Fake((4, 2, 2), torch.float64)), dict(slots=_Fake((5,), torch.int64)), dict(v=_Fake((5, 2, 64), torch.bfloat16, device=1)),
    dict(slots=_Fake((5,), torch.int32, device=1)), dict(kp=torch.zeros((4, 2, 32, 64), dtype=torch.uint8).view(torch.float8_e4m3fn))])
def test_append_checks_its_tensors(monkeypatch, bad):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    f = {**_fakes(), **bad}
    with pytest.raises(ValueError):
        aila_amd.kv_append_paged_fp8(*(f[x] for x in ("k", "v", "kp", "vp", "ks", "vs", "slots")))


@pytest.mark.parametrize("bad", [
    dict(q=_Fake((3, 4, 64), torch.float32)), dict(q=_Fake((3, 4, 128), torch.bfloat16)), dict(q=_Fake((3, 4, 64), torch.bfloat16, stride=(1, 64, 1))),
    dict(table=_Fake((3, 2), torch.int64)), dict(table=_Fake((3, 2), torch.int32, stride=(3, 1))), dict(lens=_Fake((4,), torch.int32)), dict(starts=_Fake((3,), torch.int32)),
    dict(out=_Fake((3, 4, 64), torch.float32)), dict(out=_Fake((3, 4, 64), torch.bfloat16, stride=(512, 64, 1))), dict(out=_Fake((3, 4, 64), torch.bfloat16, device=1)),
    dict(kp=_Fake((4, 2, 32, 64), torch.float8_e5m2)), dict(lens=_Fake((3,), torch.int32, device=1))])
def test_attention_checks_its_tensors(monkeypatch, bad):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    f = {**_fakes(), **bad}
    cache = [f[x] for x in ("kp", "vp", "ks", "vs")]
    if "starts" not in bad:
        with pytest.raises(ValueError):
            aila_amd.gqa_decode_paged_fp8(f["q"], *cache, f["table"], f["lens"], 64, out=f["out"])
    with pytest.raises(ValueError):
        aila_amd.gqa_prefill_paged_fp8(f["q"], *cache, f["table"], f["starts"], f["lens"], 64, out=f["out"])


def test_tensors_of_another_device_than_the_call(monkeypatch):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    f = _fakes()
    with pytest.raises(ValueError, match="cuda:1"):
        aila_amd.kv_append_paged_fp8(*(f[x] for x in ("k", "v", "kp", "vp", "ks", "vs", "slots")))


# ---- the plain forms ---------------------------------------------------------------------------
def test_plain_rounding_is_the_formats():
    v = ref.code_values()
    c = torch.arange(256, dtype=torch.int32).to(torch.uint8).view(torch.float8_e4m3fn).float().double().numpy()
    assert np.array_equal(v, c, equal_nan=True)
    x = torch.cat([torch.randn(20000, generator=torch.Generator().manual_seed(1)) * s for s in (1e-4, 0.01, 1, 100)])
    mid = torch.from_numpy(np.sort(v[np.isfinite(v)])).float()
    x = torch.cat([x, (mid[1:] + mid[:-1]) / 2]).clamp(-448, 448)      # ties too
    assert np.array_equal(ref.e4m3(x.double().numpy()), x.to(torch.float8_e4m3fn).float().double().numpy())
    assert ref.scale_exp(448.0) == 0 and ref.scale_exp(449.0) == 1 and ref.scale_exp(224.0) == -1 and ref.scale_exp(0.0) == -100
    assert ref.scale_exp(1e-40) == -100 and ref.scale_exp(3.3e38) == 119


def test_plain_append_and_reserve():
    kp = torch.zeros((2, 1, 16, 64), dtype=torch.uint8)
    c = ref.Cache(kp, torch.ones((2, 1, 1)))
    x = np.zeros((3, 1, 64))
    x[0, 0, 0], x[1, 0, 1], x[2, 0, 2] = 448.0, 1.0, 1792.0
    c.append(x[:2], [16, 17])
    assert c.scale[1, 0, 0] == 1 and c.val[1, 0, 0, 0] == 448
    c.append(x[2:], [18])                  # four times as large: the rows before shrink, their values stay
    assert c.scale[1, 0, 0] == 4 and c.val[1, 0, 0, 0] == 112 and c.val[1, 0, 1, 1] == 0.25 and c.val[1, 0, 2, 2] == 448
    t, n, starts, lens, slots = ref.reserve([3, 0, 16], [2, 20, 1], [[5, -1], [-1, -1], [7, -1]], [1, 2, 3], 3, 16, 30)
    assert (t, n, starts, lens) == ([[5, -1], [3, 2], [7, 1]], 0, [0, 2, 22, 23], [5, 20, 17])
    assert slots == [83, 84] + [48 + i for i in range(16)] + [32, 33, 34, 35] + [16] + [-1] * 7
    t, n, starts, lens, slots = ref.reserve([3, 0, 16], [2, 20, 0], [[5, -1], [-1, -1], [7, -1]], [1], 1, 16, 30)
    assert (t, n, lens) == ([[5, -1], [-1, -1], [7, -1]], 1, [5, 0, 16]) and slots[2:] == [-1] * 28
    assert ref.release([0, 1, 1], [[5, -1], [3, 2], [-1, 1]], [9, 0, 0, 0], 1) == ([[5, -1], [-1, -1], [-1, -1]], [9, 3, 2, 1], 4)


@pytest.mark.parametrize("name,args,bad", [
    ("kv_append_paged_fp8", APPEND, dict(T=1 << 28)), ("kv_append_paged_fp8", APPEND, dict(T=(1 << 28) - 15)),
    ("kv_read_paged_fp8", READ, dict(T=1 << 26, H=4)), ("kv_read_paged_fp8", READ, dict(T=2**31 - 1, H=1)),
    ("gqa_decode_paged_fp8", DECODE, dict(B=4096, H=4096, Hq=4096, stride=4096 * 128))])
def test_calls_of_more_threads_than_a_launch_has(name, args, bad):
    rc, msg = _rc(name, args, **bad)
    assert rc == -1 and msg.startswith(name + ":"), (rc, msg)
