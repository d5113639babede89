"""CPU checks of calls that the draft operators refuse before any device work."""
import ctypes
import os
import random
import subprocess

import pytest
import torch

import aila_amd

CPP = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "test_draft_refusals")


def test_cpp_refusals():
    """The C++ forms (tests/cpp/test_draft_refusals.cpp), which need no device."""
    assert os.path.exists(CPP), "build first: python -c 'import __graft_entry__ as g; g.build()'"
    r = subprocess.run([CPP], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stdout + r.stderr


# ---- what prepare writes over what it reads ------------------------------------------------------
BASE = 1 << 24                   # an address that is never dereferenced
T, HQ, HKV, D = 7, 4, 2, 64
OUT = T * HQ * D                 # values of q_out


def _prepare(qo, q=None, qs=None, qh=None, k=None, ks=None, v=None, vs=None, tokens=T):
    """Distances in values from q_out; without a device the call can only be refused, or fail at its launch."""
    far = 1 << 20

    def at(x, i):
        return BASE + 2 * (qo + (far * i if x is None else x))
    rc = aila_amd.lib().aila_hip_prepare_qkv_paged_fp8(
        at(q, 1), qs or HQ * D, qh or D, at(k, 2), ks or HKV * D, at(v, 3), vs or HKV * D, BASE + 2 * qo, None, None, BASE + (1 << 23), BASE + (1 << 23) + (1 << 20),
        BASE + (1 << 23) + (2 << 20), BASE + (1 << 23) + (3 << 20), BASE + (1 << 23) + (4 << 20), None, None, None, 0, 0, tokens, HQ, HKV, D, 16, 10, 0,
        ctypes.c_float(1e4), None, ctypes.c_float(1e-6), None)
    return rc, aila_amd.lib().aila_hip_last_error().decode()


GATED = dict(qs=2 * HQ * D + 2 * HKV * D, qh=2 * D)      # q|gate rows between k's and v's


@pytest.mark.parametrize("bad", [
    dict(k=0), dict(k=8), dict(k=OUT - 8), dict(k=-8), dict(k=-T * HKV * D + 8), dict(v=0), dict(v=OUT - 8), dict(v=-T * HKV * D + 8),
    dict(k=-3 * 1024, ks=1024), dict(k=-6 * 4096, ks=4096), dict(k=-6 * 4096 - HKV * D + 8, ks=4096), dict(v=OUT - 8 - 4096, vs=4096),
    dict(q=8), dict(q=-8), dict(q=OUT - 8), dict(q=-OUT + 8), dict(q=0, **GATED), dict(q=0, qs=512, qh=64), dict(q=-D, **GATED), dict(q=-5 * GATED["qs"], **GATED),
    dict(q=-6 * GATED["qs"] - 3 * 2 * D - D + 8, **GATED), dict(q=OUT - 8 - GATED["qs"], **GATED), dict(q=-D, qs=2 * D * HQ, qh=2 * D, tokens=1)])
def test_prepare_over_its_inputs(bad):
    rc, msg = _prepare(1 << 19, **bad)
    assert rc == -1 and ("overlaps" in msg or "q_out may be q" in msg), (rc, msg)


# What stands beside q_out, or around it, is no overlap: the gap between two tokens' rows, or between the
# rows of the only token's heads. (Without a device such a call fails at its launch.)
@pytest.mark.skipif(torch.cuda.is_available(), reason="would launch over addresses that are not there")
@pytest.mark.parametrize("good", [
    dict(), dict(q=0), dict(k=OUT), dict(k=-T * HKV * D), dict(v=OUT), dict(q=OUT), dict(q=-OUT), dict(k=-HKV * D, ks=OUT + HKV * D), dict(k=-6 * 4096 - HKV * D, ks=4096),
    dict(v=OUT, vs=4096), dict(q=-HQ * D, qs=OUT + HQ * D), dict(q=-HQ * D - 2 * (OUT + HQ * D), qs=OUT + HQ * D),
    dict(q=-6 * GATED["qs"] - 3 * 2 * D - D, **GATED), dict(q=-D, qs=4096 + 2 * HQ * D, qh=HQ * D + D, tokens=1)])
def test_prepare_beside_its_inputs(good):
    rc, msg = _prepare(1 << 19, **good)
    assert rc == -3 and "overlaps" not in msg, (rc, msg)


@pytest.mark.skipif(torch.cuda.is_available(), reason="would launch over addresses that are not there")
def test_overlaps_are_what_counting_finds():
    rng, seen = random.Random(3), [0, 0]
    for _ in range(400):
        tokens, qh = rng.choice((1, 2, 3, 7)), D + 8 * rng.choice((0, 0, 8, 33, 40))
        qs = (HQ - 1) * qh + D + 8 * rng.choice((0, 1, 30, 300))
        ks, q, k = HKV * D + 8 * rng.choice((0, 2, 32, 300)), 8 * rng.randint(-400, 300), 8 * rng.randint(-300, 300)
        out = range(tokens * HQ * D)
        over = any(k + t * ks < out.stop and k + t * ks + HKV * D > 0 for t in range(tokens))
        over |= q != 0 and any(q + t * qs + h * qh < out.stop and q + t * qs + h * qh + D > 0 for t in range(tokens) for h in range(HQ))
        rc, msg = _prepare(1 << 19, q=q, qs=qs, qh=qh, k=k, ks=ks, tokens=tokens)
        if "q_out may be q" in msg:
            continue
        assert ("overlaps" in msg) == over, (tokens, qh, qs, ks, q, k, msg)
        seen[over] += 1
    assert min(seen) > 40
