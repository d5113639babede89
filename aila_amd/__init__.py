"""MI355X-native attention hot path for Aila (Qwen3 GQA + Gated DeltaNet).

The compute lives in ``aila_amd/libaila_hip.so`` (hand-written gfx950 HIP
kernels behind the C ABI declared in ``include/aila_hip.h``). This module
is a thin host-side binding over that C ABI for torch device tensors: it
checks shapes, dtypes and contiguity on the host, then passes raw device
pointers and the current HIP stream. There is no fallback: if the library
is missing or fails to load, every call raises.
"""
from __future__ import annotations

import array
import ctypes
import functools
import itertools
import math
import operator
import os

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libaila_hip.so")
_lib = None

_P = ctypes.c_void_p
_I = ctypes.c_int
_F = ctypes.c_float
_SZ = ctypes.c_size_t
_L = ctypes.c_long

_SIGS = {
    "aila_hip_last_error": ([], ctypes.c_char_p),
    "aila_hip_version": ([], _I),
    "aila_hip_gqa_decode_workspace_size": ([_I, _I, _I], _SZ),
    "aila_hip_gqa_decode": ([_P, _P, _P, _P, _P, _SZ, _I, _I, _I, _I, _I, _I, _P, _P], _I),
    "aila_hip_gqa_decode_window": ([_P, _P, _P, _P, _P, _SZ, _I, _I, _I, _I, _I, _I, _P, _I, _I, _I, _P], _I),
    "aila_hip_gqa_decode_paged": ([_P, _P, _P, _P, _P, _SZ, _I, _I, _I, _I, _I, _P, _I, _I, _P, _P], _I),
    "aila_hip_kv_append_paged": ([_P, _P, _P, _P, _I, _I, _I, _I, _P, _I, _P, _P], _I),
    "aila_hip_gqa_decode_noalloc_max_bytes": ([], _SZ),
    "aila_hip_gqa_decode_noalloc": ([_P, _P, _P, _P, _I, _I, _I, _I, _I, _I, _P, _P], _I),
    "aila_hip_gqa_decode_append": ([_P, _P, _P, _P, _P, _P, _P, _SZ, _I, _I, _I, _I, _I, _I, _P, _P], _I),
    "aila_hip_gqa_decode_prepare_append": ([_P, _I, _P, _P, _P, _P, _P, _P, _P, _P, _P, _SZ, _I, _I, _I, _I, _I,
                                            _I, _F, _F, _I, _P, _P, _P], _I),
    "aila_hip_kv_append": ([_P, _P, _P, _P, _I, _I, _I, _I, _I, _P, _P], _I),
    "aila_hip_gqa_prefill": ([_P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _I, _I, _P], _I),
    "aila_hip_gqa_prefill_cached": ([_P, _P, _P, _P, _I, _I, _I, _I, _I, _I, _P], _I),
    "aila_hip_gqa_prefill_cached_workspace_size": ([_I, _I, _I, _I, _I], _SZ),
    "aila_hip_gqa_prefill_cached_ws": ([_P, _P, _P, _P, _P, _SZ, _I, _I, _I, _I, _I, _I, _P], _I),
    "aila_hip_copy_to_cache": ([_P, _P, _I, _I, _I, _I, _I, _P], _I),
    "aila_hip_kv_pages_reserve": ([_P, _P, _P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _I, _P], _I),
    "aila_hip_kv_pages_release": ([_P, _P, _P, _P, _I, _I, _I, _P], _I),
    "aila_hip_kv_append_paged_fp8": ([_P, _P, _L, _P, _P, _P, _P, _P, _I, _I, _I, _I, _I, _P], _I),
    "aila_hip_kv_read_paged_fp8": ([_P, _P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _I, _P], _I),
    "aila_hip_gqa_decode_paged_fp8_workspace_size": ([_I, _I, _I, _I, _I], _SZ),
    "aila_hip_gqa_decode_paged_fp8": ([_P, _L, _P, _P, _P, _P, _P, _P, _SZ, _I, _I, _I, _I, _I, _I, _P, _I, _I, _P,
                                       _P], _I),
    "aila_hip_gqa_prefill_paged_fp8_workspace_size": ([_I, _I, _I, _I, _I, _I], _SZ),
    "aila_hip_gqa_prefill_paged_fp8": ([_P, _L, _P, _P, _P, _P, _P, _P, _SZ, _I, _I, _I, _I, _I, _I, _I, _P, _I, _I,
                                        _P, _P, _P], _I),
    "aila_hip_prepare_qkv_paged_fp8": ([_P, _L, _L, _P, _L, _P, _L, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _I, _I, _I, _I,
                                        _I, _I, _I, _I, _I, _F, _P, _F, _P], _I),
    "aila_hip_gqa_tree_paged_fp8_workspace_size": ([_I, _I, _I, _I, _I, _I, _I], _SZ),
    "aila_hip_gqa_tree_paged_fp8": ([_P, _L, _P, _P, _P, _P, _P, _P, _SZ, _I, _I, _I, _I, _I, _I, _I, _P, _I, _I, _P, _P, _P,
                                     _I, _P], _I),
    "aila_hip_kv_keep_paged_fp8": ([_P, _P, _P, _P, _I, _P, _P, _P, _P, _P, _I, _I, _I, _I, _I, _I, _I, _P], _I),
    "aila_hip_kv_pages_trim": ([_P, _P, _P, _P, _I, _I, _I, _I, _P], _I),
    "aila_hip_kv_copy_paged_fp8": ([_P, _P, _P, _P, _I, _P, _P, _P, _P, _I, _I, _I, _I, _I, _I, _I, _I, _P], _I),
    "aila_hip_deltanet_decode": ([_P, _P, _P, _P, _P, _P, _P, _P, _P,
                                  _I, _I, _I, _I, _I, _F, _F, _P], _I),
    "aila_hip_deltanet_prefill_workspace_size": ([_I, _I, _I, _I, _I], _SZ),
    "aila_hip_deltanet_layer_prefill_workspace_size": ([_I, _I, _I, _I, _I, _I], _SZ),
    "aila_hip_deltanet_layer_prefill": ([_P, _I, _P, _I, _P, _P, _I, _P, _P, _I, _P, _P, _P, _P, _P, _P, _SZ,
                                         _I, _I, _I, _I, _I, _I, _I, _F, _F, _P], _I),
    "aila_hip_deltanet_layer_decode": ([_P, _I, _P, _I, _P, _P, _I, _P, _P, _I, _P, _P, _P, _P, _P, _P,
                                        _I, _I, _I, _I, _I, _I, _F, _F, _P, _P], _I),
    "aila_hip_decode_prepare_qkv": ([_P, _I, _P, _P, _P, _P, _P, _P, _P, _P,
                                     _I, _I, _I, _I, _I, _I, _F, _F, _I, _P, _P, _P], _I),
    "aila_hip_head_rms_norm": ([_P, _P, _I, _I, _I, _F, _P], _I),
    "aila_hip_apply_rope": ([_P, _P, _I, _I, _I, _I, _I, _I, _F, _P, _P], _I),
    "aila_hip_sigmoid_mul": ([_P, _P, _P, ctypes.c_long, _P], _I),
    "aila_hip_deltanet_prefill": ([_P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _SZ,
                                   _I, _I, _I, _I, _I, _I, _F, _F, _P], _I),
}


class AilaHipError(RuntimeError):
    pass


def lib() -> ctypes.CDLL:
    """Load the HIP library (raises if it has not been built)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise AilaHipError(
                f"{LIB_PATH} not found: build it with `python -m aila_amd.build`")
        l = ctypes.CDLL(LIB_PATH)
        for name, (argt, rest) in _SIGS.items():
            f = getattr(l, name)
            f.argtypes = argt
            f.restype = rest
        _lib = l
    return _lib


def exported_symbols():
    return list(_SIGS)


def _check(rc: int, what: str) -> None:
    if rc != 0:
        msg = lib().aila_hip_last_error().decode(errors="replace")
        raise AilaHipError(f"{what} failed ({rc}): {msg}")


# A decode step is a handful of microseconds on the device, and its binding a
# dozen checked tensors: the checks below test everything in one expression and
# form messages only on the failing path, addresses go to ctypes as plain
# integers, and the stream handle is read without building a Stream object
# (whole-layer decode step, back to back calls: 15.4 -> 11.0 us a call).
def _stream(stream=None):
    import torch
    if stream is None:
        raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)   # not public: torch may drop it
        if raw is not None:
            return raw(torch.cuda.current_device())
        stream = torch.cuda.current_stream()
    return stream.cuda_stream


def _ptr(t):
    return None if t is None else t.data_ptr()


def _need(t, dtype, shape, name, align=16):
    if t is not None and t.is_cuda and t.dtype is dtype and t.shape == shape and t.is_contiguous() \
            and not t.data_ptr() % align:
        return
    if t is None:
        raise ValueError(f"{name} is required")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a device tensor")
    if t.dtype != dtype:
        raise ValueError(f"{name}: dtype {t.dtype}, expected {dtype}")
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name}: shape {tuple(t.shape)}, expected {tuple(shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    if t.data_ptr() % align:
        raise ValueError(f"{name} must be {align}-byte aligned")


class RopePos(ctypes.Structure):
    """``aila_hip_rope_pos``: rotary positions that differ from the cache row
    (text shift past the prompt and interleaved mRoPE streams, the reference's
    apply_rope_partial arguments). Build it with :func:`rope_pos`."""
    _fields_ = [("interleaved", _I), ("pos_t", _P), ("pos_h", _P), ("pos_w", _P),
                ("pos_stride", _I), ("prompt_pos_len", _I), ("text_pos_delta", _I),
                ("prompt_pos_lens", _P), ("text_pos_deltas", _P),
                ("mrope_section_t", _I), ("mrope_section_h", _I), ("mrope_section_w", _I),
                ("inv_freq", _P)]


def rope_pos(prompt_pos_len: int = 0, text_pos_delta: int = 0, pos_t=None, pos_h=None, pos_w=None,
             interleaved: bool = True, sections=(0, 0, 0), prompt_pos_lens=None, text_pos_deltas=None,
             inv_freq=None):
    """Rotary position record. pos_t/pos_h/pos_w: device int32 [P] (one prompt,
    shared by every sequence) or [B, P] (per sequence); prompt_pos_lens /
    text_pos_deltas: optional device int32 [B] overriding the scalars;
    inv_freq: optional device float32 [rotary_dim/2] table (pair d rotates by
    position * inv_freq[d])."""
    import torch
    rp = RopePos()
    rp.interleaved = int(bool(interleaved))
    rp.prompt_pos_len = int(prompt_pos_len)
    rp.text_pos_delta = int(text_pos_delta)
    rp.mrope_section_t, rp.mrope_section_h, rp.mrope_section_w = (int(x) for x in sections)
    keep = []
    streams = (pos_t, pos_h, pos_w)
    if any(t is not None for t in streams):
        if any(t is None for t in streams):
            raise ValueError("pos_t, pos_h and pos_w go together")
        shape = tuple(pos_t.shape)
        if len(shape) not in (1, 2):
            raise ValueError("position streams must be [P] or [B, P]")
        for t, name in zip(streams, ("pos_t", "pos_h", "pos_w")):
            _need(t, torch.int32, shape, name, align=4)
            keep.append(t)
        rp.pos_t, rp.pos_h, rp.pos_w = (t.data_ptr() for t in streams)
        rp.pos_stride = shape[1] if len(shape) == 2 else 0
    for t, name in ((prompt_pos_lens, "prompt_pos_lens"), (text_pos_deltas, "text_pos_deltas")):
        if t is not None:
            _need(t, torch.int32, tuple(t.shape), name, align=4)
            keep.append(t)
    if prompt_pos_lens is not None:
        rp.prompt_pos_lens = prompt_pos_lens.data_ptr()
    if text_pos_deltas is not None:
        rp.text_pos_deltas = text_pos_deltas.data_ptr()
    if inv_freq is not None:
        _need(inv_freq, torch.float32, tuple(inv_freq.shape), "inv_freq", align=4)
        keep.append(inv_freq)
        rp.inv_freq = inv_freq.data_ptr()
    rp._keep = keep   # the device arrays must outlive the launches that read them
    return rp


def _rope_arg(rope):
    return None if rope is None else ctypes.byref(rope)


# ----------------------------------------------------------------- GQA ----
def gqa_decode_workspace_size(B: int, Hq: int, D: int) -> int:
    return int(lib().aila_hip_gqa_decode_workspace_size(B, Hq, D))


def gqa_decode(q, k_cache, v_cache, cached_len: int, out=None, workspace=None,
               seq_lens=None, window=None, stream=None):
    """q [B,Hq,D] bf16; k_cache/v_cache [B,Hkv,max_seq,D] bf16 -> out [B,Hq,D].

    ``workspace``: uint8 device tensor of >= gqa_decode_workspace_size bytes
    enables split-K; None runs the single-pass kernel. ``seq_lens``: optional
    int32 [B] device tensor of per-sequence lengths (<= cached_len).
    ``window``: optional (window, window_start, sink) — the reference's
    decode window with attention sinks (window_start -1: max(512, window))."""
    import torch
    B, Hq, D = q.shape
    Hkv, max_seq = k_cache.shape[1], k_cache.shape[2]
    _need(q, torch.bfloat16, (B, Hq, D), "q")
    _need(k_cache, torch.bfloat16, (B, Hkv, max_seq, D), "k_cache")
    _need(v_cache, torch.bfloat16, (B, Hkv, max_seq, D), "v_cache")
    if out is None:
        out = torch.empty_like(q)
    _need(out, torch.bfloat16, (B, Hq, D), "out")
    ws_bytes = 0
    if workspace is not None:
        if not workspace.is_cuda or not workspace.is_contiguous():
            raise ValueError("workspace must be a contiguous device tensor")
        ws_bytes = workspace.numel() * workspace.element_size()
    if seq_lens is not None:
        _need(seq_lens, torch.int32, (B,), "seq_lens", align=4)
    if window is not None:
        w, ws0, sink = (int(x) for x in window)
        rc = lib().aila_hip_gqa_decode_window(_ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(out),
                                              _ptr(workspace), ws_bytes, B, Hq, Hkv, D, max_seq,
                                              int(cached_len), _ptr(seq_lens), w, ws0, sink, _stream(stream))
        _check(rc, "aila_hip_gqa_decode_window")
        return out
    rc = lib().aila_hip_gqa_decode(_ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(out),
                                   _ptr(workspace), ws_bytes, B, Hq, Hkv, D, max_seq,
                                   int(cached_len), _ptr(seq_lens), _stream(stream))
    _check(rc, "aila_hip_gqa_decode")
    return out


def gqa_decode_paged(q, k_pages, v_pages, block_table, seq_lens, max_len: int, out=None, workspace=None,
                     stream=None):
    """Decode over a paged cache. q [B,Hq,D]; k_pages/v_pages [num_pages,Hkv,
    page_size,D] bf16; block_table int32 [B, max_pages]; seq_lens int32 [B]
    (each <= max_len) -> out [B,Hq,D]."""
    import torch
    B, Hq, D = q.shape
    num_pages, Hkv, page_size = k_pages.shape[0], k_pages.shape[1], k_pages.shape[2]
    max_pages = block_table.shape[1]
    _need(q, torch.bfloat16, (B, Hq, D), "q")
    _need(k_pages, torch.bfloat16, (num_pages, Hkv, page_size, D), "k_pages")
    _need(v_pages, torch.bfloat16, (num_pages, Hkv, page_size, D), "v_pages")
    _need(block_table, torch.int32, (B, max_pages), "block_table", align=4)
    _need(seq_lens, torch.int32, (B,), "seq_lens", align=4)
    if out is None:
        out = torch.empty_like(q)
    _need(out, torch.bfloat16, (B, Hq, D), "out")
    ws_bytes = 0
    if workspace is not None:
        if not workspace.is_cuda or not workspace.is_contiguous():
            raise ValueError("workspace must be a contiguous device tensor")
        ws_bytes = workspace.numel() * workspace.element_size()
    rc = lib().aila_hip_gqa_decode_paged(_ptr(q), _ptr(k_pages), _ptr(v_pages), _ptr(out), _ptr(workspace),
                                         ws_bytes, B, Hq, Hkv, D, page_size, _ptr(block_table), max_pages,
                                         int(max_len), _ptr(seq_lens), _stream(stream))
    _check(rc, "aila_hip_gqa_decode_paged")
    return out


def kv_append_paged(k_new, v_new, k_pages, v_pages, block_table, positions, stream=None):
    """k_new/v_new [B,Hkv,D] -> row positions[b] of sequence b in the page pool."""
    import torch
    num_pages, Hkv, page_size, D = k_pages.shape
    B, max_pages = block_table.shape
    _need(k_new, torch.bfloat16, (B, Hkv, D), "k_new")
    _need(v_new, torch.bfloat16, (B, Hkv, D), "v_new")
    _need(k_pages, torch.bfloat16, (num_pages, Hkv, page_size, D), "k_pages")
    _need(v_pages, torch.bfloat16, (num_pages, Hkv, page_size, D), "v_pages")
    _need(block_table, torch.int32, (B, max_pages), "block_table", align=4)
    _need(positions, torch.int32, (B,), "positions", align=4)
    rc = lib().aila_hip_kv_append_paged(_ptr(k_new), _ptr(v_new), _ptr(k_pages), _ptr(v_pages), B, Hkv, D,
                                        page_size, _ptr(block_table), max_pages, _ptr(positions), _stream(stream))
    _check(rc, "aila_hip_kv_append_paged")


def gqa_decode_noalloc(q, k_cache, v_cache, cached_len: int, out=None, seq_lens=None, stream=None):
    """gqa_decode with the split records in the library's static device
    scratch (no workspace argument, no allocation in the library). Calls
    that overlap on one GPU share that scratch and race."""
    import torch
    B, Hq, D = q.shape
    Hkv, max_seq = k_cache.shape[1], k_cache.shape[2]
    _need(q, torch.bfloat16, (B, Hq, D), "q")
    _need(k_cache, torch.bfloat16, (B, Hkv, max_seq, D), "k_cache")
    _need(v_cache, torch.bfloat16, (B, Hkv, max_seq, D), "v_cache")
    if out is None:
        out = torch.empty_like(q)
    _need(out, torch.bfloat16, (B, Hq, D), "out")
    if seq_lens is not None:
        _need(seq_lens, torch.int32, (B,), "seq_lens", align=4)
    rc = lib().aila_hip_gqa_decode_noalloc(_ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(out), B, Hq, Hkv, D,
                                           max_seq, int(cached_len), _ptr(seq_lens), _stream(stream))
    _check(rc, "aila_hip_gqa_decode_noalloc")
    return out


def gqa_decode_append(q, k_new, v_new, k_cache, v_cache, pos: int, out=None, workspace=None,
                      positions=None, stream=None):
    """Write k_new/v_new [B,Hkv,D] to cache row pos (or positions[b] <= pos)
    and attend rows [0, row] -> out [B,Hq,D]."""
    import torch
    B, Hq, D = q.shape
    Hkv, max_seq = k_cache.shape[1], k_cache.shape[2]
    _need(q, torch.bfloat16, (B, Hq, D), "q")
    _need(k_new, torch.bfloat16, (B, Hkv, D), "k_new")
    _need(v_new, torch.bfloat16, (B, Hkv, D), "v_new")
    _need(k_cache, torch.bfloat16, (B, Hkv, max_seq, D), "k_cache")
    _need(v_cache, torch.bfloat16, (B, Hkv, max_seq, D), "v_cache")
    if out is None:
        out = torch.empty_like(q)
    _need(out, torch.bfloat16, (B, Hq, D), "out")
    ws_bytes = 0
    if workspace is not None:
        if not workspace.is_cuda or not workspace.is_contiguous():
            raise ValueError("workspace must be a contiguous device tensor")
        ws_bytes = workspace.numel() * workspace.element_size()
    if positions is not None:
        _need(positions, torch.int32, (B,), "positions", align=4)
    rc = lib().aila_hip_gqa_decode_append(_ptr(q), _ptr(k_new), _ptr(v_new), _ptr(k_cache), _ptr(v_cache),
                                          _ptr(out), _ptr(workspace), ws_bytes, B, Hq, Hkv, D, max_seq,
                                          int(pos), _ptr(positions), _stream(stream))
    _check(rc, "aila_hip_gqa_decode_append")
    return out


def kv_append(k_new, v_new, k_cache, v_cache, pos: int = 0, positions=None, stream=None):
    """k_new/v_new [B,Hkv,D] -> cache [B,Hkv,max_seq,D] row pos (or positions[b])."""
    import torch
    B, Hkv, max_seq, D = k_cache.shape
    _need(k_new, torch.bfloat16, (B, Hkv, D), "k_new")
    _need(v_new, torch.bfloat16, (B, Hkv, D), "v_new")
    _need(k_cache, torch.bfloat16, (B, Hkv, max_seq, D), "k_cache")
    _need(v_cache, torch.bfloat16, (B, Hkv, max_seq, D), "v_cache")
    if positions is not None:
        _need(positions, torch.int32, (B,), "positions", align=4)
    rc = lib().aila_hip_kv_append(_ptr(k_new), _ptr(v_new), _ptr(k_cache), _ptr(v_cache), B, Hkv, D,
                                  max_seq, int(pos), _ptr(positions), _stream(stream))
    _check(rc, "aila_hip_kv_append")


def gqa_prefill(q, k, v, Hq: int, Hkv: int, out=None, k_cache=None, v_cache=None,
                cache_pos: int = 0, stream=None):
    """Causal prefill. q [S, Hq*D], k/v [S, Hkv*D] bf16 -> out [S, Hq*D].
    With k_cache/v_cache [Hkv, max_seq, D], k/v are also written to cache
    rows [cache_pos, cache_pos + S)."""
    import torch
    S = q.shape[0]
    D = q.shape[1] // Hq
    _need(q, torch.bfloat16, (S, Hq * D), "q")
    _need(k, torch.bfloat16, (S, Hkv * D), "k")
    _need(v, torch.bfloat16, (S, Hkv * D), "v")
    if out is None:
        out = torch.empty_like(q)
    _need(out, torch.bfloat16, (S, Hq * D), "out")
    max_seq = 0
    if k_cache is not None or v_cache is not None:
        max_seq = k_cache.shape[1]
        _need(k_cache, torch.bfloat16, (Hkv, max_seq, D), "k_cache")
        _need(v_cache, torch.bfloat16, (Hkv, max_seq, D), "v_cache")
    rc = lib().aila_hip_gqa_prefill(_ptr(q), _ptr(k), _ptr(v), _ptr(out), _ptr(k_cache),
                                    _ptr(v_cache), int(cache_pos), max_seq, S, Hq, Hkv, D,
                                    _stream(stream))
    _check(rc, "aila_hip_gqa_prefill")
    return out


def gqa_prefill_cached_workspace_size(S: int, start_pos: int, Hq: int, Hkv: int, D: int) -> int:
    """Bytes of the key-split workspace gqa_prefill_cached would use (0: none)."""
    return int(lib().aila_hip_gqa_prefill_cached_workspace_size(S, start_pos, Hq, Hkv, D))


def gqa_prefill_cached(q, k_cache, v_cache, start_pos: int, Hq: int, out=None, workspace=None, stream=None):
    """q [S, Hq*D] at positions start_pos.. attends cache [Hkv, max_seq, D].
    workspace: a uint8 device tensor for the key split (see
    gqa_prefill_cached_workspace_size), or None for no split."""
    import torch
    S = q.shape[0]
    Hkv, max_seq, D = k_cache.shape
    _need(q, torch.bfloat16, (S, Hq * D), "q")
    _need(k_cache, torch.bfloat16, (Hkv, max_seq, D), "k_cache")
    _need(v_cache, torch.bfloat16, (Hkv, max_seq, D), "v_cache")
    if out is None:
        out = torch.empty_like(q)
    _need(out, torch.bfloat16, (S, Hq * D), "out")
    if workspace is None:
        rc = lib().aila_hip_gqa_prefill_cached(_ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(out), S,
                                               int(start_pos), Hq, Hkv, D, max_seq, _stream(stream))
    else:
        if not workspace.is_cuda or not workspace.is_contiguous():
            raise ValueError("workspace must be a contiguous device tensor")
        rc = lib().aila_hip_gqa_prefill_cached_ws(_ptr(q), _ptr(k_cache), _ptr(v_cache), _ptr(out),
                                                  _ptr(workspace), workspace.numel() * workspace.element_size(),
                                                  S, int(start_pos), Hq, Hkv, D, max_seq, _stream(stream))
    _check(rc, "aila_hip_gqa_prefill_cached")
    return out


def copy_to_cache(new_kv, cache, start_pos: int, stream=None):
    """new_kv [S, H*D] bf16 -> cache [H, max_seq, D] rows [start_pos, start_pos+S)."""
    import torch
    H, max_seq, D = cache.shape
    S = new_kv.shape[0]
    _need(new_kv, torch.bfloat16, (S, H * D), "new_kv")
    _need(cache, torch.bfloat16, (H, max_seq, D), "cache")
    rc = lib().aila_hip_copy_to_cache(_ptr(new_kv), _ptr(cache), S, int(start_pos), H, D, max_seq,
                                      _stream(stream))
    _check(rc, "aila_hip_copy_to_cache")
    return cache


# ------------------------------------------------ 8-bit paged KV cache ----
_SCALE_ROWS = 16   # rows of a page that share a scale


# As above, the common call tests everything in one expression (dtype, shape,
# layout, alignment, and that every tensor is on the call's device); only if that
# fails do these functions find out what is wrong and say it.
def _device_of(stream):
    import torch
    return torch.cuda.current_device() if stream is None else stream.device_index


def _same_device(dev, *tensors):
    """The tensors' one device has to be the one whose stream the call runs on."""
    for t in tensors:
        if t is not None and t.get_device() != dev:
            raise ValueError(f"tensor on {t.device}, but the call's stream is on cuda:{dev}: "
                             "make it inside torch.cuda.device(...), with all tensors there")


def _need_rows(t, tokens, heads, dim, name):
    """[tokens, heads, dim] bf16 whose tokens may be strided (views of a fused
    projection row)."""
    import torch
    if t is None:
        raise ValueError(f"{name} is required")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a device tensor")
    if t.dtype != torch.bfloat16:
        raise ValueError(f"{name}: dtype {t.dtype}, expected {torch.bfloat16}")
    if tuple(t.shape) != (tokens, heads, dim):
        raise ValueError(f"{name}: shape {tuple(t.shape)}, expected {(tokens, heads, dim)}")
    st = t.stride()
    if st[2] != 1 or (heads > 1 and st[1] != dim):
        raise ValueError(f"{name}: strides {st}, expected a token's [{heads}, {dim}] values to be contiguous")
    if tokens > 1 and (st[0] < heads * dim or st[0] % 8):
        raise ValueError(f"{name}: token stride {st[0]} must be a multiple of 8 and at least {heads * dim}")
    if t.data_ptr() % 16:
        raise ValueError(f"{name} must be 16-byte aligned")


def _token_stride(t, tokens, heads, dim):
    """Elements between tokens of a [tokens, heads, dim] view, or 0 if it is not
    one that the kernels take."""
    a, b, c = t.stride()
    if c != 1 or (b != dim and heads > 1):
        return 0
    if tokens == 1:
        return heads * dim
    return a if a >= heads * dim and not a % 8 else 0


def _need_pages(k_pages, v_pages, k_scale, v_scale):
    """Checks the four arrays of an 8-bit paged cache."""
    import torch
    if k_pages is None or k_pages.dim() != 4:
        raise ValueError("k_pages must be [num_pages, Hkv, page_size, D]")
    P, Hkv, page_size, _ = shape = tuple(k_pages.shape)
    if page_size % _SCALE_ROWS:
        raise ValueError(f"k_pages: page_size {page_size} must be a multiple of {_SCALE_ROWS}")
    _need(k_pages, torch.float8_e4m3fn, shape, "k_pages")
    _need(v_pages, torch.float8_e4m3fn, shape, "v_pages")
    _need(k_scale, torch.float32, (P, Hkv, page_size // _SCALE_ROWS), "k_scale", align=4)
    _need(v_scale, torch.float32, (P, Hkv, page_size // _SCALE_ROWS), "v_scale", align=4)


def _pages_ok(torch, dev, kp, vp, ks, vs):
    """(k_pages.shape, pointers of the four) if all is as it has to be, else None."""
    shape = kp.shape
    if len(shape) != 4:
        return None
    f8, f32 = torch.float8_e4m3fn, torch.float32
    p = kp.data_ptr(), vp.data_ptr(), ks.data_ptr(), vs.data_ptr()
    if kp.dtype is f8 and vp.dtype is f8 and ks.dtype is f32 and vs.dtype is f32 and vp.shape == shape \
            and ks.shape == vs.shape == (shape[0], shape[1], shape[2] // _SCALE_ROWS) and not shape[2] % _SCALE_ROWS \
            and not (p[0] | p[1]) & 15 and not (p[2] | p[3]) & 3 and kp.is_contiguous() and vp.is_contiguous() \
            and ks.is_contiguous() and vs.is_contiguous() \
            and kp.get_device() == vp.get_device() == ks.get_device() == vs.get_device() == dev:
        return shape, p
    return None


def _new_out(make, stream):
    """An output for work on `stream`, from that stream's memory."""
    import torch
    if stream is None:
        return make()
    with torch.cuda.stream(stream):
        return make()


def _workspace_bytes(workspace):
    if workspace is None:
        return 0
    if not workspace.is_cuda or not workspace.is_contiguous():
        raise ValueError("workspace must be a contiguous device tensor")
    return workspace.numel() * workspace.element_size()


def paged_fp8_cache(num_pages: int, Hkv: int, page_size: int, D: int, device=None):
    """An empty 8-bit paged cache: (k_pages, v_pages, k_scale, v_scale)."""
    import torch
    if page_size <= 0 or page_size % _SCALE_ROWS:
        raise ValueError(f"page_size {page_size} must be a positive multiple of {_SCALE_ROWS}")
    dev = device if device is not None else torch.device("cuda", torch.cuda.current_device())
    pages = [torch.zeros((num_pages, Hkv, page_size, D), dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)
             for _ in range(2)]
    scales = [torch.ones((num_pages, Hkv, page_size // _SCALE_ROWS), dtype=torch.float32, device=dev) for _ in range(2)]
    return (*pages, *scales)


def kv_pages_reserve(cached_lens, new_lens, block_table, free_pages, free_count, page_size: int, slots,
                     query_start=None, seq_lens=None, stream=None):
    """Pages and slots for B requests' new tokens, on the device. cached_lens,
    new_lens int32 [B]; block_table int32 [B, max_pages] (-1: no page yet);
    free_pages int32 [num_pages], a stack whose entries [0, free_count[0]) are
    free; slots int32 [max_tokens] (written whole). -> (query_start [B+1],
    seq_lens [B], slots). seq_lens is 0 for requests that did not fit the
    table, the batch or the free pages; their slots are -1, and the rows and
    pages that they had stay theirs: the next call's cached_lens are
    torch.where(seq_lens > 0, seq_lens, cached_lens), not seq_lens."""
    import torch
    B, max_pages = block_table.shape
    i32 = torch.int32
    if query_start is None:
        query_start = _new_out(lambda: torch.empty(B + 1, dtype=i32, device=block_table.device), stream)
    if seq_lens is None:
        seq_lens = _new_out(lambda: torch.empty(B, dtype=i32, device=block_table.device), stream)
    dev = _device_of(stream)
    num_pages, max_tokens = free_pages.numel(), slots.numel()
    one = (B,)
    if not (cached_lens.dtype is i32 and new_lens.dtype is i32 and block_table.dtype is i32 and free_pages.dtype is i32
            and free_count.dtype is i32 and slots.dtype is i32 and query_start.dtype is i32 and seq_lens.dtype is i32
            and cached_lens.shape == new_lens.shape == seq_lens.shape == one and query_start.shape == (B + 1,)
            and free_count.shape == (1,) and free_pages.shape == (num_pages,) and slots.shape == (max_tokens,)
            and cached_lens.is_contiguous() and new_lens.is_contiguous() and block_table.is_contiguous()
            and free_pages.is_contiguous() and slots.is_contiguous() and query_start.is_contiguous()
            and seq_lens.is_contiguous() and cached_lens.get_device() == new_lens.get_device() == block_table.get_device()
            == free_pages.get_device() == free_count.get_device() == slots.get_device() == query_start.get_device()
            == seq_lens.get_device() == dev):
        _need(cached_lens, i32, one, "cached_lens", align=4)
        _need(new_lens, i32, one, "new_lens", align=4)
        _need(block_table, i32, (B, max_pages), "block_table", align=4)
        _need(free_pages, i32, (num_pages,), "free_pages", align=4)
        _need(free_count, i32, (1,), "free_count", align=4)
        _need(slots, i32, (max_tokens,), "slots", align=4)
        _need(query_start, i32, (B + 1,), "query_start", align=4)
        _need(seq_lens, i32, one, "seq_lens", align=4)
        _same_device(dev, block_table, cached_lens, new_lens, free_pages, free_count, slots, query_start, seq_lens)
    rc = lib().aila_hip_kv_pages_reserve(cached_lens.data_ptr(), new_lens.data_ptr(), block_table.data_ptr(),
                                         free_pages.data_ptr(), free_count.data_ptr(), query_start.data_ptr(),
                                         seq_lens.data_ptr(), slots.data_ptr(), B, max_pages, int(page_size), num_pages,
                                         max_tokens, _stream(stream))
    if rc:
        _check(rc, "aila_hip_kv_pages_reserve")
    return query_start, seq_lens, slots


def kv_pages_release(release, block_table, free_pages, free_count, stream=None):
    """Push the pages of the rows with release[b] != 0 (int32 [B]) back onto the
    free stack; their table entries become -1."""
    import torch
    B, max_pages = block_table.shape
    i32 = torch.int32
    dev = _device_of(stream)
    num_pages = free_pages.numel()
    if not (release.dtype is i32 and block_table.dtype is i32 and free_pages.dtype is i32 and free_count.dtype is i32
            and release.shape == (B,) and free_pages.shape == (num_pages,) and free_count.shape == (1,)
            and release.is_contiguous() and block_table.is_contiguous() and free_pages.is_contiguous()
            and release.get_device() == block_table.get_device() == free_pages.get_device() == free_count.get_device() == dev):
        _need(release, i32, (B,), "release", align=4)
        _need(block_table, i32, (B, max_pages), "block_table", align=4)
        _need(free_pages, i32, (num_pages,), "free_pages", align=4)
        _need(free_count, i32, (1,), "free_count", align=4)
        _same_device(dev, block_table, release, free_pages, free_count)
    rc = lib().aila_hip_kv_pages_release(release.data_ptr(), block_table.data_ptr(), free_pages.data_ptr(),
                                         free_count.data_ptr(), B, max_pages, num_pages, _stream(stream))
    if rc:
        _check(rc, "aila_hip_kv_pages_release")


def kv_append_paged_fp8(k_new, v_new, k_pages, v_pages, k_scale, v_scale, slots, stream=None):
    """Quantise k_new/v_new [T, Hkv, D] bf16 into the rows `slots` (int32 [T],
    -1: skip) of an 8-bit paged cache: k_pages/v_pages [num_pages, Hkv,
    page_size, D] float8_e4m3fn, k_scale/v_scale [num_pages, Hkv,
    page_size / 16] float32. The tokens may be strided (both alike)."""
    import torch
    dev = _device_of(stream)
    T = slots.numel()
    bf = torch.bfloat16
    pages = _pages_ok(torch, dev, k_pages, v_pages, k_scale, v_scale) if k_pages is not None else None
    ok = pages is not None and k_new is not None and v_new is not None
    if ok:
        (P, Hkv, page_size, D), (kp, vp, ks, vs) = pages
        kn, vn = k_new.data_ptr(), v_new.data_ptr()
        ok = k_new.dtype is bf and v_new.dtype is bf and slots.dtype is torch.int32 and k_new.shape == v_new.shape == (T, Hkv, D) \
            and slots.shape == (T,) and slots.is_contiguous() and not (kn | vn) & 15 \
            and k_new.get_device() == v_new.get_device() == slots.get_device() == dev
        if ok:
            step = _token_stride(k_new, T, Hkv, D)
            ok = step and step == _token_stride(v_new, T, Hkv, D)
    if not ok:
        _need_pages(k_pages, v_pages, k_scale, v_scale)
        P, Hkv, page_size, D = k_pages.shape
        _need(slots, torch.int32, (T,), "slots", align=4)
        _need_rows(k_new, T, Hkv, D, "k_new")
        _need_rows(v_new, T, Hkv, D, "v_new")
        if k_new.stride(0) != v_new.stride(0):
            raise ValueError(f"k_new and v_new: token strides {k_new.stride(0)} and {v_new.stride(0)} differ")
        _same_device(dev, k_pages, v_pages, k_scale, v_scale, k_new, v_new, slots)
        raise ValueError("kv_append_paged_fp8: bad tensors")
    rc = lib().aila_hip_kv_append_paged_fp8(kn, vn, step, kp, vp, ks, vs, slots.data_ptr(), T, Hkv, D, page_size, P,
                                            _stream(stream))
    if rc:
        _check(rc, "aila_hip_kv_append_paged_fp8")


def kv_read_paged_fp8(k_pages, v_pages, k_scale, v_scale, slots, k_out=None, v_out=None, stream=None):
    """Rows `slots` (int32 [T]; zeros for -1) of an 8-bit paged cache as the
    values they stand for -> (k, v) [T, Hkv, D] bf16."""
    import torch
    dev = _device_of(stream)
    T = slots.numel()
    bf = torch.bfloat16
    pages = _pages_ok(torch, dev, k_pages, v_pages, k_scale, v_scale) if k_pages is not None else None
    if pages is None:
        _need_pages(k_pages, v_pages, k_scale, v_scale)
        _same_device(dev, k_pages, v_pages, k_scale, v_scale)
        raise ValueError("kv_read_paged_fp8: bad cache tensors")
    (P, Hkv, page_size, D), (kp, vp, ks, vs) = pages
    shape = (T, Hkv, D)
    if k_out is None:
        k_out = _new_out(lambda: torch.empty(shape, dtype=bf, device=k_pages.device), stream)
    if v_out is None:
        v_out = _new_out(lambda: torch.empty(shape, dtype=bf, device=k_pages.device), stream)
    ko, vo = k_out.data_ptr(), v_out.data_ptr()
    if not (k_out.dtype is bf and v_out.dtype is bf and slots.dtype is torch.int32 and k_out.shape == v_out.shape == shape
            and slots.shape == (T,) and slots.is_contiguous() and k_out.is_contiguous() and v_out.is_contiguous()
            and not (ko | vo) & 15 and k_out.get_device() == v_out.get_device() == slots.get_device() == dev):
        _need(slots, torch.int32, (T,), "slots", align=4)
        _need(k_out, bf, shape, "k_out")
        _need(v_out, bf, shape, "v_out")
        _same_device(dev, slots, k_out, v_out)
    rc = lib().aila_hip_kv_read_paged_fp8(kp, vp, ks, vs, slots.data_ptr(), ko, vo, T, Hkv, D, page_size, P, _stream(stream))
    if rc:
        _check(rc, "aila_hip_kv_read_paged_fp8")
    return k_out, v_out


def gqa_decode_paged_fp8_workspace_size(B: int, Hq: int, Hkv: int, D: int, max_len: int) -> int:
    return int(lib().aila_hip_gqa_decode_paged_fp8_workspace_size(B, Hq, Hkv, D, max_len))


def _attention_args(q, k_pages, v_pages, k_scale, v_scale, block_table, query_start, seq_lens, out, workspace, stream, B):
    """Checks what both attention calls take; returns the token stride of q, the
    cache's shape and pointers, out and the workspace's pointer and size."""
    import torch
    dev = _device_of(stream)
    T, Hq, D = q.shape
    bf, i32 = torch.bfloat16, torch.int32
    if out is None:
        out = _new_out(lambda: torch.empty((T, Hq, D), dtype=q.dtype, device=q.device), stream)
    pages = _pages_ok(torch, dev, k_pages, v_pages, k_scale, v_scale) if k_pages is not None else None
    step = _token_stride(q, T, Hq, D)
    if not (pages is not None and step and q.dtype is bf and out.dtype is bf and block_table.dtype is i32 and seq_lens.dtype is i32
            and pages[0][3] == D and out.shape == q.shape and seq_lens.shape == (B,) and block_table.shape[0] == B
            and len(block_table.shape) == 2 and out.is_contiguous() and block_table.is_contiguous() and seq_lens.is_contiguous()
            and not (q.data_ptr() | out.data_ptr()) & 15
            and q.get_device() == out.get_device() == block_table.get_device() == seq_lens.get_device() == dev
            and (query_start is None or (query_start.dtype is i32 and query_start.shape == (B + 1,) and query_start.is_contiguous()
                                         and query_start.get_device() == dev))
            and (workspace is None or (workspace.get_device() == dev and workspace.is_contiguous()))):
        _need_pages(k_pages, v_pages, k_scale, v_scale)
        _need_rows(q, T, Hq, k_pages.shape[3], "q")
        _need(block_table, i32, (B, block_table.shape[1]), "block_table", align=4)
        _need(seq_lens, i32, (B,), "seq_lens", align=4)
        if query_start is not None:
            _need(query_start, i32, (B + 1,), "query_start", align=4)
        _need(out, bf, (T, Hq, D), "out")
        _workspace_bytes(workspace)
        _same_device(dev, q, k_pages, v_pages, k_scale, v_scale, block_table, query_start, seq_lens, out, workspace)
        raise ValueError("bad tensors")
    if workspace is None:
        return step, pages, out, None, 0
    return step, pages, out, workspace.data_ptr(), workspace.numel() * workspace.element_size()


def gqa_decode_paged_fp8(q, k_pages, v_pages, k_scale, v_scale, block_table, seq_lens, max_len: int, out=None,
                         workspace=None, stream=None):
    """Decode over an 8-bit paged cache. q [B,Hq,D] bf16 (sequences may be
    strided); the cache as kv_append_paged_fp8; block_table int32 [B,
    max_pages]; seq_lens int32 [B] (taken as max_len where larger) -> out
    [B,Hq,D]. Row b of q is sequence b's, which is the order of
    kv_pages_reserve's tokens only if each request adds exactly one (else gather
    q[query_start[:B].clamp(max=T - 1)], or call gqa_prefill_paged_fp8).
    workspace: uint8 device tensor (see gqa_decode_paged_fp8_workspace_size), or
    None for one workgroup per sequence and KV head."""
    B, Hq, D = q.shape
    step, ((P, Hkv, page_size, _), (kp, vp, ks, vs)), out, ws, ws_bytes = _attention_args(
        q, k_pages, v_pages, k_scale, v_scale, block_table, None, seq_lens, out, workspace, stream, B)
    rc = lib().aila_hip_gqa_decode_paged_fp8(q.data_ptr(), step, kp, vp, ks, vs, out.data_ptr(), ws, ws_bytes, B, Hq, Hkv, D,
                                             page_size, P, block_table.data_ptr(), block_table.shape[1], int(max_len),
                                             seq_lens.data_ptr(), _stream(stream))
    if rc:
        _check(rc, "aila_hip_gqa_decode_paged_fp8")
    return out


def gqa_prefill_paged_fp8_workspace_size(T: int, B: int, Hq: int, Hkv: int, D: int, max_len: int) -> int:
    return int(lib().aila_hip_gqa_prefill_paged_fp8_workspace_size(T, B, Hq, Hkv, D, max_len))


def gqa_prefill_paged_fp8(q, k_pages, v_pages, k_scale, v_scale, block_table, query_start, seq_lens, max_len: int,
                          out=None, workspace=None, stream=None):
    """Causal attention of a ragged batch over an 8-bit paged cache that holds
    the new rows already. q [T,Hq,D] bf16, request b's tokens at query_start[b]
    .. query_start[b+1] (int32 [B+1]); seq_lens int32 [B] counts the rows after
    them -> out [T,Hq,D] (rows from query_start[B] on are not touched).
    workspace: uint8 device tensor (see gqa_prefill_paged_fp8_workspace_size);
    None: one request, or one after the other, and no key split."""
    T, Hq, D = q.shape
    B, max_pages = block_table.shape
    if query_start is None:
        raise ValueError("query_start is required")
    step, ((P, Hkv, page_size, _), (kp, vp, ks, vs)), out, ws, ws_bytes = _attention_args(
        q, k_pages, v_pages, k_scale, v_scale, block_table, query_start, seq_lens, out, workspace, stream, B)
    rc = lib().aila_hip_gqa_prefill_paged_fp8(q.data_ptr(), step, kp, vp, ks, vs, out.data_ptr(), ws, ws_bytes, T, B, Hq, Hkv,
                                              D, page_size, P, block_table.data_ptr(), max_pages, int(max_len),
                                              query_start.data_ptr(), seq_lens.data_ptr(), _stream(stream))
    if rc:
        _check(rc, "aila_hip_gqa_prefill_paged_fp8")
    return out


# ---------------------- drafts, forks and trims over the 8-bit paged cache ----
def _head_strides(t, tokens, heads, dim):
    """(token, head) strides of a [tokens, heads, dim] view whose heads may stand
    apart, or (0, 0) if it is not one that the kernels take."""
    a, b, c = t.stride()
    if heads == 1:
        b = dim
    if tokens == 1:
        a = (heads - 1) * b + dim
        a += -a % 8
    ok = c == 1 and b >= dim and not b % 8 and a >= (heads - 1) * b + dim and not a % 8
    return (a, b) if ok else (0, 0)


def prepare_qkv_paged_fp8(q, k, v, k_pages, v_pages, k_scale, v_scale, slots, positions, q_norm=None, k_norm=None,
                          rotary_dim=None, theta: float = 1e6, eps: float = 1e-6, sections=None, inv_freq=None, q_out=None,
                          stream=None):
    """Between a layer's projection and its attention over an 8-bit paged cache.
    q [T,Hq,D], k/v [T,Hkv,D] bf16 (tokens may be strided, q's heads too: a view
    of packed q|gate rows); per-head RMSNorm of q and k with weights q_norm,
    k_norm [D] bf16 (None: 1); the first rotary_dim dims (None: D; a multiple
    of 8, 0: none) turned at positions int32 [T], or [3,T]: the t, h and w
    streams of interleaved mRoPE with ``sections`` (t, h, w); k and v quantised
    into the rows ``slots`` (int32 [T], -1: skip) as kv_append_paged_fp8 does
    -> q_out [T,Hq,D] bf16 (may be q itself, if contiguous; refused where it
    overlaps q, k or v otherwise). inv_freq: float32 [rotary_dim/2] in place of theta^(-2d/rotary_dim)."""
    import torch
    dev = _device_of(stream)
    T, Hq, D = q.shape
    bf, i32 = torch.bfloat16, torch.int32
    rot = D if rotary_dim is None else int(rotary_dim)
    if q_out is None:
        q_out = _new_out(lambda: torch.empty((T, Hq, D), dtype=bf, device=q.device), stream)
    pages = _pages_ok(torch, dev, k_pages, v_pages, k_scale, v_scale) if k_pages is not None else None
    ok = pages is not None and k is not None and v is not None
    streams = 0 if positions is None else 1 if positions.dim() == 1 else 3
    if ok:
        (P, Hkv, page_size, _), (kp, vp, ks, vs) = pages
        qs, qh = _head_strides(q, T, Hq, D)
        ok = qs and pages[0][3] == D and k.shape == v.shape == (T, Hkv, D) and q.dtype is bf and k.dtype is bf and v.dtype is bf \
            and q_out.dtype is bf and q_out.shape == (T, Hq, D) and q_out.is_contiguous() and slots.dtype is i32 \
            and slots.shape == (T,) and slots.is_contiguous() \
            and not (q.data_ptr() | k.data_ptr() | v.data_ptr() | q_out.data_ptr()) & 15 \
            and q.get_device() == k.get_device() == v.get_device() == q_out.get_device() == slots.get_device() == dev
    if ok:
        k_step, v_step = _token_stride(k, T, Hkv, D), _token_stride(v, T, Hkv, D)
        ok = k_step and v_step \
            and (q_norm is None or (q_norm.dtype is bf and q_norm.shape == (D,) and q_norm.is_contiguous() and q_norm.get_device() == dev)) \
            and (k_norm is None or (k_norm.dtype is bf and k_norm.shape == (D,) and k_norm.is_contiguous() and k_norm.get_device() == dev)) \
            and (positions is None or (positions.dtype is i32 and positions.shape == ((T,) if streams == 1 else (3, T))
                                       and positions.is_contiguous() and positions.get_device() == dev)) \
            and (inv_freq is None or (inv_freq.dtype is torch.float32 and inv_freq.shape == (rot // 2,) and inv_freq.is_contiguous()
                                      and inv_freq.get_device() == dev))
    if not ok:
        _need_pages(k_pages, v_pages, k_scale, v_scale)
        P, Hkv, page_size, _ = k_pages.shape
        _need_rows(k, T, Hkv, k_pages.shape[3], "k")
        _need_rows(v, T, Hkv, k_pages.shape[3], "v")
        if not q.is_cuda or q.dtype != bf or D != k_pages.shape[3] or q.data_ptr() % 16:
            raise ValueError(f"q: {q.dtype} of head dim {D} on {q.device}, expected 16-byte aligned bfloat16 device data of {k_pages.shape[3]}")
        if not _head_strides(q, T, Hq, D)[0]:
            raise ValueError(f"q: strides {q.stride()}, expected contiguous dims, and tokens and heads multiples of 8 apart")
        _need(q_out, bf, (T, Hq, D), "q_out")
        _need(slots, i32, (T,), "slots", align=4)
        for t, name in ((q_norm, "q_norm"), (k_norm, "k_norm")):
            if t is not None:
                _need(t, bf, (D,), name)
        if positions is not None:
            _need(positions, i32, (T,) if streams == 1 else (3, T), "positions", align=4)
        if inv_freq is not None:
            _need(inv_freq, torch.float32, (rot // 2,), "inv_freq", align=4)
        _same_device(dev, q, k, v, k_pages, v_pages, k_scale, v_scale, q_out, slots, q_norm, k_norm, positions, inv_freq)
        raise ValueError("prepare_qkv_paged_fp8: bad tensors")
    if streams == 3 and sections is None:
        raise ValueError("positions [3, T] need sections (t, h, w)")
    pos = _ptr(positions)
    _, sh, sw = (0, 0, 0) if streams != 3 else (int(x) for x in sections)
    rc = lib().aila_hip_prepare_qkv_paged_fp8(
        q.data_ptr(), qs, qh, k.data_ptr(), k_step, v.data_ptr(), v_step, q_out.data_ptr(), _ptr(q_norm), _ptr(k_norm), kp, vp, ks, vs,
        slots.data_ptr(), pos, pos + 4 * T if streams == 3 else None, pos + 8 * T if streams == 3 else None, sh, sw, T, Hq, Hkv, D,
        page_size, P, rot, float(theta), _ptr(inv_freq), float(eps), _stream(stream))
    if rc:
        _check(rc, "aila_hip_prepare_qkv_paged_fp8")
    return q_out


def gqa_tree_paged_fp8_workspace_size(T: int, B: int, Hq: int, Hkv: int, D: int, max_len: int, mask_words: int) -> int:
    return int(lib().aila_hip_gqa_tree_paged_fp8_workspace_size(T, B, Hq, Hkv, D, max_len, mask_words))


def gqa_tree_paged_fp8(q, k_pages, v_pages, k_scale, v_scale, block_table, query_start, seq_lens, tree_mask, max_len: int,
                       out=None, workspace=None, stream=None):
    """Attention of drafted trees over an 8-bit paged cache that holds the
    drafted rows already. Arguments as gqa_prefill_paged_fp8; tree_mask int64
    [T, W], W <= 64: token i of a request attends its rows before the draft and
    the drafted token j if bit j % 64 of tree_mask[i, j // 64] is set (its own
    bit too, if it is to attend itself). A request has 64 W tokens at most.
    workspace: uint8 device tensor (see gqa_tree_paged_fp8_workspace_size), or
    None: no key split."""
    import torch
    T, Hq, D = q.shape
    B, max_pages = block_table.shape
    if query_start is None:
        raise ValueError("query_start is required")
    if tree_mask is None or tree_mask.dim() != 2:
        raise ValueError("tree_mask must be [T, words]")
    words = tree_mask.shape[1]
    step, ((P, Hkv, page_size, _), (kp, vp, ks, vs)), out, ws, ws_bytes = _attention_args(
        q, k_pages, v_pages, k_scale, v_scale, block_table, query_start, seq_lens, out, workspace, stream, B)
    if not (tree_mask.dtype is torch.int64 and tree_mask.shape[0] == T and tree_mask.is_contiguous()
            and tree_mask.get_device() == q.get_device()):
        _need(tree_mask, torch.int64, (T, words), "tree_mask", align=8)
        _same_device(q.get_device(), tree_mask)
    rc = lib().aila_hip_gqa_tree_paged_fp8(q.data_ptr(), step, kp, vp, ks, vs, out.data_ptr(), ws, ws_bytes, T, B, Hq, Hkv, D,
                                           page_size, P, block_table.data_ptr(), max_pages, int(max_len), query_start.data_ptr(),
                                           seq_lens.data_ptr(), tree_mask.data_ptr(), words, _stream(stream))
    if rc:
        _check(rc, "aila_hip_gqa_tree_paged_fp8")
    return out


_SHAPE, _DTYPE = operator.attrgetter("shape"), operator.attrgetter("dtype")


def _layer_pointers(caches, dev):
    """(layers, shape of a cache, addresses of the four host arrays of device
    pointers, what keeps them) of one cache (k_pages, v_pages, k_scale, v_scale)
    or a list of such."""
    import torch
    if not caches:
        raise ValueError("no caches")
    if torch.is_tensor(caches[0]):
        caches = [caches]
    # a hundred tensors in a deep stack: looked at attribute by attribute, in loops of C
    n, flat = len(caches), list(itertools.chain.from_iterable(caches))
    ok = len(flat) == 4 * n and all([t is not None for t in flat])
    if ok:
        kind, shape, scales = type(flat[0]), flat[0].shape, flat[2].shape
        pages, scale = flat[0::4] + flat[1::4], flat[2::4] + flat[3::4]
        ok = all(map(kind.is_contiguous, flat)) and list(map(kind.get_device, flat)).count(dev) == 4 * n \
            and len(shape) == 4 and not shape[2] % _SCALE_ROWS and scales == (shape[0], shape[1], shape[2] // _SCALE_ROWS) \
            and list(map(_SHAPE, pages)).count(shape) == list(map(_SHAPE, scale)).count(scales) == 2 * n \
            and list(map(_DTYPE, pages)).count(torch.float8_e4m3fn) == list(map(_DTYPE, scale)).count(torch.float32) == 2 * n
    if ok:
        ptrs = array.array("Q", list(map(kind.data_ptr, pages + scale)))
        ok = not functools.reduce(operator.or_, ptrs[:2 * n]) & 15
    if not ok:
        for c in caches:
            if len(c) != 4:
                raise ValueError("a cache is (k_pages, v_pages, k_scale, v_scale)")
            _need_pages(*c)
            if c[0].shape != caches[0][0].shape:
                raise ValueError(f"caches: pages {tuple(c[0].shape)} beside {tuple(caches[0][0].shape)}")
            _same_device(dev, *c)
        raise ValueError("bad cache tensors")
    at = ptrs.buffer_info()[0]
    return n, shape, (at, at + 8 * n, at + 16 * n, at + 24 * n), ptrs


def kv_keep_paged_fp8(caches, block_table, cached_lens, kept, kept_lens, lens=None, stream=None):
    """Keep the accepted rows of drafts, in all layers: row cached_lens[b] +
    kept[b, i] of request b becomes row cached_lens[b] + i for i < kept_lens[b].
    caches: one (k_pages, v_pages, k_scale, v_scale) or a list of them, a layer
    each, of one shape; cached_lens int32 [B] (rows before the draft; negative:
    absent), kept int32 [B, max_kept] (rising in each row), kept_lens int32 [B]
    -> lens int32 [B], cached_lens + kept_lens."""
    import torch
    dev = _device_of(stream)
    B, max_pages = block_table.shape
    i32 = torch.int32
    if kept.dim() != 2:
        raise ValueError("kept must be [B, max_kept]")
    most = kept.shape[1]
    if lens is None:
        lens = _new_out(lambda: torch.empty(B, dtype=i32, device=block_table.device), stream)
    n, (P, Hkv, page_size, D), ptrs, kept_alive = _layer_pointers(caches, dev)  # noqa: F841
    one = (B,)
    if not (block_table.dtype is i32 and cached_lens.dtype is i32 and kept.dtype is i32 and kept_lens.dtype is i32 and lens.dtype is i32
            and cached_lens.shape == kept_lens.shape == lens.shape == one and kept.shape[0] == B and block_table.is_contiguous()
            and cached_lens.is_contiguous() and kept.is_contiguous() and kept_lens.is_contiguous() and lens.is_contiguous()
            and block_table.get_device() == cached_lens.get_device() == kept.get_device() == kept_lens.get_device()
            == lens.get_device() == dev):
        _need(block_table, i32, (B, max_pages), "block_table", align=4)
        _need(cached_lens, i32, one, "cached_lens", align=4)
        _need(kept, i32, (B, most), "kept", align=4)
        _need(kept_lens, i32, one, "kept_lens", align=4)
        _need(lens, i32, one, "lens", align=4)
        _same_device(dev, block_table, cached_lens, kept, kept_lens, lens)
    rc = lib().aila_hip_kv_keep_paged_fp8(*ptrs, n, block_table.data_ptr(), cached_lens.data_ptr(), kept.data_ptr(),
                                          kept_lens.data_ptr(), lens.data_ptr(), B, most, Hkv, D, page_size, P, max_pages, _stream(stream))
    if rc:
        _check(rc, "aila_hip_kv_keep_paged_fp8")
    return lens


def kv_pages_trim(lens, block_table, free_pages, free_count, page_size: int, stream=None):
    """Push the pages behind each request's rows (lens int32 [B]; negative: leave
    the row alone), up to the first entry that holds none, back onto the free
    stack; their table entries become -1."""
    import torch
    B, max_pages = block_table.shape
    i32 = torch.int32
    dev = _device_of(stream)
    num_pages = free_pages.numel()
    if not (lens.dtype is i32 and block_table.dtype is i32 and free_pages.dtype is i32 and free_count.dtype is i32
            and lens.shape == (B,) and free_pages.shape == (num_pages,) and free_count.shape == (1,)
            and lens.is_contiguous() and block_table.is_contiguous() and free_pages.is_contiguous()
            and lens.get_device() == block_table.get_device() == free_pages.get_device() == free_count.get_device() == dev):
        _need(lens, i32, (B,), "lens", align=4)
        _need(block_table, i32, (B, max_pages), "block_table", align=4)
        _need(free_pages, i32, (num_pages,), "free_pages", align=4)
        _need(free_count, i32, (1,), "free_count", align=4)
        _same_device(dev, block_table, lens, free_pages, free_count)
    rc = lib().aila_hip_kv_pages_trim(lens.data_ptr(), block_table.data_ptr(), free_pages.data_ptr(), free_count.data_ptr(), B,
                                      max_pages, int(page_size), num_pages, _stream(stream))
    if rc:
        _check(rc, "aila_hip_kv_pages_trim")


def kv_copy_paged_fp8(caches, block_table, src, dst, lens, max_len: int, stream=None):
    """Copy rows [0, lens[i]) (int32 [n], taken as max_len where larger) of row
    src[i] of block_table to the pages of row dst[i] (int32 [n] each), in all
    layers (caches as kv_keep_paged_fp8): forks, whose pages kv_pages_reserve
    has taken. Whole blocks of 16 rows are copied."""
    import torch
    dev = _device_of(stream)
    B, max_pages = block_table.shape
    i32 = torch.int32
    n, (P, Hkv, page_size, D), ptrs, kept_alive = _layer_pointers(caches, dev)  # noqa: F841
    pairs = src.numel()
    one = (pairs,)
    if not (block_table.dtype is i32 and src.dtype is i32 and dst.dtype is i32 and lens.dtype is i32
            and src.shape == dst.shape == lens.shape == one and block_table.is_contiguous() and src.is_contiguous()
            and dst.is_contiguous() and lens.is_contiguous()
            and block_table.get_device() == src.get_device() == dst.get_device() == lens.get_device() == dev):
        _need(block_table, i32, (B, max_pages), "block_table", align=4)
        _need(src, i32, one, "src", align=4)
        _need(dst, i32, one, "dst", align=4)
        _need(lens, i32, one, "lens", align=4)
        _same_device(dev, block_table, src, dst, lens)
    rc = lib().aila_hip_kv_copy_paged_fp8(*ptrs, n, block_table.data_ptr(), src.data_ptr(), dst.data_ptr(), lens.data_ptr(), pairs,
                                          int(max_len), B, Hkv, D, page_size, P, max_pages, _stream(stream))
    if rc:
        _check(rc, "aila_hip_kv_copy_paged_fp8")


# ------------------------------------------------------------ DeltaNet ----
def deltanet_decode(q, k, v, a, b, state, out=None, dt_bias=None, A_log=None,
                    eps: float = 1e-6, scale: float | None = None, stream=None):
    """One Gated DeltaNet step. q,k [B,Hk,dk] bf16; v [B,Hv,dv] bf16;
    a,b [B,Hv] bf16; state [B,Hv,dk,dv] fp32 (updated in place) -> out
    [B,Hv,dv] bf16."""
    import torch
    B, Hk, dk = q.shape
    Hv, dv = v.shape[1], v.shape[2]
    _need(q, torch.bfloat16, (B, Hk, dk), "q")
    _need(k, torch.bfloat16, (B, Hk, dk), "k")
    _need(v, torch.bfloat16, (B, Hv, dv), "v")
    _need(a, torch.bfloat16, (B, Hv), "a", align=2)
    _need(b, torch.bfloat16, (B, Hv), "b", align=2)
    _need(state, torch.float32, (B, Hv, dk, dv), "state")
    if dt_bias is not None:
        _need(dt_bias, torch.bfloat16, (Hv,), "dt_bias", align=2)
    if A_log is not None:
        _need(A_log, torch.float32, (Hv,), "A_log", align=4)
    if out is None:
        out = torch.empty((B, Hv, dv), dtype=torch.bfloat16, device=q.device)
    _need(out, torch.bfloat16, (B, Hv, dv), "out")
    if scale is None:
        scale = 1.0 / math.sqrt(dk)
    rc = lib().aila_hip_deltanet_decode(_ptr(q), _ptr(k), _ptr(v), _ptr(a), _ptr(b),
                                        _ptr(dt_bias), _ptr(A_log), _ptr(state), _ptr(out),
                                        B, Hk, Hv, dk, dv, float(eps), float(scale),
                                        _stream(stream))
    _check(rc, "aila_hip_deltanet_decode")
    return out


def _rows(t, dtype, B, width, name, align=2):
    """A [B, width] view whose rows may be strided (e.g. column slices of the
    backend's fused [qkv | z | a | b] rows); returns the row stride."""
    if t is None or not t.is_cuda or t.dtype != dtype:
        raise ValueError(f"{name}: expected a {dtype} device tensor")
    if t.shape != (B, width) or (width > 1 and t.stride(1) != 1):
        raise ValueError(f"{name}: shape {tuple(t.shape)} / strides {t.stride()}, expected [{B}, {width}] "
                         "with unit column stride")
    if t.data_ptr() % align:
        raise ValueError(f"{name} must be {align}-byte aligned")
    return t.stride(0) if B > 1 else width


def deltanet_layer_decode(qkv, z, a, b, conv_w, conv_state, conv_head, norm_w, state, num_k_heads,
                          out=None, conv_heads=None, dt_bias=None, A_log=None, eps: float = 1e-6,
                          scale: float | None = None, arrivals=None, stream=None):
    """Full Gated DeltaNet layer step for B sequences: conv1d ring (+SiLU),
    L2 norm, gated delta recurrence, RMSNorm(o) * norm_w * SiLU(z).

    qkv [B, 2*Hk*dk + Hv*dv], z [B, Hv*dv], a/b [B, Hv] bf16 (rows may be
    strided views); conv_w [ch, 4] bf16; conv_state [B, 3, ch] fp32 and
    state [B, Hv, dk, dv] fp32 are updated in place; conv_head (int) or
    conv_heads (int32 [B], device) gives the ring row of the oldest input.
    ``arrivals``: optional int32 [B*Hk] device tensor, zero before the first
    call (every call leaves it zero): one workgroup per value head instead
    of one per key head. Returns out [B, Hv*dv] bf16."""
    import torch
    B, Hv, dk, dv = state.shape
    Hk = int(num_k_heads)
    ch = 2 * Hk * dk + Hv * dv
    qs = _rows(qkv, torch.bfloat16, B, ch, "qkv")
    zs = _rows(z, torch.bfloat16, B, Hv * dv, "z", align=8)
    ast = _rows(a, torch.bfloat16, B, Hv, "a")
    bst = _rows(b, torch.bfloat16, B, Hv, "b")
    if ast != bst:
        raise ValueError("a and b must share one row stride")
    K = conv_w.shape[1]
    _need(conv_w, torch.bfloat16, (ch, K), "conv_w", align=8)
    _need(conv_state, torch.float32, (B, K - 1, ch), "conv_state", align=4)
    _need(norm_w, torch.float32, (dv,), "norm_w")
    _need(state, torch.float32, (B, Hv, dk, dv), "state")
    if conv_heads is not None:
        _need(conv_heads, torch.int32, (B,), "conv_heads", align=4)
    if dt_bias is not None:
        _need(dt_bias, torch.bfloat16, (Hv,), "dt_bias", align=2)
    if A_log is not None:
        _need(A_log, torch.float32, (Hv,), "A_log", align=4)
    if out is None:
        out = torch.empty((B, Hv * dv), dtype=torch.bfloat16, device=state.device)
    _need(out, torch.bfloat16, (B, Hv * dv), "out", align=8)
    if scale is None:
        scale = 1.0 / math.sqrt(dk)
    if arrivals is not None:
        _need(arrivals, torch.int32, (B * Hk,), "arrivals", align=4)
    rc = lib().aila_hip_deltanet_layer_decode(
        _ptr(qkv), qs, _ptr(z), zs, _ptr(a), _ptr(b), ast, _ptr(conv_w), _ptr(conv_state), int(conv_head),
        _ptr(conv_heads), _ptr(dt_bias), _ptr(A_log), _ptr(norm_w), _ptr(state), _ptr(out), B, Hk, Hv, dk, dv,
        K, float(eps), float(scale), _ptr(arrivals), _stream(stream))
    _check(rc, "aila_hip_deltanet_layer_decode")
    return out


def _tok_rows(t, dtype, B, T, width, name, align=2):
    """A [B, T, width] view whose token rows may be strided (column slices of
    fused rows); the rows of all sequences must be equally spaced."""
    if t is None or not t.is_cuda or t.dtype != dtype:
        raise ValueError(f"{name}: expected a {dtype} device tensor")
    if t.shape != (B, T, width) or (width > 1 and t.stride(2) != 1):
        raise ValueError(f"{name}: shape {tuple(t.shape)} / strides {t.stride()}, expected [{B}, {T}, {width}]")
    rs = t.stride(1) if T > 1 else (t.stride(0) if B > 1 else width)
    if B > 1 and t.stride(0) != T * rs:
        raise ValueError(f"{name}: sequences must follow each other (stride(0) = T * stride(1))")
    if t.data_ptr() % align:
        raise ValueError(f"{name} must be {align}-byte aligned")
    return rs


def deltanet_layer_prefill_workspace_size(B: int, T: int, Hk: int, Hv: int, dk: int = 128, dv: int = 128) -> int:
    return int(lib().aila_hip_deltanet_layer_prefill_workspace_size(B, T, Hk, Hv, dk, dv))


def deltanet_layer_prefill(qkv, z, a, b, conv_w, conv_state, conv_head, norm_w, state, num_k_heads,
                           out=None, workspace=None, dt_bias=None, A_log=None, eps: float = 1e-6,
                           scale: float | None = None, stream=None):
    """Full Gated DeltaNet layer over T tokens: qkv [B,T,ch], z [B,T,Hv*dv],
    a/b [B,T,Hv] bf16 (token rows may be strided views of fused rows);
    conv_state [B,3,ch] and state [B,Hv,dk,dv] fp32 updated in place.
    Returns out [B,T,Hv*dv] bf16; the caller advances conv_head by T."""
    import torch
    B, Hv, dk, dv = state.shape
    T = qkv.shape[1]
    Hk = int(num_k_heads)
    ch = 2 * Hk * dk + Hv * dv
    qs = _tok_rows(qkv, torch.bfloat16, B, T, ch, "qkv", align=8)
    zs = _tok_rows(z, torch.bfloat16, B, T, Hv * dv, "z", align=16)
    ast = _tok_rows(a, torch.bfloat16, B, T, Hv, "a")
    bst = _tok_rows(b, torch.bfloat16, B, T, Hv, "b")
    if ast != bst:
        raise ValueError("a and b must share one row stride")
    K = conv_w.shape[1]
    _need(conv_w, torch.bfloat16, (ch, K), "conv_w")
    _need(conv_state, torch.float32, (B, K - 1, ch), "conv_state")
    _need(norm_w, torch.float32, (dv,), "norm_w", align=16)
    _need(state, torch.float32, (B, Hv, dk, dv), "state")
    if dt_bias is not None:
        _need(dt_bias, torch.bfloat16, (Hv,), "dt_bias", align=2)
    if A_log is not None:
        _need(A_log, torch.float32, (Hv,), "A_log", align=4)
    if out is None:
        out = torch.empty((B, T, Hv * dv), dtype=torch.bfloat16, device=state.device)
    _need(out, torch.bfloat16, (B, T, Hv * dv), "out")
    need = deltanet_layer_prefill_workspace_size(B, T, Hk, Hv, dk, dv)
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=state.device)
    if scale is None:
        scale = 1.0 / math.sqrt(dk)
    rc = lib().aila_hip_deltanet_layer_prefill(
        _ptr(qkv), qs, _ptr(z), zs, _ptr(a), _ptr(b), ast, _ptr(conv_w), _ptr(conv_state), int(conv_head),
        _ptr(dt_bias), _ptr(A_log), _ptr(norm_w), _ptr(state), _ptr(out), _ptr(workspace),
        workspace.numel() * workspace.element_size(), B, T, Hk, Hv, dk, dv, K, float(eps), float(scale),
        _stream(stream))
    _check(rc, "aila_hip_deltanet_layer_prefill")
    return out


def deltanet_prefill_workspace_size(B: int, T: int, Hv: int, dk: int, dv: int) -> int:
    return int(lib().aila_hip_deltanet_prefill_workspace_size(B, T, Hv, dk, dv))


def deltanet_prefill(q, k, v, a, b, state, out=None, workspace=None, dt_bias=None,
                     A_log=None, eps: float = 1e-6, scale: float | None = None, stream=None):
    """Chunked prefill over T tokens. q,k [B,T,Hk,dk]; v [B,T,Hv,dv]; a,b
    [B,T,Hv] bf16; state [B,Hv,dk,dv] fp32 (in/out) -> out [B,T,Hv,dv] bf16.
    ``workspace``: uint8 device tensor (allocated here when None)."""
    import torch
    B, T, Hk, dk = q.shape
    Hv, dv = v.shape[2], v.shape[3]
    _need(q, torch.bfloat16, (B, T, Hk, dk), "q")
    _need(k, torch.bfloat16, (B, T, Hk, dk), "k")
    _need(v, torch.bfloat16, (B, T, Hv, dv), "v")
    _need(a, torch.bfloat16, (B, T, Hv), "a", align=2)
    _need(b, torch.bfloat16, (B, T, Hv), "b", align=2)
    _need(state, torch.float32, (B, Hv, dk, dv), "state")
    if dt_bias is not None:
        _need(dt_bias, torch.bfloat16, (Hv,), "dt_bias", align=2)
    if A_log is not None:
        _need(A_log, torch.float32, (Hv,), "A_log", align=4)
    if out is None:
        out = torch.empty((B, T, Hv, dv), dtype=torch.bfloat16, device=q.device)
    _need(out, torch.bfloat16, (B, T, Hv, dv), "out")
    need = deltanet_prefill_workspace_size(B, T, Hv, dk, dv)
    if workspace is None:
        workspace = torch.empty(max(need, 1), dtype=torch.uint8, device=q.device)
    ws_bytes = workspace.numel() * workspace.element_size()
    if scale is None:
        scale = 1.0 / math.sqrt(dk)
    rc = lib().aila_hip_deltanet_prefill(_ptr(q), _ptr(k), _ptr(v), _ptr(a), _ptr(b),
                                         _ptr(dt_bias), _ptr(A_log), _ptr(state), _ptr(out),
                                         _ptr(workspace), ws_bytes, B, T, Hk, Hv, dk, dv,
                                         float(eps), float(scale), _stream(stream))
    _check(rc, "aila_hip_deltanet_prefill")
    return out


# ------------------------------------------ QK-norm, RoPE, output gate ----
def decode_prepare_qkv(q_in, k, v, q_norm_w=None, k_norm_w=None, k_cache=None, v_cache=None,
                       pos: int = 0, positions=None, rotary_dim=None, theta: float = 1e6,
                       eps: float = 1e-6, packed_gate: bool = False, q_out=None, gate_out=None,
                       rope=None, stream=None):
    """Per-head RMSNorm + RoPE of one token per sequence, and the K/V append.

    q_in [B,Hq,D] (or [B,Hq,2D] q|gate when ``packed_gate``); k [B,Hkv,D] is
    updated in place; v [B,Hkv,D]; caches [B,Hkv,max_seq,D] or None. Returns
    q_out (and gate_out when packed). rope: a :func:`rope_pos` record (text
    shift / mRoPE positions); None rotates at the cache row."""
    import torch
    B, Hkv, D = k.shape
    Hq = q_in.shape[1]
    _need(q_in, torch.bfloat16, (B, Hq, 2 * D if packed_gate else D), "q_in")
    _need(k, torch.bfloat16, (B, Hkv, D), "k")
    _need(v, torch.bfloat16, (B, Hkv, D), "v")
    if q_out is None:
        q_out = torch.empty((B, Hq, D), dtype=torch.bfloat16, device=k.device) if packed_gate else q_in
    _need(q_out, torch.bfloat16, (B, Hq, D), "q_out")
    if packed_gate:
        if gate_out is None:
            gate_out = torch.empty((B, Hq, D), dtype=torch.bfloat16, device=k.device)
        _need(gate_out, torch.bfloat16, (B, Hq, D), "gate_out")
    for w, name in ((q_norm_w, "q_norm_w"), (k_norm_w, "k_norm_w")):
        if w is not None:
            _need(w, torch.bfloat16, (D,), name, align=2)
    max_seq = 0
    if k_cache is not None or v_cache is not None:
        max_seq = k_cache.shape[2]
        _need(k_cache, torch.bfloat16, (B, Hkv, max_seq, D), "k_cache")
        _need(v_cache, torch.bfloat16, (B, Hkv, max_seq, D), "v_cache")
    if positions is not None:
        _need(positions, torch.int32, (B,), "positions", align=4)
    rc = lib().aila_hip_decode_prepare_qkv(
        _ptr(q_in), int(bool(packed_gate)), _ptr(q_out), _ptr(gate_out) if packed_gate else None,
        _ptr(k), _ptr(v), _ptr(q_norm_w), _ptr(k_norm_w), _ptr(k_cache), _ptr(v_cache), B, Hq, Hkv, D,
        max_seq, D if rotary_dim is None else int(rotary_dim), float(theta), float(eps), int(pos),
        _ptr(positions), _rope_arg(rope), _stream(stream))
    _check(rc, "decode_prepare_qkv")
    return (q_out, gate_out) if packed_gate else q_out


def gqa_decode_prepare_append(q_in, k_new, v_new, k_cache, v_cache, pos: int, q_norm_w=None, k_norm_w=None,
                              rotary_dim=None, theta: float = 1e6, eps: float = 1e-6, packed_gate: bool = False,
                              out=None, gate_out=None, workspace=None, positions=None, apply_gate: bool = False,
                              rope=None, stream=None):
    """QK-norm + RoPE + K/V append + split-K decode in one launch.
    q_in [B,Hq,D] (or [B,Hq,2D] q|gate when packed_gate); k_new/v_new [B,Hkv,D];
    caches [B,Hkv,max_seq,D]. Returns out (and gate_out when packed).
    apply_gate (packed only): out = attention * sigmoid(gate), the gated
    attention epilogue, instead of returning the gate.
    Without a workspace the decode runs single-pass (one workgroup per KV
    head), as gqa_decode_append."""
    import torch
    if apply_gate and not packed_gate:
        raise ValueError("apply_gate needs packed_gate")
    B, Hkv, max_seq, D = k_cache.shape
    Hq = q_in.shape[1]
    _need(q_in, torch.bfloat16, (B, Hq, 2 * D if packed_gate else D), "q_in")
    _need(k_new, torch.bfloat16, (B, Hkv, D), "k_new")
    _need(v_new, torch.bfloat16, (B, Hkv, D), "v_new")
    _need(k_cache, torch.bfloat16, (B, Hkv, max_seq, D), "k_cache")
    _need(v_cache, torch.bfloat16, (B, Hkv, max_seq, D), "v_cache")
    for w, name in ((q_norm_w, "q_norm_w"), (k_norm_w, "k_norm_w")):
        if w is not None:
            _need(w, torch.bfloat16, (D,), name, align=2)
    if out is None:
        out = torch.empty((B, Hq, D), dtype=torch.bfloat16, device=k_cache.device)
    _need(out, torch.bfloat16, (B, Hq, D), "out")
    if packed_gate and not apply_gate:
        if gate_out is None:
            gate_out = torch.empty((B, Hq, D), dtype=torch.bfloat16, device=k_cache.device)
        _need(gate_out, torch.bfloat16, (B, Hq, D), "gate_out")
    ws_bytes = 0
    if workspace is not None:
        if not workspace.is_cuda or not workspace.is_contiguous():
            raise ValueError("workspace must be a contiguous device tensor")
        ws_bytes = workspace.numel() * workspace.element_size()
    if positions is not None:
        _need(positions, torch.int32, (B,), "positions", align=4)
    rc = lib().aila_hip_gqa_decode_prepare_append(
        _ptr(q_in), 2 if apply_gate else int(bool(packed_gate)), _ptr(gate_out) if packed_gate and not apply_gate else None,
        _ptr(k_new), _ptr(v_new),
        _ptr(q_norm_w), _ptr(k_norm_w), _ptr(k_cache), _ptr(v_cache), _ptr(out), _ptr(workspace),
        ws_bytes, B, Hq, Hkv, D, max_seq,
        D if rotary_dim is None else int(rotary_dim), float(theta), float(eps), int(pos), _ptr(positions),
        _rope_arg(rope), _stream(stream))
    _check(rc, "gqa_decode_prepare_append")
    return (out, gate_out) if packed_gate and not apply_gate else out


def head_rms_norm(x, weight=None, eps: float = 1e-6, stream=None):
    """In-place per-head RMSNorm of x [S, H, D] bf16 (weight [D] bf16 or None)."""
    import torch
    S, H, D = x.shape
    _need(x, torch.bfloat16, (S, H, D), "x")
    if weight is not None:
        _need(weight, torch.bfloat16, (D,), "weight", align=2)
    _check(lib().aila_hip_head_rms_norm(_ptr(x), _ptr(weight), S, H, D, float(eps), _stream(stream)),
           "head_rms_norm")
    return x


def apply_rope(q, k, start_pos: int = 0, rotary_dim=None, theta: float = 1e6, rope=None, stream=None):
    """In-place RoPE of q [S,Hq,D] and k [S,Hkv,D] bf16 for the tokens of cache
    rows start_pos + s (at those rows, or at the positions of ``rope``)."""
    import torch
    S, Hq, D = q.shape
    Hkv = k.shape[1]
    _need(q, torch.bfloat16, (S, Hq, D), "q")
    _need(k, torch.bfloat16, (S, Hkv, D), "k")
    _check(lib().aila_hip_apply_rope(_ptr(q), _ptr(k), S, int(start_pos), Hq, Hkv, D,
                                     D if rotary_dim is None else int(rotary_dim), float(theta),
                                     _rope_arg(rope), _stream(stream)), "apply_rope")
    return q, k


def sigmoid_mul(inp, gate, out=None, stream=None):
    """out = inp * sigmoid(gate), bf16 tensors of equal shape (out may be inp)."""
    import torch
    if out is None:
        out = torch.empty_like(inp)
    for t, name in ((inp, "input"), (gate, "gate"), (out, "output")):
        _need(t, torch.bfloat16, tuple(inp.shape), name)
    _check(lib().aila_hip_sigmoid_mul(_ptr(inp), _ptr(gate), _ptr(out), inp.numel(), _stream(stream)),
           "sigmoid_mul")
    return out
