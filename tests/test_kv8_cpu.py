"""Argument checks of the 8-bit KV cache and scoring entry points (no GPU: every
refusal happens on the host, before anything is enqueued)."""
from __future__ import annotations

import ctypes

import pytest


@pytest.fixture(scope="module")
def lib():
    from polar_pack_b200 import _lib
    return _lib


def _cache(lib, **kw):
    p = ctypes.c_void_p * 2
    d = dict(codes=p(256, 512), scales=p(256, 512), tail=p(256, 512), batch=2, kv_heads=2, capacity=128, head_dim=128)
    d.update(kw)
    return ctypes.byref(lib.Kv8CacheDesc(**d))


S3 = (ctypes.c_int64 * 3)(1024, 256, 128)
S2 = (ctypes.c_int64 * 2)(256, 128)


@pytest.mark.parametrize("bad", [dict(batch=0), dict(batch=4097), dict(kv_heads=0), dict(capacity=100),
                                 dict(capacity=0), dict(head_dim=96), dict(codes=(ctypes.c_void_p * 2)(0, 256)),
                                 dict(tail=(ctypes.c_void_p * 2)(264, 256)),
                                 dict(scales=(ctypes.c_void_p * 2)(256, 0))])
def test_descriptor(lib, bad):
    L, c = lib.load(), _cache(lib, **bad)
    rcs = [L.pp_kv8_append(c, 256, S3, 256, S3, 1, 256, None, None, None, None, 0, None, None),
           L.pp_kv8_restore(c, 256, None, 1, 256, 256, None, None),
           L.pp_kv8_attention(c, 256, S3, 1, 4, 256, None, 1.0, 256, S3, None, None, None, 0, 256, 1 << 30, None, None),
           L.pp_kv8_decode(c, 256, S2, 4, 256, S2, 256, S2, 256, 1.0, None, 256, S2, None, None, None, 0, 256, 1 << 30,
                           None, None),
           L.pp_kv8_evict(c, _cache(lib), 256, 256, 512, 256, 256, 64, 0, 0, None, None),
           L.pp_kv8_attention_workspace_bytes(c, 1, 4, 0, ctypes.byref(ctypes.c_size_t()))]
    assert rcs == [lib.PP_ERR_INVALID] * 6


def test_arguments(lib):
    L, c = lib.load(), _cache(lib)
    odd = (ctypes.c_int64 * 3)(1024, 256, 100)
    bad = [L.pp_kv8_append(c, None, S3, 256, S3, 1, 256, None, None, None, None, 0, None, None),
           L.pp_kv8_append(c, 256, S3, 264, S3, 1, 256, None, None, None, None, 0, None, None),
           L.pp_kv8_append(c, 256, odd, 256, S3, 1, 256, None, None, None, None, 0, None, None),
           L.pp_kv8_append(c, 256, S3, 256, S3, -1, 256, None, None, None, None, 0, None, None),
           L.pp_kv8_append(c, 256, S3, 256, S3, 1, 256, None, 256, None, 256, 10, None, None),    # half a rotation
           L.pp_kv8_restore(c, None, None, 1, 256, 256, None, None),
           L.pp_kv8_restore(c, 256, None, 1, 256, 8, None, None),
           L.pp_kv8_attention(c, 256, S3, 1, 5, 256, None, 1.0, 256, S3, None, None, None, 0, 256, 1 << 30, None, None),
           L.pp_kv8_attention(c, 256, S3, 1, 40, 256, None, 1.0, 256, S3, None, None, None, 0, 256, 1 << 30, None, None),
           L.pp_kv8_attention(c, 256, S3, 70000, 4, 256, None, 1.0, 256, S3, None, None, None, 0, 256, 1 << 30, None,
                              None),
           L.pp_kv8_attention(c, 256, odd, 1, 4, 256, None, 1.0, 256, S3, None, None, None, 0, 256, 1 << 30, None, None),
           L.pp_kv8_evict(c, c, 256, 256, 512, 256, 256, 64, 0, 0, None, None),
           L.pp_kv8_evict(c, _cache(lib, kv_heads=1), 256, 256, 512, 256, 256, 64, 0, 0, None, None)]
    assert bad == [lib.PP_ERR_INVALID] * len(bad)
    assert L.pp_kv8_append(c, 256, S3, 256, S3, 0, 256, None, None, None, None, 0, None, None) == 0
    for args in ((9, 100, 1, 0), (0, 0, 1, 0), (0, 100, 1, 33), (0, 5, 1, 6), (2, 100, 1, -1), (2, 100, -1, 0)):
        dtype, vocab, rows, top = args
        assert L.pp_token_logprobs(256, dtype, 100, rows, vocab, 256, top, 256, 256, 256, 256, None,
                                   None) == lib.PP_ERR_INVALID
    assert L.pp_token_logprobs(257, 0, 100, 1, 100, 256, 0, 256, 256, 256, 256, None, None) == lib.PP_ERR_INVALID
    assert L.pp_token_logprobs(256, 0, 100, 0, 100, 256, 0, 256, 256, 256, 256, None, None) == 0


def test_capture_waits_for_the_current_stream(monkeypatch):
    """The step that a capture warms up with runs behind the work that the
    current stream holds: it shares the decoder's buffers and position."""
    import contextlib

    import torch
    from polar_pack_b200.decoder import QuadDecoder
    log = []

    class Stream:
        cuda_stream = 0

        def wait_stream(self, other):
            log.append(("wait", other))

        def synchronize(self):
            log.append("synchronize")

    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: "current")
    monkeypatch.setattr(torch.cuda, "stream", lambda s: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "graph", lambda g, stream=None, **kw: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "CUDAGraph", object)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: None)
    dec = QuadDecoder.__new__(QuadDecoder)
    dec.kv8, dec.device, dec.pos = None, torch.device("cpu"), torch.zeros(1, dtype=torch.int32)
    dec._run = lambda s: log.append("run")
    dec.capture(Stream())
    assert log[:3] == [("wait", "current"), "run", "synchronize"] and int(dec.pos) == 0


def test_coherent_loads():
    """With launch overlap a kernel runs while the one before it writes its
    inputs: none of these operators reads through the read-only path, which
    need not see such writes."""
    import re
    from pathlib import Path

    import polar_pack_b200
    src = Path(polar_pack_b200.__file__).parent / "csrc"
    for f in (*src.glob("kv8*"), src / "token_logprobs.cu"):
        assert not re.search(r"\bldg_\w+\(|__ldg\(|\.nc\b", f.read_text()), f.name


def test_evict_refuses_what_overlaps(lib):
    """Arrays that are written may share no byte with another one."""
    L, M = lib.load(), 1 << 20
    pair = lambda a, step: (ctypes.c_void_p * 2)(a, a + step)
    old = dict(codes=pair(M, M), scales=pair(3 * M, M), tail=pair(5 * M, M), batch=1, kv_heads=1, capacity=256)
    into = dict(codes=pair(11 * M, M), scales=pair(13 * M, M), tail=pair(15 * M, M), batch=1, kv_heads=1, capacity=256)
    args = dict(lens=20 * M, weights=21 * M, into_weights=22 * M, new_lens=23 * M, kept=24 * M)

    def call(new=into, **kw):
        a = {**args, **kw}
        return L.pp_kv8_evict(_cache(lib, **old), _cache(lib, **new), a["lens"], a["weights"], a["into_weights"],
                              a["new_lens"], a["kept"], 64, 0, 0, None, None)

    codes, tail, wts = 256 * 128, 64 * 128 * 2, 256 * 4
    for at in (M + codes - 16, 2 * M + 64, 12 * M - codes + 16):            # old keys, old values, the new values
        assert call({**into, "codes": (ctypes.c_void_p * 2)(at, 12 * M)}) == lib.PP_ERR_INVALID
    assert call({**into, "tail": (ctypes.c_void_p * 2)(5 * M + tail - 16, 16 * M)}) == lib.PP_ERR_INVALID
    assert call({**into, "scales": (ctypes.c_void_p * 2)(3 * M + 12, 14 * M)}) == lib.PP_ERR_INVALID
    assert call(into_weights=21 * M + wts - 4) == lib.PP_ERR_INVALID
    assert call(into_weights=21 * M - wts + 4) == lib.PP_ERR_INVALID
    assert call(new_lens=20 * M) == lib.PP_ERR_INVALID
    assert call(kept=20 * M - 63 * 4) == lib.PP_ERR_INVALID
    assert call(kept=22 * M + 4) == lib.PP_ERR_INVALID
