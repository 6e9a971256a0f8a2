"""What the paged-cache operators refuse (include/cuflash/paged_cache.h), without a GPU: every call
here ends in the checks before the first HIP call, or in those of the tensor helpers."""

from __future__ import annotations

import ctypes
import os
import re
import subprocess

import pytest

import cuflash_attn
from conftest import REPO
from cuflash_attn import (DIMENSION_MISMATCH, INVALID_DIMENSION, NULL_POINTER,
                          OUT_OF_MEMORY, UNSUPPORTED_HEAD_DIM)

HEADER = os.path.join(REPO, "include", "cuflash", "paged_cache.h")

# Host memory stands in for device pointers: validation never reads it. 16-byte aligned.
_RAW = (ctypes.c_char * 80)()
P = (ctypes.addressof(_RAW) + 15) // 16 * 16

APPEND = dict(q=P, k=P, v=P, q_out=P, k_cache=P, v_cache=P, table=P, lens=P, starts=P, cos=P,
              sin=P, tokens=8, batch=2, heads=8, kv_heads=2, q_stride=512, k_stride=128,
              v_stride=128, pages=4, page=16, max_pages=3, d=64, rotary=32, positions=48,
              interleaved=False, stream=None)


def _call(lib, kind, sfx, ok, **kw):
    assert not set(kw) - set(ok), kw
    return lib.fn(kind, sfx)(*dict(ok, **kw).values())


def test_every_declared_symbol_is_bound_and_exported(lib):
    text = open(HEADER).read()
    declared = {m.replace("##SFX", s) for m in re.findall(r"(cuflash_\w+##SFX)\(", text)
                for s in ("f32", "f16", "bf16")}
    assert declared == set(cuflash_attn.PAGED_CACHE_SYMBOLS)
    out = subprocess.run(["nm", "-D", "--defined-only", lib.path], capture_output=True, text=True,
                         check=True).stdout
    exported = {line.split()[-1] for line in out.splitlines() if line.strip()}
    assert declared <= exported


@pytest.mark.parametrize("sfx", ["f32", "f16", "bf16"])
def test_append_refusals(lib, sfx):
    def call(**kw):
        return _call(lib, "append_paged", sfx, APPEND, **kw)

    for name in ("k", "v", "k_cache", "v_cache", "table", "lens"):
        assert call(**{name: None}) == NULL_POINTER, name
    for name in ("q", "q_out", "cos", "sin"):  # in pairs
        assert call(**{name: None}) == NULL_POINTER, name
    for name in ("tokens", "batch", "heads", "kv_heads", "pages", "page", "max_pages", "d",
                 "rotary", "positions"):
        for bad in (0, -1):
            assert call(**{name: bad}) == INVALID_DIMENSION, name
    for d in (16, 48, 96, 256):
        assert call(d=d) == UNSUPPORTED_HEAD_DIM
    assert call(rotary=24) == INVALID_DIMENSION  # not a multiple of 16
    assert call(rotary=80) == DIMENSION_MISMATCH  # more than head_dim
    assert call(cos=None, sin=None) == INVALID_DIMENSION  # rotary_dim without tables
    assert call(kv_heads=3) == DIMENSION_MISMATCH
    assert call(starts=None) == DIMENSION_MISMATCH  # one token per sequence, 8 for 2
    for name in ("q_stride", "k_stride", "v_stride"):
        assert call(**{name: APPEND[name] - 64}) == DIMENSION_MISMATCH, name
        assert call(**{name: APPEND[name] + 1}) == INVALID_DIMENSION, name
    assert call(page=1 << 16, max_pages=1 << 16) == INVALID_DIMENSION
    big = 1 << 25
    assert call(heads=big, kv_heads=big, q_stride=1 << 30, k_stride=1 << 30,
                v_stride=1 << 30) == DIMENSION_MISMATCH  # rows longer than any stride
    for name in ("q", "k", "v", "q_out", "k_cache", "v_cache", "cos", "sin"):
        assert call(**{name: P + 8}) == INVALID_DIMENSION, name
    assert call(q_stride=768) == DIMENSION_MISMATCH  # rotated in place, but not packed
    assert call(page=1 << 10, max_pages=1 << 21) == INVALID_DIMENSION
    assert call(tokens=1 << 26, batch=1, heads=64, kv_heads=64, d=128, q_stride=1 << 13,
                k_stride=1 << 13, v_stride=1 << 13) == INVALID_DIMENSION  # 2^32 threads and more
    # Order: null, dimension, head_dim, relations.
    assert call(k=None, d=48, tokens=0) == NULL_POINTER
    assert call(tokens=0, d=48) == INVALID_DIMENSION
    assert call(d=48, kv_heads=3) == UNSUPPORTED_HEAD_DIM

FORWARD = dict(q=P, k_cache=P, v_cache=P, o=P, l=P, table=P, lens=P, starts=P, tokens=8, batch=2,
               heads=8, kv_heads=2, page=16, max_pages=3, d=64, scale=0.125, causal=True,
               ws=None, ws_bytes=0, stream=None)
SHARED = dict(q=P, k_cache=P, v_cache=P, o=P, l=P, prefix_table=P, table=P, lens=P, batch=2,
              heads=8, kv_heads=2, prefix=20, page=16, max_pages=3, d=64, scale=0.125,
              ws=None, ws_bytes=0, stream=None)


@pytest.mark.parametrize("sfx", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kind,ok", [("forward_paged", FORWARD), ("decode_shared", SHARED)])
def test_attention_refusals(lib, sfx, kind, ok):
    def call(**kw):
        return _call(lib, kind, sfx, ok, **kw)

    for name in (n for n in ok if ok[n] == P):
        assert call(**{name: None}) == NULL_POINTER, name
    for name in ("tokens", "batch", "heads", "kv_heads", "page", "max_pages", "d"):
        for bad in (0, -1):
            if name in ok:
                assert call(**{name: bad}) == INVALID_DIMENSION, name
    for d in (16, 48, 96, 256):
        assert call(d=d) == UNSUPPORTED_HEAD_DIM
    for scale in (float("nan"), float("inf"), -1.0):
        assert call(scale=scale) == INVALID_DIMENSION
    assert call(kv_heads=3) == DIMENSION_MISMATCH
    assert call(page=1 << 16, max_pages=1 << 16) == INVALID_DIMENSION
    many = {"tokens": 1 << 28} if "tokens" in ok else {"batch": 1 << 28}
    assert call(**many) == INVALID_DIMENSION  # tokens times heads beyond 32 bits
    for name in ("q", "k_cache", "v_cache", "o"):
        assert call(**{name: P + 8}) == INVALID_DIMENSION, name
    assert call(ws=(P + 255) // 256 * 256 + 16, ws_bytes=1 << 30) == INVALID_DIMENSION
    assert call(ws=(P + 255) // 256 * 256, ws_bytes=16) == OUT_OF_MEMORY
    if kind == "decode_shared":
        assert call(prefix=-1) == INVALID_DIMENSION
        assert call(prefix=49) == DIMENSION_MISMATCH  # past the block table
    assert call(q=None, d=48) == NULL_POINTER
    assert call(heads=0, d=48) == INVALID_DIMENSION
    assert call(d=48, scale=-1.0) == UNSUPPORTED_HEAD_DIM
    assert call(scale=-1.0, kv_heads=3) == INVALID_DIMENSION


@pytest.mark.parametrize("sfx", ["f32", "f16", "bf16"])
def test_grids_beyond_32_bits_are_refused(lib, sfx):
    """One token each of many sequences, one key/value head for every query head: valid sizes whose
    workgroups are too many."""
    n = 1 << 22
    assert _call(lib, "forward_paged", sfx, FORWARD, tokens=n, batch=n, heads=500, kv_heads=500,
                 d=32) == INVALID_DIMENSION
    assert _call(lib, "decode_shared", sfx, SHARED, batch=1 << 24) == INVALID_DIMENSION  # the merge
    assert lib.fn("decode_shared_workspace", sfx)(1 << 24, 8, 2, 64) == -1
    for kind, ok in (("forward_paged", FORWARD), ("decode_shared", SHARED)):
        assert _call(lib, kind, sfx, ok, heads=65536) == INVALID_DIMENSION
        assert _call(lib, kind, sfx, ok, page=1 << 10, max_pages=1 << 21) == INVALID_DIMENSION
    assert lib.fn("forward_paged_workspace", sfx)(4, 2, 65536, 2, 64) == -1


@pytest.mark.parametrize("sfx", ["f32", "f16", "bf16"])
def test_workspace_sizes(lib, sfx):
    forward, shared = (lib.fn(f"{kind}_workspace", sfx) for kind in ("forward_paged",
                                                                     "decode_shared"))
    assert forward(4, 2, 8, 2, 64) > 0 and shared(4, 8, 2, 64) > 0
    assert forward(1 << 20, 2, 8, 2, 64) == 0  # enough rows without chunks
    for bad in ((0, 2, 8, 2, 64), (4, -1, 8, 2, 64), (4, 2, 8, 3, 64), (4, 2, 8, 2, 48),
                (1 << 28, 2, 8, 2, 64)):
        assert forward(*bad) == -1
    for bad in ((0, 8, 2, 64), (4, 8, 3, 64), (4, 8, 2, 256)):
        assert shared(*bad) == -1


class _Fake:
    """A tensor's outside on a made-up device, for the helpers' own checks."""

    def __init__(self, t, index=0):
        self._t, self.is_cuda = t, True
        self.device = type("Device", (), {"index": index})()

    def __getattr__(self, name):
        return getattr(self._t, name)


def _fakes(torch, index=0):
    z = lambda *s, **k: _Fake(torch.zeros(s, **k), index)  # noqa: E731
    return dict(k=z(4, 2, 64), v=z(4, 2, 64), k_cache=z(3, 16, 2, 64), v_cache=z(3, 16, 2, 64),
                block_table=z(2, 3, dtype=torch.int32), seq_lens=z(2, dtype=torch.int32),
                query_starts=z(3, dtype=torch.int32))


def test_append_helper_refusals(monkeypatch):
    import torch

    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    append = cuflash_attn.flash_attention_append_paged
    good = _fakes(torch)

    def refused(match, error=ValueError, **kw):
        with pytest.raises(error, match=match):
            append(**dict(good, **kw), lib=object())

    f = lambda *s, **k: _Fake(torch.zeros(s, **k))  # noqa: E731
    with pytest.raises(ValueError, match="on the GPU"):
        append(**dict(good, k=torch.zeros(4, 2, 64)), lib=object())
    with pytest.raises(ValueError, match="current device"):
        append(**_fakes(torch, index=1), lib=object())
    refused("one dtype", v=f(4, 2, 64, dtype=torch.float16))
    refused("int32", TypeError, seq_lens=f(2, dtype=torch.int64))
    refused("contiguous", k_cache=_Fake(torch.zeros(3, 16, 64, 2).transpose(2, 3)))
    refused("k_cache, v_cache", v_cache=f(4, 16, 2, 64))
    refused("block_table", seq_lens=f(3, dtype=torch.int32))
    refused("query_starts", query_starts=f(2, dtype=torch.int32))
    refused(r"k, v \[T,Hkv,D\]", k=f(4, 1, 64))
    refused(r"k, v \[T,Hkv,D\]", q=f(5, 4, 64))
    refused("come together", cos=f(9, 16))
    refused("cos, sin", cos=f(9, 16), sin=f(9, 8))
    refused("float32", cos=f(9, 16, dtype=torch.float16), sin=f(9, 16, dtype=torch.float16))
    refused("heads of a token", k=_Fake(torch.zeros(4, 64, 2).transpose(1, 2)))
    refused("tokens of v", v=_Fake(torch.zeros(1, 2, 64).expand(4, 2, 64)))
    refused("tokens of k", k=_Fake(torch.empty((4, 2, 64), device="meta").as_strided(
        (4, 2, 64), (1 << 31, 64, 1))))
    refused("multiple of 16 bytes", k=_Fake(torch.zeros(4 * 2 * 64 + 1)[1:].view(4, 2, 64)))
    refused("needs q", out=f(4, 2, 64))
    with pytest.raises(cuflash_attn.CuFlashError):
        append(**dict(good, k_cache=f(3, 16, 2, 64, dtype=torch.float64)), lib=object())


def test_attention_helper_refusals(monkeypatch):
    import torch

    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    f = lambda *s, **k: _Fake(torch.zeros(s, **k))  # noqa: E731
    i = dict(dtype=torch.int32)
    good = _fakes(torch)
    del good["k"], good["v"]
    forward = dict(good, q=f(4, 4, 64))
    shared = dict(good, q=f(2, 4, 1, 64), prefix_table=f(2, **i), prefix_len=20)
    del shared["query_starts"]

    def refused(fn, args, match, error=ValueError, **kw):
        with pytest.raises(error, match=match):
            fn(**dict(args, **kw), lib=object())

    fwd, dec = cuflash_attn.flash_attention_forward_paged, cuflash_attn.flash_attention_decode_shared
    refused(fwd, forward, r"q \[T,H,D\]", q=f(4, 4, 32))
    refused(fwd, forward, r"q \[T,H,D\]", q=_Fake(torch.zeros(4, 64, 4).transpose(1, 2)))
    refused(fwd, forward, "one dtype", q=f(4, 4, 64, dtype=torch.float16))
    refused(fwd, forward, "query_starts", query_starts=f(4, **i))
    refused(fwd, forward, "16 bytes", q=_Fake(torch.zeros(4 * 4 * 64 + 1)[1:].view(4, 4, 64)))
    refused(dec, shared, r"q \[B,H,1,D\]", q=f(3, 4, 1, 64))
    refused(dec, shared, r"q \[B,H,1,D\]", q=f(2, 4, 2, 64))
    refused(dec, shared, "int32", TypeError, prefix_table=f(2))
    for fn, args in ((fwd, forward), (dec, shared)):
        with pytest.raises(ValueError, match="on the GPU"):
            fn(**dict(args, q=torch.zeros(4, 4, 64)), lib=object())


def test_cut_into_workgroups_stays_in_bounds(tmp_path):
    """The host run of the kernels' plan (tests/cpp/test_paged_plan.cpp)."""
    from test_host_rules import run_program

    run_program("test_paged_plan", tmp_path, 6000, 1)
