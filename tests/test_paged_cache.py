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
                          UNSUPPORTED_HEAD_DIM)

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
    declared = {m.replace("##SFX", s) for m in re.findall(r"int (cuflash_\w+##SFX)\(", text)
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
    # Order: null, dimension, head_dim, relations.
    assert call(k=None, d=48, tokens=0) == NULL_POINTER
    assert call(tokens=0, d=48) == INVALID_DIMENSION
    assert call(d=48, kv_heads=3) == UNSUPPORTED_HEAD_DIM


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
    refused("multiple of 16 bytes", k=_Fake(torch.zeros(4 * 2 * 64 + 1)[1:].view(4, 2, 64)))
    refused("needs q", out=f(4, 2, 64))
    with pytest.raises(cuflash_attn.CuFlashError):
        append(**dict(good, k_cache=f(3, 16, 2, 64, dtype=torch.float64)), lib=object())
