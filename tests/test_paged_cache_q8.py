"""What the operators on an 8-bit paged cache refuse (include/cuflash/paged_cache_q8.h), without a GPU: every
call here ends in the checks before the first HIP call, or in those of the tensor helpers. And their cut
into waves on the host."""

from __future__ import annotations

import os
import re
import subprocess

import pytest

import cuflash_attn
from conftest import REPO
from cuflash_attn import (DIMENSION_MISMATCH, INVALID_DIMENSION, NULL_POINTER, OUT_OF_MEMORY,
                          UNSUPPORTED_DTYPE, UNSUPPORTED_HEAD_DIM)
from test_host_rules import run_program
from test_paged_cache import APPEND as APPEND_16
from test_paged_cache import P, _call, _Fake

HEADER = os.path.join(REPO, "include", "cuflash", "paged_cache_q8.h")
SFX = ["f32", "f16", "bf16"]


def _with(args, at, **more):
    """`args` with `more` behind its key `at`: the arguments in the order of the C ABI."""
    out = {}
    for k, v in args.items():
        out[k] = v
        if k == at:
            out.update(more)
    return out


APPEND = _with(_with(APPEND_16, "v_cache", k_exp=P, v_exp=P), "interleaved", code=1)
READ = dict(k_cache=P, v_cache=P, k_exp=P, v_exp=P, k_out=P, v_out=P, table=P, lens=P, starts=P,
            tokens=8, batch=2, kv_heads=2, pages=4, page=16, max_pages=3, d=64, code=0, stream=None)
FORWARD = dict(q=P, k_cache=P, v_cache=P, k_exp=P, v_exp=P, o=P, l=P, table=P, lens=P, starts=P,
               tokens=8, batch=2, heads=8, kv_heads=2, page=16, max_pages=3, d=64, scale=0.125,
               causal=True, code=1, ws=None, ws_bytes=0, stream=None)
DECODE = {k: v for k, v in FORWARD.items() if k not in ("starts", "tokens", "causal")}


def test_every_declared_symbol_is_bound_and_exported(lib):
    text = open(HEADER).read()
    declared = {m.replace("##SFX", s) for m in re.findall(r"(cuflash_\w+##SFX)\(", text)
                for s in SFX}
    assert declared == set(cuflash_attn.PAGED_CACHE_Q8_SYMBOLS)
    out = subprocess.run(["nm", "-D", "--defined-only", lib.path], capture_output=True, text=True,
                         check=True).stdout
    assert declared <= {line.split()[-1] for line in out.splitlines() if line.strip()}


@pytest.mark.parametrize("sfx", SFX)
def test_append_refusals(lib, sfx):
    def call(**kw):
        return _call(lib, "append_paged_q8", sfx, APPEND, **kw)

    for name in ("k", "v", "k_cache", "v_cache", "k_exp", "v_exp", "table", "lens", "q", "q_out",
                 "cos", "sin"):
        assert call(**{name: None}) == NULL_POINTER, name
    for code in (-1, 2, 7):
        assert call(code=code) == UNSUPPORTED_DTYPE
    for name in ("tokens", "batch", "heads", "kv_heads", "pages", "page", "max_pages", "d",
                 "rotary", "positions"):
        for bad in (0, -1):
            assert call(**{name: bad}) == INVALID_DIMENSION, name
    for d in (16, 48, 96, 256):
        assert call(d=d) == UNSUPPORTED_HEAD_DIM
    assert call(rotary=24) == INVALID_DIMENSION
    assert call(rotary=80) == DIMENSION_MISMATCH
    assert call(cos=None, sin=None) == INVALID_DIMENSION
    assert call(kv_heads=3) == DIMENSION_MISMATCH
    assert call(starts=None) == DIMENSION_MISMATCH
    for name in ("q_stride", "k_stride", "v_stride"):
        assert call(**{name: APPEND[name] - 64}) == DIMENSION_MISMATCH, name
        assert call(**{name: APPEND[name] + 1}) == INVALID_DIMENSION, name
    for name in ("q", "k", "v", "q_out", "k_cache", "v_cache", "k_exp", "v_exp", "cos", "sin"):
        assert call(**{name: P + 8}) == INVALID_DIMENSION, name
    assert call(q_stride=768) == DIMENSION_MISMATCH
    assert call(page=1 << 10, max_pages=1 << 21) == INVALID_DIMENSION
    assert call(tokens=1 << 26, batch=1, heads=64, kv_heads=64, d=128, q_stride=1 << 13,
                k_stride=1 << 13, v_stride=1 << 13) == INVALID_DIMENSION  # 2^32 threads and more
    # Order: null, code, dimension, head_dim, relations.
    assert call(v_exp=None, code=3) == NULL_POINTER
    assert call(code=3, tokens=0) == UNSUPPORTED_DTYPE
    assert call(tokens=0, d=48) == INVALID_DIMENSION
    assert call(d=48, kv_heads=3) == UNSUPPORTED_HEAD_DIM


@pytest.mark.parametrize("sfx", SFX)
def test_read_refusals(lib, sfx):
    def call(**kw):
        return _call(lib, "read_paged_q8", sfx, READ, **kw)

    for name in (n for n in READ if READ[n] == P):
        assert call(**{name: None}) == NULL_POINTER, name
    for code in (-1, 2):
        assert call(code=code) == UNSUPPORTED_DTYPE
    for name in ("tokens", "batch", "kv_heads", "pages", "page", "max_pages", "d"):
        for bad in (0, -1):
            assert call(**{name: bad}) == INVALID_DIMENSION, name
    assert call(d=256) == UNSUPPORTED_HEAD_DIM
    for name in ("k_cache", "v_cache", "k_exp", "v_exp", "k_out", "v_out"):
        assert call(**{name: P + 8}) == INVALID_DIMENSION, name
    assert call(page=1 << 10, max_pages=1 << 21) == INVALID_DIMENSION
    assert call(kv_heads=1 << 25) == INVALID_DIMENSION  # a token's rows beyond 32 bits
    assert call(tokens=1 << 26, kv_heads=64) == INVALID_DIMENSION  # 2^32 threads and more
    assert call(k_out=None, code=3) == NULL_POINTER
    assert call(code=3, page=0) == UNSUPPORTED_DTYPE


@pytest.mark.parametrize("sfx", SFX)
@pytest.mark.parametrize("kind,ok", [("forward_paged_q8", FORWARD), ("decode_paged_q8", DECODE)])
def test_attention_refusals(lib, sfx, kind, ok):
    def call(**kw):
        return _call(lib, kind, sfx, ok, **kw)

    for name in (n for n in ok if ok[n] == P):
        assert call(**{name: None}) == NULL_POINTER, name
    for code in (-1, 2):
        assert call(code=code) == UNSUPPORTED_DTYPE
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
    assert call(page=1 << 24) == INVALID_DIMENSION  # a page of 2^31 bytes
    many = {"tokens": 1 << 28} if "tokens" in ok else {"batch": 1 << 28}
    assert call(**many) == INVALID_DIMENSION  # tokens times heads beyond 32 bits
    assert call(heads=65536) == INVALID_DIMENSION
    for name in ("q", "k_cache", "v_cache", "k_exp", "v_exp", "o"):
        assert call(**{name: P + 8}) == INVALID_DIMENSION, name
    assert call(ws=(P + 255) // 256 * 256 + 16, ws_bytes=1 << 30) == INVALID_DIMENSION
    # (A decode from a short table has no workspace.)
    assert call(ws=(P + 255) // 256 * 256, ws_bytes=16, max_pages=100) == OUT_OF_MEMORY
    assert call(k_exp=None, code=9, d=48) == NULL_POINTER
    assert call(code=9, heads=0) == UNSUPPORTED_DTYPE
    assert call(heads=0, d=48) == INVALID_DIMENSION
    assert call(d=48, scale=-1.0) == UNSUPPORTED_HEAD_DIM
    assert call(scale=-1.0, kv_heads=3) == INVALID_DIMENSION


@pytest.mark.parametrize("sfx", SFX)
def test_workspace_sizes(lib, sfx):
    forward, decode = (lib.fn(f"{kind}_paged_q8_workspace", sfx) for kind in ("forward", "decode"))
    assert forward(4, 2, 8, 2, 64) > 0 and decode(4, 8, 2, 64) > 0
    for bad in ((0, 2, 8, 2, 64), (4, -1, 8, 2, 64), (4, 2, 8, 3, 64), (4, 2, 8, 2, 48),
                (1 << 28, 2, 8, 2, 64), (4, 2, 65536, 2, 64)):
        assert forward(*bad) == -1
    for bad in ((0, 8, 2, 64), (4, 8, 3, 64), (4, 8, 2, 256), (1 << 28, 8, 2, 64)):
        assert decode(*bad) == -1


def test_helper_refusals(monkeypatch):
    import torch

    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)

    def z(*s, index=0, **k):
        t = _Fake(torch.zeros(s, **k), index)
        t.get_device = lambda: index
        return t

    i32, u8, i8 = (dict(dtype=d) for d in (torch.int32, torch.uint8, torch.int8))
    cache = dict(k_cache=z(3, 16, 2, 64, **i8), v_cache=z(3, 16, 2, 64, **i8),
                 k_exp=z(3, 2, 16, **u8), v_exp=z(3, 2, 16, **u8), block_table=z(2, 3, **i32),
                 seq_lens=z(2, **i32))
    starts = z(3, **i32)
    calls = {
        cuflash_attn.flash_attention_append_paged_q8:
            dict(cache, k=z(4, 2, 64), v=z(4, 2, 64), query_starts=starts),
        cuflash_attn.flash_attention_read_paged_q8: dict(cache, key_starts=starts, num_tokens=4),
        cuflash_attn.flash_attention_decode_paged_q8: dict(cache, q=z(2, 4, 1, 64)),
        cuflash_attn.flash_attention_forward_paged_q8:
            dict(cache, q=z(4, 4, 64), query_starts=starts)}
    for fn, good in calls.items():
        def refused(match, error=ValueError, **kw):
            with pytest.raises(error, match=match):
                fn(**dict(good, **kw), lib=object())

        refused("int8 or float8", TypeError, k_cache=z(3, 16, 2, 64))
        refused("int8 or float8", TypeError, v_cache=z(3, 16, 2, 64, dtype=torch.float8_e4m3fn))
        refused("uint8", TypeError, k_exp=z(3, 2, 16, **i8))
        refused("current device", k_cache=z(3, 16, 2, 64, index=1, **i8))
        refused("int32", TypeError, seq_lens=z(2, dtype=torch.int64))
        refused("contiguous", v_cache=_strided(torch, i8))
        refused("k_exp, v_exp", k_exp=z(3, 16, 2, **u8))
        refused("k_cache, v_cache", v_cache=z(4, 16, 2, 64, **i8))
        refused("block_table", seq_lens=z(3, **i32))
        name = next((n for n in ("query_starts", "key_starts") if n in good), None)
        if name:
            refused(r"starts \[B\+1\]", **{name: z(2, **i32)})
    append, read, decode, forward = calls
    for match, kw in ((r"k, v \[T,Hkv,D\]", dict(k=z(4, 1, 64))),
                      (r"q \[T,H,D\]", dict(q=z(5, 4, 64))),
                      ("one dtype", dict(v=z(4, 2, 64, dtype=torch.float16))),
                      ("come together", dict(cos=z(9, 16))), ("needs q", dict(out=z(4, 2, 64)))):
        with pytest.raises(ValueError, match=match):
            append(**dict(calls[append], **kw), lib=object())
    for fn, q in ((decode, z(3, 4, 1, 64)), (decode, z(2, 4, 2, 64)), (forward, z(4, 4, 32))):
        with pytest.raises(ValueError, match="contiguous q"):
            fn(**dict(calls[fn], q=q), lib=object())
    with pytest.raises(cuflash_attn.CuFlashError):
        forward(**dict(calls[forward], q=z(4, 4, 64, dtype=torch.float64)), lib=object())
    for fn, name in ((read, "key_starts"), (forward, "query_starts")):
        with pytest.raises(ValueError, match=r"starts \[B\+1\]"):
            fn(**dict(calls[fn], **{name: None}), lib=object())


def _strided(torch, kind):
    t = _Fake(torch.zeros(3, 16, 64, 2, **kind).transpose(2, 3))
    t.get_device = lambda: 0
    return t


def test_cut_into_waves_stays_in_bounds(tmp_path):
    """The host run of the kernels' plan (tests/cpp/test_paged_q8_plan.cpp)."""
    run_program("test_paged_q8_plan", tmp_path, 6000, 1)
