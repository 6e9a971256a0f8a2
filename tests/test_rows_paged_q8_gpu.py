"""flash_attention_append_paged_q8 and flash_attention_read_paged_q8: codes, exponents and rotated
queries bit for bit what the definition gives (paged_q8_reference.py), everything else as it was."""

from __future__ import annotations

import numpy as np
import pytest

import cuflash_attn
from cuflash_attn import synth
from paged_q8_reference import quantise, rotate32, torch_cache, values
from paged_reference import positions

DTYPES = ["float32", "float16", "bfloat16"]
CODES = ["int8", "e4m3"]


def _bits(t):
    import torch

    return t.view(torch.uint8).cpu().numpy()


class Case:
    def __init__(self, dtype, code, d, heads, kv_heads, page, new, old, rotary, interleaved=False,
                 extra=0, apart=0, seed=1, rows=None):
        import torch

        self.dtype, self.code, self.d = dtype, code, d
        self.heads, self.kv_heads, self.page = heads, kv_heads, page
        self.interleaved, self.rotary = interleaved, rotary
        B = len(new)
        self.lens = [n + o for n, o in zip(new, old)]
        self.starts = [sum(new[:b]) for b in range(B + 1)]
        T = self.T = self.starts[-1] + extra  # `extra` padding tokens
        width = (heads + 2 * kv_heads) * d + apart
        if rows is None:
            rows = synth.normal(seed, (T, width))
            # Rows of all magnitudes.
            rows *= (2.0 ** np.random.default_rng(seed).integers(-12, 10, (T, 1))).astype(np.float32)
        rows = synth.round_to(rows, dtype)
        heads_of = lambda x, at, n: x[:, at * d:(at + n) * d].reshape(T, n, d)  # noqa: E731
        self.q, self.k, self.v = (heads_of(rows, at, n) for at, n in (
            (0, heads), (heads, kv_heads), (heads + kv_heads, kv_heads)))
        max_pages = max(1, max(-(-n // page) for n in self.lens))
        self.pages = B * max_pages + 2
        rng = np.random.default_rng(seed)
        self.table = rng.permutation(self.pages)[:B * max_pages].reshape(B, max_pages)
        shape = (self.pages, page, kv_heads, d)
        self.codes0 = [rng.integers(0, 256, shape).astype(np.uint8) for _ in range(2)]
        self.exps0 = [rng.integers(0, 256, shape[:3]).astype(np.uint8) for _ in range(2)]
        n = max(1, max(self.lens))
        if rotary:
            angle = np.arange(n)[:, None] * 1e4 ** (-np.arange(rotary // 2) / (rotary // 2))
            self.cos, self.sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
        t = synth.to_torch(rows, dtype)
        self.tq, self.tk, self.tv = (
            t[:, at * d:(at + n) * d].unflatten(1, (n, d)) for at, n in (
                (0, heads), (heads, kv_heads), (heads + kv_heads, kv_heads)))
        ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
        self.t_table, self.t_lens, self.t_starts = (
            ints(self.table.tolist()), ints(self.lens), ints(self.starts))
        self.t_cos, self.t_sin = ((torch.from_numpy(x).cuda() for x in (self.cos, self.sin))
                                  if rotary else (None, None))
        self.caches = [torch_cache(c, code) for c in self.codes0]
        self.exps = [torch.from_numpy(e.transpose(0, 2, 1).copy()).cuda() for e in self.exps0]

    def run(self, **kw):
        args = dict(q=self.tq, cos=self.t_cos, sin=self.t_sin, interleaved=self.interleaved,
                    query_starts=self.t_starts)
        args.update(kw)
        return cuflash_attn.flash_attention_append_paged_q8(
            self.tk, self.tv, *self.caches, *self.exps, self.t_table, self.t_lens, **args)

    def turned(self, x):
        if not self.rotary:
            return x
        pos = np.zeros(self.T, dtype=np.int64)
        for t, _, p in positions(self.lens, self.starts):
            pos[t] = max(p, 0)
        return rotate32(x, pos, self.cos, self.sin, self.interleaved)

    def want(self, skip=()):
        """Codes and exponents of the caches after the append, without the tokens of `skip`."""
        codes, exps = [c.copy() for c in self.codes0], [e.copy() for e in self.exps0]
        for i, x in enumerate((self.turned(self.k), self.v)):
            c, e = quantise(x, self.code, self.dtype)
            for t, b, p in positions(self.lens, self.starts):
                if p >= 0 and t not in skip:
                    at = self.table[b, p // self.page], p % self.page
                    codes[i][at], exps[i][at] = c[t], e[t]
        return codes, exps

    def check(self, got_q, skip=(), nan=()):
        codes, exps = self.want(set(skip) | set(nan))
        for i in range(2):
            assert np.array_equal(_bits(self.caches[i]), codes[i]), "kv"[i]
            assert np.array_equal(self.exps[i].cpu().numpy().transpose(0, 2, 1), exps[i]), "kv"[i]
        if got_q is not None:
            want = synth.round_to(self.turned(self.q), self.dtype)
            keep = [t for t in range(self.starts[-1]) if t not in nan]
            assert np.array_equal(synth.to_numpy(got_q)[keep], want[keep])


@pytest.mark.gpu
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,heads,kv_heads,page,rotary,interleaved", [
    (128, 8, 2, 16, 128, False), (128, 4, 4, 7, 64, True), (64, 6, 3, 24, 64, True),
    (64, 4, 1, 1, 32, False), (32, 8, 8, 32, 32, False), (32, 2, 1, 5, 16, True),
    (128, 40, 8, 16, 128, True), (128, 5, 5, 16, 0, False)])
def test_append(torch_gpu, dtype, code, d, heads, kv_heads, page, rotary, interleaved):
    c = Case(dtype, code, d, heads, kv_heads, page, new=[1, 33, 0, 7, 2], old=[0, 15, 40, 100, 63],
             rotary=rotary, interleaved=interleaved, extra=3, apart=32)
    out = torch_gpu.full((c.T, heads, d), 3.0, dtype=c.tq.dtype, device="cuda")
    c.check(c.run(out=out))
    assert bool((out[c.starts[-1]:] == 3.0).all())  # padding


@pytest.mark.gpu
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_append_one_token_each_without_queries(torch_gpu, dtype, code):
    c = Case(dtype, code, 64, 4, 2, 16, new=[1] * 70, old=list(range(70)), rotary=64)
    assert c.run(q=None, query_starts=None) is None
    c.check(None)


@pytest.mark.gpu
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_at_the_edges(torch_gpu, dtype, code):
    """Zeros, signed zeros, ties, numbers just above and below a power of the top code, the type's largest and
    smallest, subnormal ones, infinities and NaN."""
    d = 64
    top = {"int8": 127.0, "e4m3": 448.0}[code]
    big = {"float32": 3.4028235e38, "float16": 65504.0, "bfloat16": 3.3895314e38}[dtype]
    least = {"float32": 1e-45, "float16": 2.0 ** -24, "bfloat16": 2.0 ** -133}[dtype]
    rows = [np.zeros(d), -np.zeros(d), np.full(d, big), np.full(d, -big), np.full(d, least),
            np.linspace(-big, big, d), np.linspace(-least * 9, least * 9, d)]
    for e in (-30, -9, -1, 0, 3):
        for f in (1.0, 1.0 + 2.0 ** -7, 1.0 - 2.0 ** -8, 1.0 + 2.0 ** -10, 1.0 + 2.0 ** -23):
            r = np.linspace(-1.0, 1.0, d) * top * 2.0 ** e * f
            r[5:9] = np.array([0.5, 1.5, 2.5, 17.0]) * 2.0 ** e  # ties where the top fits
            rows.append(r)
    for bad in (np.inf, -np.inf, np.nan):
        r = np.linspace(-1.0, 1.0, d)
        r[17] = bad
        rows.append(r)
    with np.errstate(over="ignore"):
        one = np.stack(rows).astype(np.float32)
    T = len(rows)
    c = Case(dtype, code, d, 1, 1, 16, new=[T], old=[3], rotary=0,
             rows=np.concatenate((one, one, one[::-1]), 1))
    c.run(q=None)
    c.check(None)
    k, v = cuflash_attn.flash_attention_read_paged_q8(
        *c.caches, *c.exps, c.t_table, c.t_lens, c.t_starts, T, dtype=c.tk.dtype)
    k = synth.to_numpy(k)[:, 0]
    bad = ~np.isfinite(one).all(1) if dtype != "float32" else ~np.isfinite(one).all(1)
    rounded = synth.round_to(one, dtype)
    bad |= ~np.isfinite(rounded).all(1)
    assert np.isnan(k[bad]).all() and np.isfinite(k[~bad]).all()
    # Half a step of the code, relative to the element or to the row's largest (int8: of its exponent's
    # 127 steps; e4m3: 2^-4 of the element, 2^-10 of the exponent's unit); the largest, where the
    # exponent is at its greatest, up to what it is past the top.
    with np.errstate(invalid="ignore", over="ignore"):
        err = abs(k.astype(np.float64) - rounded)[~bad]
        amax = abs(rounded.astype(np.float64)).max(1)[~bad, None]
    unit = np.maximum(amax / top * 2.0, 2.0 ** -100)
    step = unit / 2 if code == "int8" else np.maximum(abs(rounded[~bad]) * 2.0 ** -4, unit * 2.0 ** -10)
    over = np.maximum(amax - top * 2.0 ** {"float16": 9 if code == "int8" else 7}.get(
        dtype, 121 if code == "int8" else 119), 0.0)
    assert (err <= step + over + 2.0 ** -25 * (dtype == "float16")).all()


@pytest.mark.gpu
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_tokens_without_a_row(torch_gpu, dtype, code):
    """Positions before 0 and past the table, pages outside the cache: not written, read as NaN."""
    c = Case(dtype, code, 64, 2, 2, 8, new=[5, 6, 4], old=[-2, 10, 20], rotary=32)
    c.table[1, 1] = -1
    c.table[2, 2] = c.pages
    c.t_table = torch_gpu.tensor(c.table.tolist(), dtype=torch_gpu.int32, device="cuda")
    places = positions(c.lens, c.starts)
    skip = [t for t, b, p in places
            if p < 0 or (b == 1 and p // 8 == 1) or (b == 2 and p // 8 == 2)]
    nan = [t for t, _, p in places if p < 0]
    assert len(skip) == 2 + 6 + 4
    got = c.run()
    c.check(got, skip=skip, nan=nan)
    assert bool(torch_gpu.isnan(got[nan][..., :32]).all())
    k, v = cuflash_attn.flash_attention_read_paged_q8(
        *c.caches, *c.exps, c.t_table, c.t_lens, c.t_starts, c.T, dtype=c.tk.dtype)
    gone = torch_gpu.isnan(k).all(-1).all(-1)
    assert gone.nonzero().flatten().tolist() == skip
    assert torch_gpu.equal(gone, torch_gpu.isnan(v).all(-1).all(-1))


@pytest.mark.gpu
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,kv_heads,page", [(128, 8, 16), (64, 3, 5), (32, 1, 1), (128, 9, 32)])
def test_read(torch_gpu, dtype, code, d, kv_heads, page):
    """Every code and every exponent, as the definition has them, rounded once to the type."""
    torch = torch_gpu
    rng = np.random.default_rng(d)
    lens, new = [37, 0, 5, 260], [30, 0, 5, 255]
    starts = np.cumsum([0] + new)
    pages = sum(-(-n // page) for n in lens) + 3
    order, at = rng.permutation(pages), 0
    table = np.zeros((4, -(-260 // page)), dtype=np.int64)
    for b, n in enumerate(lens):
        m = -(-n // page)
        table[b, :m] = order[at:at + m]
        at += m
    codes = [rng.integers(0, 256, (pages, page, kv_heads, d)).astype(np.uint8) for _ in range(2)]
    exps = [rng.integers(0, 256, (pages, page, kv_heads)).astype(np.uint8) for _ in range(2)]
    codes = [np.where(c == 128, 1, c) for c in codes]
    ints = lambda x: torch.tensor(np.asarray(x).tolist(), dtype=torch.int32,  # noqa: E731
                                  device="cuda")
    t_dtype = getattr(torch, dtype)
    T = int(starts[-1])
    outs = [torch.full((T + 2, kv_heads, d), 5.0, dtype=t_dtype, device="cuda") for _ in range(2)]
    cuflash_attn.flash_attention_read_paged_q8(
        *(torch_cache(c, code) for c in codes),
        *(torch.from_numpy(e.transpose(0, 2, 1).copy()).cuda() for e in exps), ints(table),
        ints(lens), ints(starts), T + 2, k_out=outs[0], v_out=outs[1])
    for out, c, e in zip(outs, codes, exps):
        got = synth.to_numpy(out)
        assert (got[T:] == 5.0).all()
        for t, b, p in positions(lens, starts):
            pg = table[b, p // page]
            with np.errstate(over="ignore"):
                want = values(c[pg, p % page], e[pg, p % page], code)
                want = (want.astype(np.float16) if dtype == "float16"
                        else synth.round_to(want.astype(np.float32), dtype)).astype(np.float32)
            assert np.array_equal(got[t], want, equal_nan=True), (t, b, p)


@pytest.mark.gpu
def test_append_past_32_bit_offsets(torch_gpu):
    """Pages of a cache of over 2^32 bytes: rows on its last ones, and what is read there."""
    torch = torch_gpu
    page, Hkv, D = 64, 8, 128
    pages = (1 << 32) // (page * Hkv * D) + 40
    cache = [torch.zeros((pages, page, Hkv, D), dtype=torch.int8, device="cuda") for _ in range(2)]
    exps = [torch.zeros((pages, Hkv, page), dtype=torch.uint8, device="cuda") for _ in range(2)]
    table = torch.arange(pages - 4, pages, device="cuda", dtype=torch.int32).view(1, 4)
    lens = torch.tensor([256], dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, 256], dtype=torch.int32, device="cuda")
    k, v = (torch.randn((256, Hkv, D), device="cuda").bfloat16() for _ in range(2))
    cuflash_attn.flash_attention_append_paged_q8(k, v, *cache, *exps, table, lens, starts)
    for x, c, e in zip((k, v), cache, exps):
        codes, want = quantise(synth.to_numpy(x), "int8", "bfloat16")
        assert np.array_equal(c[-4:].cpu().numpy().view(np.uint8).reshape(256, Hkv, D), codes)
        assert np.array_equal(e[-4:].cpu().numpy().transpose(0, 2, 1).reshape(256, Hkv), want)
        assert int(c[:40].count_nonzero()) == 0
    got = cuflash_attn.flash_attention_read_paged_q8(*cache, *exps, table, lens, starts, 256)
    for x, y in zip((k, v), got):
        assert float((x.float() - y.float()).abs().max()) <= 2.0 ** -5  # half a step of |x| < 8
