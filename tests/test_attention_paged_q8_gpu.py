"""flash_attention_decode_paged_q8 and flash_attention_forward_paged_q8 against float64 on the values that
the cache holds (paged_q8_reference.py), with NaN in every row that no key has."""

from __future__ import annotations

import numpy as np
import pytest

import cuflash_attn
from cuflash_attn import synth
from paged_q8_reference import Q8Case

DTYPES = ["float32", "float16", "bfloat16"]
CODES = ["int8", "e4m3"]


def decode(c, q, **kw):
    return cuflash_attn.flash_attention_decode_paged_q8(q, *c.cache, c.t_table, c.t_lens, **kw)


def forward(c, q, starts, **kw):
    return cuflash_attn.flash_attention_forward_paged_q8(q, *c.cache, c.t_table, c.t_lens, starts,
                                                         **kw)


def queries(c, n, seed=9, std=1.0):
    x = synth.round_to(synth.normal(seed, (n, c.heads, c.d), std), c.dtype)
    return x, synth.to_torch(x, c.dtype)


def check_decode(c, scale=None, only=None):
    """Twice: from a table of the sequences' length, and from one that is too long for a decode in one
    launch."""
    if c.max_pages * c.page <= 1024:
        table = c.t_table
        more = -(-1040 // c.page) - c.max_pages
        c.t_table = c.ints(np.concatenate((c.table, np.repeat(c.table[:, :1] * 0 + c.unused, more, 1)), 1))
        if (np.asarray(c.lens) <= c.max_pages * c.page).all():
            _check_decode(c, scale, only)
        c.t_table = table
    _check_decode(c, scale, only)


def _check_decode(c, scale, only):
    B = len(c.lens)
    x, q = queries(c, B)
    o, lse = decode(c, q.view(B, c.heads, 1, c.d), scale=scale)
    c.check(x, [1] * B, False, synth.to_numpy(o)[:, :, 0], synth.to_numpy(lse)[:, :, 0], scale,
            only)


def check_forward(c, new, causal, extra=0, scale=None, only=None):
    """Twice, too: no table of 4900 keys is short for any number of rows."""
    table = c.t_table
    if int(c.t_lens.max()) <= c.max_pages * c.page < 4900:
        c.t_table = longer(c, 4900)
        _check_forward(c, new, causal, extra, scale, only)
        c.t_table = table
    _check_forward(c, new, causal, extra, scale, only)


def longer(c, keys):
    """The block table with unused pages behind, for that many keys."""
    more = -(-keys // c.page) - c.max_pages
    return c.ints(np.concatenate((c.table, np.repeat(c.table[:, :1] * 0 + c.unused, more, 1)), 1))


def _check_forward(c, new, causal, extra, scale, only):
    import torch

    T = sum(new) + extra
    x, q = queries(c, T)
    starts = c.ints([sum(new[:b]) for b in range(len(new) + 1)])
    out = torch.full_like(q, 3.0)
    o, lse = forward(c, q, starts, causal=causal, scale=scale, out=out)
    o, lse = synth.to_numpy(o), synth.to_numpy(lse)
    c.check(x, new, causal, o, lse, scale, only)
    assert (o[sum(new):] == 3.0).all()  # padding


LENS = [1, 0, 15, 16, 17, 31, 32, 33, 64, 200, 777]


@pytest.mark.gpu
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,heads,kv_heads,page", [
    (128, 8, 2, 16), (128, 4, 4, 32), (128, 40, 1, 24), (64, 6, 2, 48), (64, 32, 2, 5),
    (32, 8, 8, 16), (32, 17, 1, 1), (128, 12, 3, 64)])
def test_decode(torch_gpu, dtype, code, d, heads, kv_heads, page):
    check_decode(Q8Case(dtype, code, d, heads, kv_heads, page, LENS))


@pytest.mark.gpu
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,heads,kv_heads,page,lens", [
    (128, 32, 8, 16, [20011]), (64, 8, 1, 24, [9001, 40, 5000]), (32, 16, 16, 32, [4097] * 3)])
def test_decode_of_long_sequences(torch_gpu, dtype, code, d, heads, kv_heads, page, lens):
    check_decode(Q8Case(dtype, code, d, heads, kv_heads, page, lens, capacity=max(lens) + 700))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_decode_of_many_short_sequences(torch_gpu, dtype):
    lens = [(7 * i) % 300 for i in range(150)]
    check_decode(Q8Case(dtype, "int8", 64, 4, 2, 16, lens))


@pytest.mark.gpu
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d,heads,kv_heads,page", [
    (128, 8, 2, 16), (64, 6, 2, 24), (32, 5, 1, 32), (128, 3, 3, 64), (64, 40, 2, 16)])
def test_forward(torch_gpu, dtype, code, causal, d, heads, kv_heads, page):
    """Few and many tokens, none, more tokens than keys (rows that see no key), keys past the table."""
    new = [1, 5, 0, 40, 3, 130, 20]
    lens = [1, 64, 30, 40, 0, 301, 9]
    check_forward(Q8Case(dtype, code, d, heads, kv_heads, page, lens), new, causal, extra=4)


@pytest.mark.gpu
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,heads,kv_heads,page,new,lens", [
    (128, 8, 2, 16, [700, 61], [1500, 3001]), (64, 4, 4, 32, [1025], [1025]),
    (32, 12, 2, 8, [300, 300, 2], [300, 1000, 5000]), (128, 32, 8, 64, [5] * 6, [2000] * 6)])
def test_forward_of_prompts(torch_gpu, dtype, code, d, heads, kv_heads, page, new, lens):
    check_forward(Q8Case(dtype, code, d, heads, kv_heads, page, lens), new, True)


@pytest.mark.gpu
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,heads,kv_heads,page,new,lens", [
    (64, 8, 8, 24, [700, 500, 2, 0, 60], [0, 120, 900, 40, 61]),
    (128, 16, 2, 7, [600, 1, 1, 300], [650, 2000, 0, 299]),
    (32, 24, 1, 16, [90, 257], [0, 100]), (128, 8, 8, 16, [1, 1100], [5, 1100])])
def test_prompts_with_rows_that_see_no_key(torch_gpu, dtype, code, d, heads, kv_heads, page, new,
                                           lens):
    """So many rows that the merge goes by shares: empty sequences, more tokens than keys, tiles without a
    key, single tokens between prompts, pages of any size."""
    assert sum(new) * heads >= 8192
    c = Q8Case(dtype, code, d, heads, kv_heads, page, lens)
    check_forward(c, new, True, extra=3)
    check_forward(c, new, False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_lengths_past_the_table(torch_gpu, dtype):
    """A longer sequence is taken for as many keys as the table has."""
    c = Q8Case(dtype, "e4m3", 64, 4, 2, 16, [500, 90], capacity=96)
    check_decode(c)
    c.lens = [96, 90]  # as many keys are there
    check_forward(c, [7, 3], False)


@pytest.mark.gpu
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_scale_zero_and_large_scores(torch_gpu, dtype, code):
    c = Q8Case(dtype, code, 64, 4, 2, 16, [100, 0, 33])
    check_decode(c, scale=0.0)
    check_forward(c, [3, 2, 40], True, scale=0.0)
    check_decode(c, scale=4.0)


@pytest.mark.gpu
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("std", [2.0 ** -8, 2.0 ** 9])
def test_small_and_large_rows(torch_gpu, dtype, code, std):
    """Keys and values, and so their exponents, far from 1; one value row much larger than the rest."""
    c = Q8Case(dtype, code, 64, 4, 2, 16, [130, 40], std=std)
    pg, row = c.places[0]
    c.exps[1][pg[7], row[7]] += 5
    c.upload()
    check_decode(c, scale=1.0 / (8.0 * std))
    check_forward(c, [5, 33], True, scale=1.0 / (8.0 * std))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_poisoned_row_reaches_those_that_see_it(torch_gpu, dtype):
    """x = 255 in a value row that one of two sequences has: NaN there, and only there. In a causal forward
    queries some tokens before it, whose block of keys has it, may be NaN too (up to 94; here the tokens of a
    wave and the blocks begin at 192)."""
    torch = torch_gpu
    c = Q8Case(dtype, "int8", 64, 4, 2, 16, [300, 300])
    pg, row = c.places[1]
    c.exps[1][pg[200], row[200]] = 255
    c.upload()
    x, q = queries(c, 2)
    o, _ = decode(c, q.view(2, 4, 1, 64))
    assert bool(torch.isfinite(o[0]).all()) and bool(torch.isnan(o[1]).all())
    x, q = queries(c, 600)
    o, _ = forward(c, q, c.ints([0, 300, 600]), causal=True)
    assert bool(torch.isfinite(o[:300 + 192]).all()) and bool(torch.isnan(o[500:]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,heads,kv_heads,new", [
    (64, 4, 2, 300), (128, 8, 1, 300), (32, 2, 2, 150), (128, 8, 8, 20), (64, 8, 2, 5)])
@pytest.mark.parametrize("at", [140, 200, 298])
@pytest.mark.parametrize("table", ["short", "long"])
def test_the_reach_of_a_hidden_value(torch_gpu, dtype, d, heads, kv_heads, new, at, table):
    """A NaN value at a position changes no bit of queries that stand 95 or more before it, nor of another
    sequence, and makes those from it on NaN. The keys' rows there are NaN too in a second run: no query before
    sees them."""
    torch = torch_gpu
    c = Q8Case(dtype, "int8", d, heads, kv_heads, 16, [300, 300])
    pg, row = c.places[1]
    if table == "long":
        c.t_table = longer(c, 4900)
    t_table = c.t_table
    x, q = queries(c, 2 * new)
    starts = c.ints([0, new, 2 * new])
    clean = forward(c, q, starts, causal=True)
    c.exps[1][pg[at], row[at]] = 255
    c.upload()
    c.t_table = t_table
    o, lse = forward(c, q, starts, causal=True)
    far = new + max(0, at - 94 - (300 - new))  # tokens of both sequences before the reach
    seen = new + max(0, at - (300 - new))
    assert torch.equal(o[:far], clean[0][:far]) and torch.equal(lse, clean[1])
    assert bool(torch.isnan(o[seen:]).all())
    c.exps[1][pg[at], row[at]] = 127
    c.exps[0][pg[at], row[at]] = 255
    c.upload()
    c.t_table = t_table
    o, lse = forward(c, q, starts, causal=True)
    assert torch.equal(lse[:seen], clean[1][:seen])
    assert bool(torch.isnan(lse[seen:]).all() and torch.isnan(o[seen:]).all())


@pytest.mark.gpu
def test_decode_of_more_sequences_than_a_launch_has_workgroups(torch_gpu):
    """A million sequences of one key, or none, in one launch: O is the key's value."""
    torch = torch_gpu
    c = Q8Case("float16", "int8", 32, 8, 8, 16, [16])
    B = (1 << 20) + 1
    q = torch.ones(B, 8, 1, 32, dtype=torch.float16, device="cuda")
    lens = torch.ones(B, dtype=torch.int32, device="cuda")
    lens[::3] = 0
    table = c.t_table[0, :1].expand(B, 1).contiguous()
    o, lse = cuflash_attn.flash_attention_decode_paged_q8(q, *c.cache, table, lens)
    _, v = cuflash_attn.flash_attention_read_paged_q8(*c.cache, c.t_table, c.t_lens,
                                                      c.ints([0, 16]), 16, dtype=torch.float16)
    some = lens == 1
    assert bool((o[some] == v[0].view(1, 8, 1, 32)).all())
    assert bool((o[~some] == 0).all()) and bool(torch.isneginf(lse[~some]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_infinite_and_nan_queries(torch_gpu, dtype):
    """Of one head: NaN where scores are; the others as without."""
    torch = torch_gpu
    c = Q8Case(dtype, "e4m3", 128, 8, 2, 16, [700])
    _, q = queries(c, 1)
    q = q.view(1, 8, 1, 128)
    want, _ = decode(c, q)
    for bad in (float("nan"), float("inf")):
        p = q.clone()
        p[0, 3, 0, 5] = bad
        o, _ = decode(c, p)
        keep = [0, 1, 2, 4, 5, 6, 7]
        assert torch.equal(o[:, keep], want[:, keep])
        # An infinite score of either sign: infinity minus itself.
        assert bool(torch.isnan(o[:, 3]).all())


@pytest.mark.gpu
def test_past_32_bit_offsets(torch_gpu):
    """Keys on the last pages of a cache of over 2^32 bytes give what they give in a small one."""
    torch = torch_gpu
    c = Q8Case("bfloat16", "int8", 128, 8, 8, 64, [500, 300])
    n = c.t_k.shape[0]
    pages = (1 << 32) // (64 * 8 * 128) + n
    big = [torch.zeros((pages, *t.shape[1:]), dtype=t.dtype, device="cuda") for t in c.cache]
    for t, b in zip(c.cache, big):
        b[-n:] = t
    table = c.t_table + (pages - n)
    x, q = queries(c, 2)
    q = q.view(2, 8, 1, 128)
    want = decode(c, q)
    got = cuflash_attn.flash_attention_decode_paged_q8(q, *big, table, c.t_lens)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    x, q = queries(c, 300)
    starts = c.ints([0, 200, 300])
    want = forward(c, q, starts, causal=True)
    got = cuflash_attn.flash_attention_forward_paged_q8(q, *big, table, c.t_lens, starts,
                                                        causal=True)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
