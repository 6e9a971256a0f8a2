"""Numbers of an 8-bit paged cache that fp16 has not (a cache that a bf16 or fp32 append wrote, read by fp16
queries): each takes part as its nearest fp16 number, or as an infinity, whichever kernel a call takes. Keys and
values in float64 are those that numpy rounds to fp16."""

from __future__ import annotations

import numpy as np
import pytest

import cuflash_attn
from cuflash_attn import synth
from paged_q8_reference import Q8Case, values
from paged_reference import attention, attention_bounds
from test_attention_paged_q8_gpu import decode, longer, queries

# head_dim, heads, key/value heads, page: pages of 16 n, 4 n and other rows.
SHAPES = [(64, 16, 2, 16), (128, 8, 1, 24), (32, 32, 4, 5)]
NEW = [40, 25]
LENS = [40, 61]


def rounded(x):
    with np.errstate(over="ignore"):
        return x.astype(np.float16).astype(np.float64)


def check(c, x, new, causal, o, lse, scale, dead=()):
    """Against float64. Keys of sequence 0 in `dead` are infinite in element 3 and 0 elsewhere: a row whose
    element 3 is negative gives them no weight, one that is positive is NaN where it sees one."""
    group, t0 = c.heads // c.kv_heads, 0
    for b, n in enumerate(new):
        keys, vals = (rounded(v) for v in c.sequence(b))
        drop = list(dead) if b == 0 else []
        for h in range(c.kv_heads):
            at = (slice(t0, t0 + n), slice(h * group, (h + 1) * group))
            rows = x[at].reshape(n * group, c.d)
            limits = np.repeat([max(0, len(keys) - n + i + 1) if causal else len(keys)
                                for i in range(n)], group)
            nan = (rows[:, 3] > 0) & (limits > min(drop, default=1 << 30))
            left = limits - sum((limits > j).astype(int) for j in drop)
            k, v = (np.delete(t[:, h], drop, 0) for t in (keys, vals))
            want = attention(rows, k, v, scale, left)
            o_bound, l_bound = attention_bounds("float16", c.d, len(k), *want, abs(v).sum(0))
            got_o, got_l = o[at].reshape(n * group, c.d), lse[at].reshape(n * group)
            assert np.isnan(got_o[nan]).all(), (b, h)
            assert (abs(got_o - want[0]) <= o_bound)[~nan].all(), (b, h)
            some = ~nan & (left > 0)
            assert (abs(got_l - want[1])[some] <= l_bound[some]).all(), (b, h)
            assert np.isneginf(got_l[~nan & (left == 0)]).all()
        t0 += n


def check_all(c, x, q, scale, dead=()):
    """Tokens of several rows a tile and one, in one launch (short tables) and not: NEW's rows are many enough
    for the prompts' kernel, two tokens of each sequence are not, a decode has one."""
    short = c.t_table
    for table in (short, longer(c, 4900)):
        c.t_table = table
        for new in (NEW, [2, 2]):
            T = sum(new)
            starts = c.ints([0, new[0], T])
            for causal in (True, False):
                o, lse = cuflash_attn.flash_attention_forward_paged_q8(
                    q[:T], *c.cache, table, c.t_lens, starts, scale=scale, causal=causal)
                check(c, x[:T], new, causal, synth.to_numpy(o), synth.to_numpy(lse), scale, dead)
        o, lse = decode(c, q[:2].reshape(2, c.heads, 1, c.d), scale=scale)
        check(c, x[:2], [1, 1], False, synth.to_numpy(o)[:, :, 0], synth.to_numpy(lse)[:, :, 0],
              scale, dead)
    c.t_table = short


@pytest.mark.gpu
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("d,heads,kv_heads,page", SHAPES)
def test_keys_below_the_numbers_of_fp16(torch_gpu, code, d, heads, kv_heads, page):
    """Exponents around 103, from which on fp16 has every number of int8 codes."""
    c = Q8Case("float16", code, d, heads, kv_heads, page, LENS)
    for b in range(2):
        pg, row = c.places[b]
        j = np.arange(len(pg))
        c.exps[0][pg, row] = (98 + j % 7)[:, None]
    c.upload()
    x, q = queries(c, sum(NEW))
    check_all(c, x, q, 2.0 ** 16)


@pytest.mark.gpu
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("d,heads,kv_heads,page", SHAPES)
def test_keys_above_the_numbers_of_fp16(torch_gpu, code, d, heads, kv_heads, page):
    """Large finite elements, from exponents within fp16's range and beyond it, beside infinite ones."""
    c = Q8Case("float16", code, d, heads, kv_heads, page, LENS)
    one = {"int8": lambda n: n, "e4m3": lambda n: {1: 0x38, 7: 0x4E, 100: 0x6C, 127: 0x70}[n]}[code]
    pg, row = c.places[0]
    # key: element, code, exponent. 1, 7 and 128 (int8: 127) are numbers of e4m3, too; 0x6c is 96.
    for key, (at, n, exp) in {9: (5, 127, 135), 11: (6, 1, 140), 14: (2, 7, 139),
                              17: (3, 100, 137), 20: (3, 100, 145)}.items():
        c.codes[0][pg[key], row[key]] = 0
        c.codes[0][pg[key], row[key], :, at] = one(n)
        c.exps[0][pg[key], row[key]] = exp
        k = values(c.codes[0][pg[key], row[key]], c.exps[0][pg[key], row[key]], code)
        assert np.isinf(rounded(k)).any() == (key in (17, 20))
    c.upload()
    x, q = queries(c, sum(NEW))
    x[:, ::2, 3], x[:, 1::2, 3] = -abs(x[:, ::2, 3]) - 0.125, abs(x[:, 1::2, 3]) + 0.125
    x = synth.round_to(x, "float16")
    check_all(c, x, synth.to_torch(x, "float16"), 2.0 ** -17, dead=(17, 20))


@pytest.mark.gpu
@pytest.mark.parametrize("d,heads,kv_heads,page", SHAPES)
def test_a_key_within_a_block_of_others(torch_gpu, d, heads, kv_heads, page):
    """int8 keys of ordinary exponents give the same bits whether a key of their block that no query sees is
    beyond fp16's numbers or not: the block's codes are scaled before the product or after it."""
    torch = torch_gpu
    c = Q8Case("float16", "int8", d, heads, kv_heads, page, [61, 61])
    x, q = queries(c, 4)
    c.t_table = table = longer(c, 4900)
    c.t_lens = lens = c.ints([60, 60])
    starts = c.ints([0, 2, 4])

    def run():
        c.t_table, c.t_lens = table, lens
        return torch.cat([cuflash_attn.flash_attention_forward_paged_q8(
            q, *c.cache, table, lens, starts, causal=True)[0].flatten(),
            decode(c, q[:2].reshape(2, heads, 1, d))[0].flatten()])

    pg, row = c.places[0]
    c.exps[0][pg[60], row[60]] = 120
    c.upload()
    want = run()
    c.exps[0][pg[60], row[60]] = 150
    c.upload()
    assert torch.equal(run(), want)
