"""NaN and infinite VALUES of keys that a query does not see (include/cuflash/paged_cache.h): how far they
reach in the paged forward and in the shared decode. Finite hidden values change nothing, as their weight is
0, so what is out of reach must give the clean run's bits."""

from __future__ import annotations

import pytest

import cuflash_attn
from paged_reference import PagedCase

DTYPES = ["float32", "float16", "bfloat16"]
INF, NAN = float("inf"), float("nan")


def put(c, keys, value, table=None):
    """`value` into the values of keys of sequence 0, or of the pages that `table` names."""
    table = c.table[0] if table is None else table
    for j in keys:
        c.t_v[int(table[j // c.page]), j % c.page] = value


def same(a, b):
    import torch

    return torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,heads,kv_heads", [(32, 2, 2), (64, 1, 1), (64, 6, 2), (128, 2, 2), (128, 8, 2)])
@pytest.mark.parametrize("n,old", [(96, 40), (300, 40), (300, 1000), (700, 0)])
def test_later_tokens_of_a_prompt(torch_gpu, dtype, d, heads, kv_heads, n, old):
    """The value of one token: NaN where it is seen, nothing more than 94 positions before it."""
    torch = torch_gpu
    c = PagedCase(dtype, d, heads, kv_heads, 16, lens=[old + n])
    q = torch.randn((n, heads, d), device="cuda").to(c.t_k.dtype)
    starts = c.ints([0, n])

    def run():
        return cuflash_attn.flash_attention_forward_paged(q, c.t_k, c.t_v, c.t_table, c.t_lens, starts,
                                                          causal=True)

    clean, values = run(), c.t_v.clone()
    for j, value in ((old + n - 1, NAN), (old + 95, INF), (old + n // 2 + 50, -INF)):
        if j >= old + n:
            continue
        put(c, [j], value)
        o, lse = run()
        c.t_v.copy_(values)
        out = max(0, j - 95 - old + 1)  # queries from positions old to j - 95
        assert torch.equal(o[:out], clean[0][:out]), (j, "out of reach")
        assert torch.equal(lse, clean[1]), j  # no value has a part in L
        seen = o[j - old:].float()
        assert not bool(torch.isfinite(seen).any()), (j, "seen")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("n", [20, 200])
def test_queries_without_keys(torch_gpu, dtype, d, n):
    """More tokens than keys: the first ones see nothing, however the values behind look."""
    torch = torch_gpu
    c = PagedCase(dtype, d, 4, 4, 16, lens=[n - 9])
    put(c, range(n - 9), NAN)
    q = torch.randn((n, 4, d), device="cuda").to(c.t_k.dtype)
    o, lse = cuflash_attn.flash_attention_forward_paged(q, c.t_k, c.t_v, c.t_table, c.t_lens,
                                                        c.ints([0, n]), causal=True)
    assert bool((o[:9] == 0).all() and (lse[:9] == -INF).all())
    assert bool(torch.isnan(o[9:].float()).all() and torch.isfinite(lse[9:]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("value", [NAN, INF])
def test_waves_without_keys_of_a_short_sequence(torch_gpu, dtype, d, value):
    """Few rows behind 128 shared keys, one block of 32 per wave: the waves whose blocks a sequence of 20
    keys does not reach have no say in its result."""
    torch = torch_gpu
    c = PagedCase(dtype, d, 8, 2, 16, prefix=128, lens=[129, 20, 200, 0, 32])
    q = torch.randn((5, 8, 1, d), device="cuda").to(c.t_k.dtype)

    def run():
        return cuflash_attn.flash_attention_decode_shared(q, c.t_k, c.t_v, c.t_prefix, 128, c.t_table,
                                                          c.t_lens)

    clean = run()
    put(c, range(32, 128), value, c.prefix_table)
    o, lse = run()
    short = [1, 3, 4]
    assert torch.equal(o[short], clean[0][short]) and torch.equal(lse, clean[1])
    assert bool((o[3] == 0).all() and (lse[3] == -INF).all())
    assert not bool(torch.isfinite(o[[0, 2]].float()).any())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128])
def test_chunks_without_keys_of_a_short_sequence(torch_gpu, dtype, d):
    """Many rows behind a prefix in chunks: those that a sequence does not reach have no say."""
    torch = torch_gpu
    prefix = 8190
    c = PagedCase(dtype, d, 8, 2, 16, prefix=prefix, lens=[prefix + b % 5 for b in range(60)] + [20, 0])
    q = torch.randn((62, 8, 1, d), device="cuda").to(c.t_k.dtype)

    def run():
        return cuflash_attn.flash_attention_decode_shared(q, c.t_k, c.t_v, c.t_prefix, prefix,
                                                          c.t_table, c.t_lens)

    clean = run()
    put(c, range(prefix - 40, prefix), NAN, c.prefix_table)
    o, lse = run()
    assert torch.equal(o[60:], clean[0][60:]) and torch.equal(lse, clean[1])
    assert bool(torch.isnan(o[:60].float()).all())
