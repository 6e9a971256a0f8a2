"""flash_attention_decode_shared against float64 (paged_reference.py), with NaN in every cache row that
no key has."""

from __future__ import annotations

import pytest

import cuflash_attn
from cuflash_attn import synth
from paged_reference import PagedCase

DTYPES = ["float32", "float16", "bfloat16"]


def run(c, scale=None, seed=9, **kw):
    B = len(c.lens)
    q = synth.round_to(synth.normal(seed, (B, c.heads, c.d)), c.dtype)
    tq = synth.to_torch(q, c.dtype).unsqueeze(2)
    o, lse = cuflash_attn.flash_attention_decode_shared(
        tq, c.t_k, c.t_v, c.t_prefix, c.prefix, c.t_table, c.t_lens, scale=scale, **kw)
    c.check(q, [1] * B, False, synth.to_numpy(o)[:, :, 0], synth.to_numpy(lse)[:, :, 0], scale)
    return tq, o, lse


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(4, 4), (8, 2), (8, 1), (6, 2)])
@pytest.mark.parametrize("prefix", [1, 48, 200])
def test_own_lengths(torch_gpu, dtype, d, heads, kv_heads, prefix):
    """Sequences with some, one and no key of their own, shorter than the prefix, and empty."""
    c = PagedCase(dtype, d, heads, kv_heads, 16, prefix=prefix,
                  lens=[prefix + 1, prefix + 100, prefix, prefix + 33, max(1, prefix - 7), 0,
                        prefix + 515])
    run(c)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [1, 6, 24, 100, 512])
@pytest.mark.parametrize("prefix", [97, 300])
def test_page_sizes(torch_gpu, dtype, page, prefix):
    """Prefixes that end inside a page, and pages that hold all of it."""
    c = PagedCase(dtype, 128, 8, 2, page, prefix=prefix,
                  lens=[prefix + 3, prefix + page, prefix + 2 * page + 1])
    run(c)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch", [2, 9, 64, 65, 150])
@pytest.mark.parametrize("heads,kv_heads", [(8, 2), (5, 1), (3, 3)])
def test_batches(torch_gpu, dtype, batch, heads, kv_heads):
    """Shared rows from one tile to several, more sequences than lanes of a wave."""
    c = PagedCase(dtype, 64, heads, kv_heads, 16, prefix=700,
                  lens=[700 + (13 * b) % 90 for b in range(batch)])
    run(c)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("prefix", [900, 8192, 8300])
def test_long_prefixes(torch_gpu, dtype, prefix):
    """Many shared rows at head_dim 128, on either side of the prefix from which other workgroups take
    them; own keys in chunks, one of them long."""
    c = PagedCase(dtype, 128, 8, 2, 16, prefix=prefix,
                  lens=[prefix + (29 * b) % 300 for b in range(37)] + [prefix + 1500, 70, 0])
    run(c)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads", [40, 128])
def test_many_heads_over_one(torch_gpu, dtype, heads):
    """More query heads of a key/value head than a tile's rows, and so many that a sequence alone
    has many rows."""
    c = PagedCase(dtype, 64, heads, 1, 16, prefix=130, lens=[131, 500, 130])
    run(c)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [0.0, 1.0])
def test_scales(torch_gpu, dtype, scale):
    c = PagedCase(dtype, 64, 8, 2, 16, prefix=333, lens=[340, 400, 333])
    run(c, scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_no_prefix_is_the_paged_decode(torch_gpu, dtype):
    torch = torch_gpu
    c = PagedCase(dtype, 64, 8, 2, 16, lens=[340, 0, 33])
    q = torch.randn((3, 8, 1, 64), device="cuda").to(c.t_k.dtype)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    got = cuflash_attn.flash_attention_decode_shared(q, c.t_k, c.t_v, none, 0, c.t_table, c.t_lens)
    want = cuflash_attn.flash_attention_decode_paged(q, c.t_k, c.t_v, c.t_table, c.t_lens)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_no_prefix_captured(torch_gpu, dtype):
    """A server's graph without a prefix yet: its memory is the caller's here, too."""
    torch = torch_gpu
    c = PagedCase(dtype, 64, 8, 2, 16, lens=[340, 0, 33, 1])
    q = torch.randn((4, 8, 1, 64), device="cuda").to(c.t_k.dtype)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, lse = cuflash_attn.flash_attention_decode_shared(q, c.t_k, c.t_v, none, 0, c.t_table,
                                                            c.t_lens)
    torch.cuda.synchronize()
    for rep in range(3):
        print(f"[no prefix, captured] replay {rep}", flush=True)
        q.normal_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        c.check(synth.to_numpy(q)[:, :, 0], [1] * 4, False, synth.to_numpy(o)[:, :, 0],
                synth.to_numpy(lse)[:, :, 0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_non_finite_scores(torch_gpu, dtype):
    """Shared keys of -inf leave the own ones; a NaN among the shared keys reaches the sequences that
    see it, not those that end before it."""
    torch = torch_gpu
    inf = float("inf")
    c = PagedCase(dtype, 64, 2, 2, 16, prefix=40, lens=[41, 40, 20, 60])
    q = torch.ones((4, 2, 1, 64), device="cuda", dtype=c.t_k.dtype)
    args = (c.t_prefix, 40, c.t_table, c.t_lens)
    for j in range(40):
        c.t_k[int(c.prefix_table[j // 16]), j % 16] = -inf
    o, lse = cuflash_attn.flash_attention_decode_shared(q, c.t_k, c.t_v, *args)
    page = int(c.table[0, 40 // 16])
    assert torch.equal(o[0, :, 0], c.t_v[page, 40 % 16])
    assert bool((o[1:3] == 0).all() and (lse[1:3] == -inf).all())
    assert bool(torch.isfinite(o[3].float()).all() and torch.isfinite(lse[3]).all())
    c.t_k[int(c.prefix_table[30 // 16]), 30 % 16] = float("nan")
    o, lse = cuflash_attn.flash_attention_decode_shared(q, c.t_k, c.t_v, *args)
    assert bool(torch.isnan(lse[[0, 1, 3]]).all() and torch.isnan(o[[0, 1, 3]].float()).all())
    assert bool((o[2] == 0).all() and (lse[2] == -inf).all())


@pytest.mark.gpu
def test_captured_and_on_another_stream(torch_gpu):
    torch = torch_gpu
    c = PagedCase("bfloat16", 128, 32, 8, 16, prefix=1000, lens=[1001, 1300, 1100, 1200, 900])
    q = torch.randn((5, 32, 1, 128), device="cuda").bfloat16()

    def fn(**kw):
        return cuflash_attn.flash_attention_decode_shared(q, c.t_k, c.t_v, c.t_prefix, 1000,
                                                          c.t_table, c.t_lens, **kw)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    there = fn(stream=side)
    side.synchronize()
    here = fn()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(there, here))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fn()
    torch.cuda.synchronize()
    for rep in range(3):
        print(f"[decode_shared graph] replay {rep}", flush=True)
        q.normal_()
        c.t_lens.copy_(torch.tensor([1001, 1300 - rep, 1100, 1200, 0], device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in out]
        eager = fn()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, eager)), rep
