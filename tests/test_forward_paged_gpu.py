"""flash_attention_forward_paged against float64 (paged_reference.py), with NaN in every cache row
that no key has."""

from __future__ import annotations

import numpy as np
import pytest

import cuflash_attn
from cuflash_attn import synth
from paged_reference import PagedCase

DTYPES = ["float32", "float16", "bfloat16"]


def run(c, new, causal=True, scale=None, padding=0, seed=9, std=1.0, **kw):
    """One call with new[b] tokens of sequence b and its check; O and L as they came."""
    T = sum(new) + padding
    q = synth.round_to(synth.normal(seed, (T, c.heads, c.d), std), c.dtype)
    starts = np.concatenate([[0], np.cumsum(new)])
    o, lse = cuflash_attn.flash_attention_forward_paged(
        synth.to_torch(q, c.dtype), c.t_k, c.t_v, c.t_table, c.t_lens, c.ints(starts), scale=scale,
        causal=causal, **kw)
    c.check(q, new, causal, synth.to_numpy(o), synth.to_numpy(lse), scale)
    return o, lse


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("heads,kv_heads", [(4, 4), (8, 2), (8, 1), (6, 2)])
@pytest.mark.parametrize("causal", [True, False])
def test_mixed_lengths(torch_gpu, dtype, d, heads, kv_heads, causal):
    """Prompts, next turns, single tokens and sequences without tokens in one call."""
    new = [70, 1, 0, 5, 300, 33]
    c = PagedCase(dtype, d, heads, kv_heads, 16, lens=[70, 500, 40, 260, 333, 33])
    run(c, new, causal)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("page", [1, 2, 6, 8, 24, 100, 512])
def test_page_sizes(torch_gpu, dtype, d, page):
    c = PagedCase(dtype, d, 4, 2, page, lens=[257, 90, 31, 3])
    run(c, [150, 9, 31, 1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n", [1, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257])
def test_row_and_key_borders(torch_gpu, dtype, d, n):
    """Rows and keys around the tiles' borders, in a sequence of its own and behind another."""
    c = PagedCase(dtype, d, 3, 1, 16, lens=[n, 4 * n + 1])
    run(c, [n, n])
    run(c, [n, 1], causal=False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv_heads", [(40, 1), (32, 8), (5, 5)])
def test_long_caches_in_chunks(torch_gpu, dtype, heads, kv_heads):
    """Few tokens against long caches: keys in chunks, merged; one sequence and several."""
    c = PagedCase(dtype, 128, heads, kv_heads, 32, lens=[5000])
    run(c, [3])
    run(c, [40])
    c = PagedCase(dtype, 64, heads, kv_heads, 32, lens=[4100, 17, 2500, 0])
    run(c, [2, 2, 60, 0])
    run(c, [1, 1, 1, 0], causal=False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_many_sequences(torch_gpu, dtype):
    """More sequences than lanes of a wave, with and without tokens."""
    lens = [(37 * b) % 200 for b in range(150)]
    new = [min(n, (b * 7) % 5) for b, n in enumerate(lens)]
    new[70] = lens[70] = 120
    c = PagedCase(dtype, 64, 4, 2, 16, lens=lens)
    run(c, new)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch", [700, 4200])
def test_hundreds_of_sequences(torch_gpu, dtype, batch):
    """So many that a workgroup keeps their lengths in LDS, and more than it has room for."""
    lens = [(37 * b) % 90 for b in range(batch)]
    new = [min(n, (b * 7) % 3) for b, n in enumerate(lens)]
    for b, n in ((batch // 2, 2000), (batch - 1, 700), (3, 300)):
        lens[b], new[b] = n, min(n, 150) if b > 3 else 1
    c = PagedCase(dtype, 32, 2, 1, 16, lens=lens)
    run(c, new)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_prompts_of_a_hundred_sequences(torch_gpu, dtype):
    """Rows that fill the chip, so that no keys are cut."""
    lens = [100 + (53 * b) % 130 for b in range(100)]
    lens[40] = 1500
    c = PagedCase(dtype, 32, 8, 8, 16, lens=lens)
    run(c, [n - b % 3 for b, n in enumerate(lens)])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [32, 128])
def test_rows_without_keys_and_padding(torch_gpu, dtype, d):
    """Lengths of zero and below, fewer keys than tokens (the first ones see nothing), a length past
    the block table, padding tokens that stay as they were."""
    torch = torch_gpu
    lens = [0, -3, 4, 2, 130]
    c = PagedCase(dtype, d, 4, 2, 16, lens=lens, capacity=96)
    new = [2, 1, 9, 120, 40]
    for causal in (True, False):
        T = sum(new) + 7
        out = torch.full((T, 4, d), 5.0, device="cuda", dtype=c.t_k.dtype)
        lse = torch.full((T, 4), 5.0, device="cuda")
        run(c, new, causal, padding=7, out=out, lse=lse)
        assert bool((out[sum(new):] == 5.0).all() and (lse[sum(new):] == 5.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [0.0, 1.0, 0.37])
def test_scales(torch_gpu, dtype, scale):
    """Scale 0 weighs every visible key alike; 1 has scores of some tens."""
    c = PagedCase(dtype, 64, 4, 2, 16, lens=[300, 70])
    run(c, [130, 3], scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_non_finite_scores(torch_gpu, dtype):
    """A key that gives -inf has no weight, a row of such scores O = 0 and L = -inf; +inf and NaN
    make NaN, in the rows that see them only (their values are finite)."""
    torch = torch_gpu
    inf = float("inf")
    for rows in (6, 160):  # few rows, many rows
        c = PagedCase(dtype, 64, 1, 1, 16, lens=[rows, rows])
        q = torch.ones((2 * rows, 1, 64), device="cuda", dtype=c.t_k.dtype)
        starts = c.ints([0, rows, 2 * rows])
        pages = [(int(c.table[b, j // 16]), j % 16) for b in (0, 1) for j in range(rows)]
        for b, j in pages[:rows]:
            c.t_k[b, j] = -inf
        b, j = pages[rows + 4]
        c.t_k[b, j] = inf
        o, lse = cuflash_attn.flash_attention_forward_paged(q, c.t_k, c.t_v, c.t_table, c.t_lens,
                                                            starts, causal=True)
        assert bool((o[:rows] == 0).all() and (lse[:rows] == -inf).all())
        assert bool(torch.isfinite(o[rows:rows + 4].float()).all())
        assert bool(torch.isfinite(lse[rows:rows + 4]).all())
        assert bool(torch.isnan(o[rows + 4:].float()).all() and torch.isnan(lse[rows + 4:]).all())
        # Sequence 0 with one finite key: its value, from there on.
        b, j = pages[2]
        c.t_k[b, j] = 0.5
        o, lse = cuflash_attn.flash_attention_forward_paged(q, c.t_k, c.t_v, c.t_table, c.t_lens,
                                                            starts, causal=True)
        assert bool((o[:2] == 0).all() and torch.equal(o[2:rows, 0],
                                                       c.t_v[b, j].expand(rows - 2, 64)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "float16"])
def test_captured_and_on_another_stream(torch_gpu, dtype):
    """Captured calls, one with chunks, share nothing: replayed in turn on new inputs, with eager
    calls in between; and a call on a side stream."""
    torch = torch_gpu
    calls = []
    for lens, new in (([3000, 40], [2, 3]), ([200, 333], [200, 130])):
        c = PagedCase(dtype, 128, 8, 2, 16, lens=lens)
        q = torch.empty((sum(new), 8, 128), device="cuda", dtype=c.t_k.dtype)
        starts = c.ints(np.concatenate([[0], np.cumsum(new)]))
        fn = lambda c=c, q=q, s=starts, **kw: cuflash_attn.flash_attention_forward_paged(  # noqa: E731
            q, c.t_k, c.t_v, c.t_table, c.t_lens, s, causal=True, **kw)
        q.normal_()
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
        calls.append((c, q, fn, graph, out, lens))
    for rep in range(3):
        print(f"[forward_paged graphs] replay {rep}", flush=True)
        for c, q, fn, graph, out, lens in calls:
            q.normal_()
            c.t_lens.copy_(torch.tensor([n - rep for n in lens], device="cuda"))
        torch.cuda.synchronize()
        for *_, graph, out, lens in calls:
            graph.replay()
        torch.cuda.synchronize()
        kept = [[x.clone() for x in call[4]] for call in calls]
        for (c, q, fn, *_), got in zip(calls, kept):
            eager = fn()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, eager)), rep


@pytest.mark.gpu
def test_equals_the_paged_decode_and_the_forward(torch_gpu):
    """One token per sequence is the paged decode's work, a whole prompt the forward's: the same
    values within the roundings of both."""
    torch = torch_gpu
    c = PagedCase("bfloat16", 128, 32, 8, 16, lens=[700, 3, 64])
    q = torch.randn((3, 32, 128), device="cuda").bfloat16()
    o, lse = cuflash_attn.flash_attention_forward_paged(
        q, c.t_k, c.t_v, c.t_table, c.t_lens, c.ints([0, 1, 2, 3]), causal=True)
    o2, lse2 = cuflash_attn.flash_attention_decode_paged(q.unsqueeze(2), c.t_k, c.t_v, c.t_table,
                                                         c.t_lens)
    # Each rounds P and its output by half a step: |v| <= 6 bounds what P's rounding moves.
    assert float((o.float() - o2.squeeze(2).float()).abs().max()) <= 2 * 2 * 2.0 ** -8 * 6
    assert float((lse - lse2.squeeze(2)).abs().max()) <= 1e-4
