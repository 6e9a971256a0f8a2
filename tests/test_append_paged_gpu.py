"""flash_attention_append_paged against float64 (paged_reference.py): rotated queries and keys
within their roundings, values and everything else in the caches bit for bit."""

from __future__ import annotations

import numpy as np
import pytest

import cuflash_attn
from cuflash_attn import synth
from paged_reference import positions, rotate, rotated_bound

DTYPES = ["float32", "float16", "bfloat16"]


def _tables(n, half):
    angle = np.arange(n)[:, None] * 1e4 ** (-np.arange(half) / half)
    return np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)


class Case:
    """One append on the GPU and its parts on the host."""

    def __init__(self, dtype, d, heads, kv_heads, page, new, old, rotary, interleaved=False,
                 extra=0, apart=0, seed=1, order=None):
        import torch

        self.dtype, self.d, self.heads, self.kv_heads, self.page = dtype, d, heads, kv_heads, page
        self.interleaved, self.rotary = interleaved, rotary
        B = len(new)
        self.lens = [n + o for n, o in zip(new, old)]
        self.starts = [sum(new[:b]) for b in range(B + 1)]
        T = self.starts[-1] + extra  # `extra` padding tokens
        width = (heads + 2 * kv_heads) * d + apart
        rows = synth.round_to(synth.normal(seed, (T, width)), dtype)
        self.rows = rows
        heads_of = lambda x, at, n: x[:, at * d:(at + n) * d].reshape(T, n, d)  # noqa: E731
        self.q, self.k, self.v = (heads_of(rows, at, n) for at, n in (
            (0, heads), (heads, kv_heads), (heads + kv_heads, kv_heads)))
        max_pages = max(1, max(-(-n // page) for n in self.lens))
        self.pages = B * max_pages + 2
        rng = np.random.default_rng(seed)
        self.table = rng.permutation(self.pages)[:B * max_pages].reshape(B, max_pages)
        shape = (self.pages, page, kv_heads, d)
        self.k0, self.v0 = (synth.round_to(synth.normal(seed + s, shape), dtype) for s in (1, 2))
        self.cos, self.sin = _tables(max(1, max(self.lens)), rotary // 2) if rotary else (None,
                                                                                         None)
        self.t_rows = synth.to_torch(rows, dtype)
        self.tq, self.tk, self.tv = (
            self.t_rows[:, at * d:(at + n) * d].unflatten(1, (n, d)) for at, n in (
                (0, heads), (heads, kv_heads), (heads + kv_heads, kv_heads)))
        ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
        self.t_table, self.t_lens, self.t_starts = (
            ints(self.table.tolist()), ints(self.lens), ints(self.starts))
        self.t_cos, self.t_sin = ((None, None) if not rotary else
                                  (torch.from_numpy(x).cuda() for x in (self.cos, self.sin)))
        self.reset()

    def reset(self):
        self.k_cache, self.v_cache = (synth.to_torch(x, self.dtype) for x in (self.k0, self.v0))

    def run(self, **kw):
        args = dict(q=self.tq, cos=self.t_cos, sin=self.t_sin, interleaved=self.interleaved,
                    query_starts=self.t_starts)
        args.update(kw)
        return cuflash_attn.flash_attention_append_paged(
            self.tk, self.tv, self.k_cache, self.v_cache, self.t_table, self.t_lens, **args)

    def check(self, got_q, skip=(), nan=()):
        """Compares caches and queries; tokens of `skip` are not in the cache, those of `nan` have
        NaN queries (and are not in the cache)."""
        k_want, v_want = self.k0.astype(np.float64), self.v0.astype(np.float64)
        k_bound = np.zeros_like(k_want)
        places = positions(self.lens, self.starts)
        T = self.starts[-1]
        pos = np.zeros(T, dtype=np.int64)
        for t, _, p in places:
            pos[t] = p if t not in nan else 0

        def turned(x):
            y, size = x[:T].astype(np.float64), np.zeros(x[:T].shape)
            if self.rotary:
                y, size = rotate(x[:T], pos, self.cos, self.sin, self.interleaved)
            bound = rotated_bound(self.dtype, y, size)
            bound[..., self.rotary:] = 0.0
            return y, bound if self.rotary else np.zeros_like(bound)

        q_want, q_bound = turned(self.q)
        k_rows, k_rows_bound = turned(self.k)
        for t, b, p in places:
            if t in skip or t in nan:
                continue
            page, row = self.table[b, p // self.page], p % self.page
            k_want[page, row], k_bound[page, row] = k_rows[t], k_rows_bound[t]
            v_want[page, row] = self.v[t]
        k_got, v_got = synth.to_numpy(self.k_cache), synth.to_numpy(self.v_cache)
        assert np.array_equal(v_got, v_want.astype(np.float32))
        assert (abs(k_got - k_want) <= k_bound).all(), abs(k_got - k_want).max()
        if got_q is None:
            return
        q_got = synth.to_numpy(got_q)[:T]
        keep = [t for t in range(T) if t not in nan]
        assert (abs(q_got - q_want) <= q_bound)[keep].all(), abs(q_got - q_want)[keep].max()
        for t in nan:
            assert np.isnan(q_got[t, :, :self.rotary]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,rotary", [(32, 32), (32, 16), (64, 64), (64, 48), (128, 128),
                                      (128, 32), (64, 0)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("heads,kv_heads", [(8, 2), (3, 1), (4, 4)])
def test_append(torch_gpu, dtype, d, rotary, interleaved, heads, kv_heads):
    """New tokens across page borders, none and one of them, sequences that begin."""
    c = Case(dtype, d, heads, kv_heads, 16, new=[5, 0, 1, 40, 17], old=[0, 9, 15, 3, 31],
             rotary=rotary, interleaved=interleaved)
    c.check(c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [1, 6, 24, 128])
@pytest.mark.parametrize("batch", [1, 63, 64, 65, 150])
def test_one_token_per_sequence(torch_gpu, dtype, page, batch):
    """With and without query_starts: the same rows, more sequences than lanes of a wave."""
    c = Case(dtype, 64, 4, 2, page, new=[1] * batch, old=[(7 * b) % 301 for b in range(batch)],
             rotary=64)
    first = c.run()
    c.check(first)
    caches = c.k_cache.clone(), c.v_cache.clone()
    c.reset()
    second = c.run(query_starts=None)
    assert torch_gpu.equal(first, second)
    assert torch_gpu.equal(caches[0], c.k_cache) and torch_gpu.equal(caches[1], c.v_cache)


@pytest.mark.gpu
def test_many_sequences_some_without_tokens(torch_gpu):
    new = [(b * 5) % 4 for b in range(200)]
    c = Case("bfloat16", 32, 2, 1, 16, new=new, old=[b % 37 for b in range(200)], rotary=32)
    c.check(c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_tokens_apart_in_place_and_without_queries(torch_gpu, dtype):
    """Rows apart by more than their heads; queries rotated in their own place; keys alone."""
    c = Case(dtype, 64, 4, 2, 16, new=[9, 30], old=[20, 0], rotary=64, apart=64)
    got = c.run()
    c.check(got)
    kept = (c.k_cache.clone(), c.v_cache.clone())
    c.reset()
    packed = c.tq.contiguous()
    assert c.run(q=packed, out=packed) is packed
    assert torch_gpu.equal(packed, got) and torch_gpu.equal(kept[0], c.k_cache)
    c.reset()
    assert c.run(q=None) is None
    assert torch_gpu.equal(kept[0], c.k_cache) and torch_gpu.equal(kept[1], c.v_cache)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_padding_tokens_are_left_alone(torch_gpu, dtype):
    c = Case(dtype, 64, 4, 2, 16, new=[3, 4], old=[20, 0], rotary=64, extra=6)
    out = torch_gpu.full((13, 4, 64), 7.0, device="cuda", dtype=c.tq.dtype)
    got = c.run(out=out)
    c.check(got)
    assert bool((got[7:] == 7.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("rotary", [64, 0])
def test_tokens_that_have_no_row(torch_gpu, rotary):
    """Pages that the cache does not have, positions below zero, past the block table and past the
    rotation's tables: not written; queries only need a row of the tables."""
    c = Case("float16", 64, 4, 2, 16, new=[4, 4, 6, 2], old=[14, 60, 0, 3], rotary=rotary)
    table = c.t_table.clone()
    table[0, 1] = -1         # positions 16, 17 of sequence 0: tokens 2, 3
    table[3, 0] = c.pages    # sequence 3: tokens 14, 15
    c.t_table = table
    c.t_lens[2] = 4          # sequence 2 has 6 new tokens of 4: tokens 8, 9 stand before it
    c.lens[2] = 4
    narrow = c.t_table[:, :4].contiguous()  # 64 positions: sequence 1's 60 .. 63 still fit
    c.t_table = narrow
    got = c.run()
    c.check(got, skip=(2, 3, 14, 15) + (() if rotary else (8, 9)), nan=(8, 9) if rotary else ())
    # One page less: sequence 1's positions 60 .. 63 are past the table.
    c.reset()
    c.t_table = c.t_table[:, :3].contiguous()
    got = c.run()
    c.check(got, skip=(2, 3, 14, 15, 4, 5, 6, 7) + (() if rotary else (8, 9)),
            nan=(8, 9) if rotary else ())
    if rotary:
        # Tables of 62 positions: tokens 6 and 7 (positions 62, 63) are past them.
        c.reset()
        c.t_table = narrow
        got = c.run(cos=c.t_cos[:62].contiguous(), sin=c.t_sin[:62].contiguous())
        c.check(got, skip=(2, 3, 14, 15), nan=(8, 9, 6, 7))


@pytest.mark.gpu
def test_non_finite_values_pass(torch_gpu):
    """NaN and infinities of values arrive; a rotated infinity is what the formula makes of it."""
    c = Case("bfloat16", 64, 2, 1, 16, new=[3], old=[0], rotary=64)
    c.t_rows[1, -64:] = float("inf")
    c.t_rows[2, -64] = float("nan")
    c.run()
    torch_gpu.cuda.synchronize()
    v = synth.to_numpy(c.v_cache)[c.table[0, 0]]
    assert np.isinf(v[1]).all() and np.isnan(v[2, 0, 0]) and np.isfinite(v[2, 0, 1:]).all()


@pytest.mark.gpu
def test_captured_and_on_another_stream(torch_gpu):
    """A captured append replayed on new tokens and lengths, and one on a side stream."""
    torch = torch_gpu
    c = Case("bfloat16", 128, 8, 2, 16, new=[1] * 5, old=[3, 15, 16, 40, 0], rotary=128)
    out = torch.empty((5, 8, 128), device="cuda", dtype=torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = c.run(stream=side)
    side.synchronize()
    c.check(got)
    c.reset()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.run(out=out, query_starts=None)
    torch.cuda.synchronize()
    for rep in range(3):
        print(f"[append graph] replay {rep}", flush=True)
        c.t_rows.copy_(torch.randn_like(c.t_rows))
        c.t_lens.copy_(torch.tensor([4 - rep, 16 - rep, 17, 41 - rep, 1], device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        kept = [x.clone() for x in (out, c.k_cache, c.v_cache)]
        eager = c.run(query_starts=None)
        torch.cuda.synchronize()
        for a, b in zip(kept, (eager, c.k_cache, c.v_cache)):
            assert torch.equal(a, b), rep
