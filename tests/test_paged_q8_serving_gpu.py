"""The operators on an 8-bit paged cache as a server runs them, one after the other, captured, on several
streams and with workspaces of the caller."""

from __future__ import annotations

import numpy as np
import pytest

import cuflash_attn
from cuflash_attn import synth
from paged_q8_reference import Q8Case, quantise, rotate32, torch_cache, values
from paged_reference import attention, attention_bounds


class Server:
    """Sequences that grow in one cache, and what it should hold."""

    def __init__(self, torch, dtype, code, d, heads, kv_heads, page, batch, most, seed=3):
        self.torch, self.dtype, self.code, self.d = torch, dtype, code, d
        self.heads, self.kv_heads, self.page, self.batch = heads, kv_heads, page, batch
        max_pages = -(-most // page)
        rng = np.random.default_rng(seed)
        self.table = rng.permutation(batch * max_pages).reshape(batch, max_pages)
        shape = (batch * max_pages, page, kv_heads, d)
        # NaN until a token is written.
        self.k, self.v = (torch_cache(np.full(shape, 0x7F, np.uint8), code) for _ in range(2))
        self.kx, self.vx = (torch.full((shape[0], kv_heads, page), 255, dtype=torch.uint8, device="cuda")
                            for _ in range(2))
        self.cache = (self.k, self.v, self.kx, self.vx)
        angle = np.arange(most)[:, None] * 1e4 ** (-np.arange(d // 2) / (d // 2))
        self.cos, self.sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
        self.t_cos, self.t_sin = (torch.from_numpy(x).cuda() for x in (self.cos, self.sin))
        self.t_table = self.ints(self.table)
        self.lens = [0] * batch
        self.keys, self.vals = ([np.zeros((0, kv_heads, d)) for _ in range(batch)] for _ in range(2))
        self.seed = seed

    def ints(self, x):
        return self.torch.tensor(np.asarray(x).tolist(), dtype=self.torch.int32, device="cuda")

    def tokens(self, new):
        """Rows of new tokens, their queries as the append should rotate them; the sequences grow."""
        T = sum(new)
        self.seed += 1
        H, Hkv, D = self.heads, self.kv_heads, self.d
        rows = synth.round_to(synth.normal(self.seed, (T, H + 2 * Hkv, D)), self.dtype)
        pos = np.concatenate([np.arange(n, n + m) for n, m in zip(self.lens, new)]).astype(int)
        q = synth.round_to(rotate32(rows[:, :H], pos, self.cos, self.sin, False), self.dtype)
        k = values(*quantise(rotate32(rows[:, H:H + Hkv], pos, self.cos, self.sin, False), self.code,
                             self.dtype), self.code)
        v = values(*quantise(rows[:, H + Hkv:], self.code, self.dtype), self.code)
        t0 = 0
        for b, m in enumerate(new):
            self.keys[b] = np.concatenate((self.keys[b], k[t0:t0 + m]))
            self.vals[b] = np.concatenate((self.vals[b], v[t0:t0 + m]))
            self.lens[b] += m
            t0 += m
        starts = [sum(new[:b]) for b in range(self.batch + 1)]
        return synth.to_torch(rows, self.dtype), q, self.ints(self.lens), self.ints(starts)

    def append(self, rows, lens, starts, **kw):
        H, Hkv = self.heads, self.kv_heads
        return cuflash_attn.flash_attention_append_paged_q8(
            rows[:, H:H + Hkv], rows[:, H + Hkv:], *self.cache, self.t_table, lens, starts,
            q=rows[:, :H], cos=self.t_cos, sin=self.t_sin, **kw)

    def check(self, q, new, o, lse, where):
        o, lse, t0 = synth.to_numpy(o), synth.to_numpy(lse), 0
        o, lse = o.reshape(len(q), self.heads, self.d), lse.reshape(len(q), self.heads)
        group = self.heads // self.kv_heads
        times = 3 if self.dtype == "float32" else 1
        for b, n in enumerate(new):
            keys, vals = self.keys[b], self.vals[b]
            limits = np.repeat([len(keys) - n + i + 1 for i in range(n)], group)
            for h in range(self.kv_heads if n else 0):
                at = (slice(t0, t0 + n), slice(h * group, (h + 1) * group))
                want = attention(q[at].reshape(n * group, -1), keys[:, h], vals[:, h], self.d ** -0.5,
                                 limits)
                o_bound, l_bound = attention_bounds(self.dtype, times * self.d, times * len(keys),
                                                    *want, abs(vals[:, h]).sum(0))
                assert (abs(o[at].reshape(n * group, -1) - want[0]) <= o_bound).all(), (where, b, h)
                assert (abs(lse[at].reshape(-1) - want[1]) <= l_bound).all(), (where, b, h)
            t0 += n


@pytest.mark.gpu
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_conversations(torch_gpu, lib, dtype, code):
    """Prompts, next turns and decode steps; then everything is read back, and attention over the numbers
    read, in a 16-bit cache, gives the same."""
    torch = torch_gpu
    s = Server(torch, dtype, code, 64, 8, 2, 16, batch=4, most=1300)
    for new in ([700, 33, 1, 120], [5, 0, 60, 3], [1, 1, 1, 1], [1, 1, 1, 1]):
        rows, q, lens, starts = s.tokens(new)
        turned = s.append(rows, lens, starts)
        assert np.array_equal(synth.to_numpy(turned), q)
        if max(new) > 1:
            got = cuflash_attn.flash_attention_forward_paged_q8(turned, *s.cache, s.t_table, lens,
                                                                starts, causal=True)
        else:
            got = cuflash_attn.flash_attention_decode_paged_q8(turned.unsqueeze(2), *s.cache,
                                                               s.t_table, lens)
        s.check(q, new, *got, new)
    T = sum(s.lens)
    starts_all = s.ints([sum(s.lens[:b]) for b in range(5)])
    k, v = cuflash_attn.flash_attention_read_paged_q8(*s.cache, s.t_table, lens, starts_all, T,
                                                      dtype=turned.dtype)
    for got, want in ((k, s.keys), (v, s.vals)):
        assert np.array_equal(synth.to_numpy(got), np.concatenate(want).astype(np.float32))
    cache = [torch.zeros(s.k.shape, dtype=turned.dtype, device="cuda") for _ in range(2)]
    cuflash_attn.flash_attention_append_paged(k, v, *cache, s.t_table, lens, starts_all)
    want = cuflash_attn.flash_attention_decode_paged(turned.unsqueeze(2), *cache, s.t_table, lens)
    half = {"float32": 2.0 ** -18, "float16": 2.0 ** -9, "bfloat16": 2.0 ** -6}[dtype]
    assert float((got_o := cuflash_attn.flash_attention_decode_paged_q8(
        turned.unsqueeze(2), *s.cache, s.t_table, lens)[0].float() - want[0].float()).abs().max()) \
        <= half * float(want[0].float().abs().max()), got_o


@pytest.mark.gpu
@pytest.mark.parametrize("most", [1000, 3000])  # decodes in one launch and in two
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_captured_steps_follow_the_sequences(torch_gpu, lib, dtype, most):
    """Append, decode, forward and read in a graph, replayed as the sequences grow: the bits of the same
    calls made eagerly, before and after which other work runs."""
    torch = torch_gpu
    s = Server(torch, dtype, "e4m3", 128, 8, 2, 16, batch=3, most=most)
    rows, q, lens, starts = s.tokens([400, 31, 600])
    s.append(rows, lens, starts)
    ones = s.ints([0, 1, 2, 3])
    t_rows, t_lens = torch.zeros((3, 12, 128), device="cuda").to(rows.dtype), lens.clone()

    def step():
        turned = s.append(t_rows, t_lens, ones)
        return [turned,
                *cuflash_attn.flash_attention_decode_paged_q8(turned.unsqueeze(2), *s.cache, s.t_table,
                                                              t_lens),
                *cuflash_attn.flash_attention_forward_paged_q8(turned, *s.cache, s.t_table, t_lens,
                                                               ones, causal=True),
                *cuflash_attn.flash_attention_read_paged_q8(*s.cache, s.t_table, t_lens, ones, 3,
                                                            dtype=rows.dtype)]

    step()
    for x in (*s.keys, *s.vals):  # the rows of zeros that this wrote in the newest tokens' place
        x[-1] = 0.0
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for rep in range(3):
        rows, q, lens, _ = s.tokens([1, 1, 1])
        t_rows.copy_(rows)
        t_lens.copy_(lens)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in out]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), rep
        s.check(q, [1, 1, 1], got[1], got[2], rep)
        s.check(q, [1, 1, 1], got[3], got[4], rep)


@pytest.mark.gpu
def test_two_graphs_in_a_row(torch_gpu, lib):
    """Two captured attentions with workspaces of their own, replayed in turn without a wait between."""
    torch = torch_gpu
    cases = [Q8Case("bfloat16", "int8", 128, 8, 2, 16, [3000, 40, 1200], seed=i) for i in (1, 5)]
    q = torch.randn((3, 8, 1, 128), device="cuda").bfloat16()

    def call(c):
        return cuflash_attn.flash_attention_decode_paged_q8(q, *c.cache, c.t_table, c.t_lens)

    want = [call(c) for c in cases]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(c))
        graphs.append(g)
    for rep in range(3):
        for o, lse in outs:
            o.fill_(7.0)
        for g in graphs + graphs:
            g.replay()
        torch.cuda.synchronize()
        for got, w in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(got, w)), rep


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("new", [1, 3, 200])
def test_callers_workspace(torch_gpu, lib, dtype, new):
    """A given workspace gives what the library's own does; too small a one is refused, and so is a capture
    without one, which goes on."""
    torch = torch_gpu
    sfx = cuflash_attn._DTYPE_SUFFIX[dtype]
    c = Q8Case(dtype, "int8", 64, 8, 2, 16, [1900, 2100, 230])
    T = 3 * new
    q = torch.randn((T, 8, 64), device="cuda").to(getattr(torch, dtype))
    o, lse = torch.empty_like(q), torch.empty((T, 8), device="cuda")
    starts = c.ints([0, new, 2 * new, T])
    cache = [t.data_ptr() for t in c.cache]

    def call(ptr, size):
        stream = torch.cuda.current_stream().cuda_stream
        if new == 1:
            return lib.fn("decode_paged_q8", sfx)(
                q.data_ptr(), *cache, o.data_ptr(), lse.data_ptr(), c.t_table.data_ptr(),
                c.t_lens.data_ptr(), 3, 8, 2, 16, c.max_pages, 64, 0.125, 0, ptr, size, stream)
        return lib.fn("forward_paged_q8", sfx)(
            q.data_ptr(), *cache, o.data_ptr(), lse.data_ptr(), c.t_table.data_ptr(),
            c.t_lens.data_ptr(), starts.data_ptr(), T, 3, 8, 2, 16, c.max_pages, 64, 0.125, True, 0,
            ptr, size, stream)

    need = lib.fn("decode_paged_q8_workspace", sfx)(3, 8, 2, 64) if new == 1 else \
        lib.fn("forward_paged_q8_workspace", sfx)(T, 3, 8, 2, 64)
    assert need > 0
    guard = 4096
    ws = torch.full((need + guard,), 255, dtype=torch.uint8, device="cuda")
    results = []
    for ptr, size in ((None, 0), (ws.data_ptr(), need)):
        o.fill_(7.0)
        assert call(ptr, size) == 0
        torch.cuda.synchronize()
        results.append((o.clone(), lse.clone()))
    assert all(torch.equal(a, b) for a, b in zip(*results))
    assert bool((ws[need:] == 255).all())
    assert call(ws.data_ptr(), need - 1) == cuflash_attn.OUT_OF_MEMORY
    assert call(ws.data_ptr() + 16, need) == cuflash_attn.INVALID_DIMENSION
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        assert call(None, 0) == cuflash_attn.OUT_OF_MEMORY
        assert call(ws.data_ptr(), need) == 0
    for rep in range(3):
        o.fill_(7.0)
        ws.fill_(255)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, results[0][0]) and torch.equal(lse, results[0][1]), rep


@pytest.mark.gpu
def test_streams(torch_gpu, lib):
    """Calls on two streams at once, one of them given by argument while another is current."""
    torch = torch_gpu
    c = Q8Case("bfloat16", "e4m3", 128, 8, 2, 16, [4000, 900, 2500])
    starts = c.ints([0, 150, 300, 450])
    q = torch.randn((450, 8, 128), device="cuda").bfloat16()
    one = torch.randn((3, 8, 1, 128), device="cuda").bfloat16()
    want = (cuflash_attn.flash_attention_forward_paged_q8(q, *c.cache, c.t_table, c.t_lens, starts,
                                                          causal=True),
            cuflash_attn.flash_attention_decode_paged_q8(one, *c.cache, c.t_table, c.t_lens))
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(4):
        with torch.cuda.stream(a):
            got.append((0, cuflash_attn.flash_attention_forward_paged_q8(
                q, *c.cache, c.t_table, c.t_lens, starts, causal=True)))
            got.append((1, cuflash_attn.flash_attention_decode_paged_q8(
                one, *c.cache, c.t_table, c.t_lens, stream=b)))
    torch.cuda.synchronize()
    for which, g in got:
        assert all(torch.equal(x, y) for x, y in zip(g, want[which]))


@pytest.mark.gpu
def test_rotation_in_place(torch_gpu, lib):
    """Packed queries may be rotated where they are."""
    torch = torch_gpu
    s = Server(torch, "bfloat16", "int8", 64, 8, 2, 16, batch=2, most=100)
    rows, q, lens, starts = s.tokens([40, 7])
    H, Hkv = 8, 2
    packed = rows[:, :H].contiguous()
    out = cuflash_attn.flash_attention_append_paged_q8(
        rows[:, H:H + Hkv], rows[:, H + Hkv:], *s.cache, s.t_table, lens, starts, q=packed,
        cos=s.t_cos, sin=s.t_sin, out=packed)
    assert out is packed and np.array_equal(synth.to_numpy(out), q)
