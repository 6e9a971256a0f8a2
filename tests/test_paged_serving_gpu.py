"""The paged-cache operators as a server runs them: prompts appended and attended to, then decode steps,
one model's layer after another on one cache, against float64 attention over the whole sequences; and the
calls around them: workspaces, streams, caches past 32-bit offsets."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest

import cuflash_attn
from cuflash_attn import synth
from paged_reference import HALF_STEP, PagedCase, attention, attention_bounds, rotate


class Server:
    """Sequences behind a shared prompt of `prefix` tokens on one cache, and what float64 makes of them:
    the rotated keys as the cache must hold them are rounded once, like the operator's."""

    def __init__(self, dtype, d, heads, kv_heads, page, batch, prefix, seed=3):
        import torch

        self.torch, self.dtype, self.d, self.page = torch, dtype, d, page
        self.heads, self.kv_heads, self.batch, self.prefix = heads, kv_heads, batch, prefix
        self.rng = np.random.default_rng(seed)
        self.seed = seed
        pages = 4 + batch * 12 + -(-prefix // page)
        t_dtype = getattr(torch, dtype)
        self.k, self.v = (torch.full((pages, page, kv_heads, d), float("nan"), device="cuda",
                                     dtype=t_dtype) for _ in range(2))
        self.free = list(self.rng.permutation(pages))
        half = d // 2
        angle = np.arange(prefix + 400)[:, None] * 1e4 ** (-np.arange(half) / half)
        self.cos, self.sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
        self.t_cos, self.t_sin = (torch.from_numpy(x).cuda() for x in (self.cos, self.sin))
        self.first = prefix // page
        self.prefix_pages = [self.free.pop() for _ in range(-(-prefix // page))]
        self.tables = [[] for _ in range(batch)]  # own pages, from entry `first` on
        self.lens = [0] * batch
        self.tokens = [[] for _ in range(batch)]  # projections of every token, [heads + 2 kv, d]
        self.shared = []

    def ints(self, x):
        return self.torch.tensor(x, dtype=self.torch.int32, device="cuda")

    def project(self, n):
        self.seed += 1
        return synth.round_to(synth.normal(self.seed, (n, self.heads + 2 * self.kv_heads, self.d)),
                              self.dtype)

    def run_tokens(self, rows, table, lens, starts):
        """Appends packed tokens; the rotated queries."""
        x = synth.to_torch(rows, self.dtype)
        H, K = self.heads, self.kv_heads
        return cuflash_attn.flash_attention_append_paged(
            x[:, H:H + K], x[:, H + K:], self.k, self.v, table, lens, starts, q=x[:, :H],
            cos=self.t_cos, sin=self.t_sin)

    def want(self, tokens, queries):
        """O, L and bounds of the last `queries` tokens of a sequence, [queries, heads, d]."""
        rows = np.stack(tokens)
        n, H, K = len(tokens), self.heads, self.kv_heads
        turned, size = rotate(rows[:, :H + K], np.arange(n), self.cos, self.sin, False)
        q = synth.round_to(turned[:, :H].astype(np.float32), self.dtype).astype(np.float64)
        k = synth.round_to(turned[:, H:].astype(np.float32), self.dtype).astype(np.float64)
        v = rows[:, H + K:]
        # The cache's and the queries' last bit may differ from these roundings: a score moves by up to
        # one step (two halves) of either operand.
        wobble = 2 * 2 * HALF_STEP[self.dtype] * self.d ** -0.5
        group = H // K
        out = []
        for h in range(K):
            x = q[n - queries:, h * group:(h + 1) * group].reshape(-1, self.d)
            limits = np.repeat(np.arange(n - queries, n) + 1, group)
            o, lse, mag, top, prod = attention(x, k[:, h], v[:, h], self.d ** -0.5, limits)
            shift = wobble * (abs(x) @ abs(k[:, h]).T).max(1)
            o_b, l_b = attention_bounds(self.dtype, self.d, n, o, lse, mag, top, prod,
                                        abs(v[:, h]).sum(0))
            out.append((o, lse, o_b + 2 * np.expm1(2 * shift)[:, None] * mag, l_b + shift))
        return out

    def check(self, tokens, queries, o, lse, where):
        group = self.heads // self.kv_heads
        for h, (wo, wl, ob, lb) in enumerate(self.want(tokens, queries)):
            at = slice(h * group, (h + 1) * group)
            assert (abs(o[:, at].reshape(-1, self.d) - wo) <= ob).all(), (where, h)
            assert (abs(lse[:, at].reshape(-1) - wl) <= lb).all(), (where, h, "L")

    def prefill_shared(self):
        rows = self.project(self.prefix)
        self.shared = list(rows)
        table = self.ints([self.prefix_pages])
        lens, starts = self.ints([self.prefix]), self.ints([0, self.prefix])
        q = self.run_tokens(rows, table, lens, starts)
        o, lse = cuflash_attn.flash_attention_forward_paged(q, self.k, self.v, table, lens, starts,
                                                            causal=True)
        self.check(self.shared, self.prefix, synth.to_numpy(o), synth.to_numpy(lse), "prompt")

    def table(self):
        width = self.first + max(1, max(len(t) for t in self.tables))
        out = np.zeros((self.batch, width), dtype=np.int64)
        for b, own in enumerate(self.tables):
            out[b, :self.first] = self.prefix_pages[:self.first]
            out[b, self.first:self.first + len(own)] = own
        return self.ints(out.tolist())

    def grow(self, new):
        """new[b] more tokens of sequence b: pages, projections, lengths."""
        rows = []
        for b, n in enumerate(new):
            if self.lens[b] == 0 and n:
                self.lens[b] = self.prefix
                self.tokens[b] = list(self.shared)
                if self.prefix % self.page:  # a copy of the page that the prompt ends in
                    page = self.free.pop()
                    self.tables[b].append(page)
                    self.k[page] = self.k[self.prefix_pages[-1]]
                    self.v[page] = self.v[self.prefix_pages[-1]]
            x = self.project(n) if n else np.zeros((0, self.heads + 2 * self.kv_heads, self.d),
                                                   np.float32)
            self.tokens[b] += list(x)
            rows.append(x)
            self.lens[b] += n
            while len(self.tables[b]) + self.first < -(-self.lens[b] // self.page):
                self.tables[b].append(self.free.pop())
        starts = np.concatenate([[0], np.cumsum(new)]).tolist()
        return np.concatenate(rows), self.table(), self.ints(self.lens), self.ints(starts)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,d,heads,kv_heads,page,prefix", [
    ("bfloat16", 128, 8, 2, 16, 100), ("float16", 64, 8, 8, 16, 64), ("float32", 64, 6, 2, 24, 50),
    ("bfloat16", 32, 16, 1, 32, 33)])
def test_prompt_turns_and_decode(torch_gpu, dtype, d, heads, kv_heads, page, prefix):
    s = Server(dtype, d, heads, kv_heads, page, batch=4, prefix=prefix)
    s.prefill_shared()
    # The sequences' own prompts, one of them only now and then.
    for new in ([9, 40, 1, 0], [2, 0, 33, 70]):
        rows, table, lens, starts = s.grow(new)
        q = s.run_tokens(rows, table, lens, starts)
        o, lse = cuflash_attn.flash_attention_forward_paged(q, s.k, s.v, table, lens, starts,
                                                            causal=True)
        o, lse = synth.to_numpy(o), synth.to_numpy(lse)
        at = 0
        for b, n in enumerate(new):
            if n:
                s.check(s.tokens[b], n, o[at:at + n], lse[at:at + n], f"turn {new} of {b}")
            at += n
    # Decode steps: over each sequence's own table, and with the prompt read once.
    prefix_table = s.ints(s.prefix_pages)
    for step in range(3):
        rows, table, lens, _ = s.grow([1, 1, 1, 1])
        q = s.run_tokens(rows, table, lens, None).unsqueeze(2)
        got = cuflash_attn.flash_attention_decode_shared(q, s.k, s.v, prefix_table, prefix, table,
                                                         lens)
        o, lse = (synth.to_numpy(x) for x in got)
        for b in range(4):
            s.check(s.tokens[b], 1, o[b:b + 1, :, 0], lse[b:b + 1, :, 0], f"step {step} of {b}")
        plain = cuflash_attn.flash_attention_decode_paged(q, s.k, s.v, table, lens)
        for a, b_ in zip(got, plain):
            assert float((a.float() - b_.float()).abs().max()) <= 8 * HALF_STEP[dtype] * 6


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_callers_workspace(torch_gpu, lib, dtype):
    """A given workspace gives what the library's own does; too small a one is refused."""
    torch = torch_gpu
    sfx = cuflash_attn._DTYPE_SUFFIX[dtype]
    c = PagedCase(dtype, 64, 8, 2, 16, prefix=200, lens=[900, 2100, 230])
    q = torch.randn((3, 8, 1, 64), device="cuda").to(c.t_k.dtype)
    starts = c.ints([0, 1, 2, 3])
    need = lib.fn("decode_shared_workspace", sfx)(3, 8, 2, 64)
    need_fwd = lib.fn("forward_paged_workspace", sfx)(3, 3, 8, 2, 64)
    assert need > 0 and need_fwd > 0
    ws = torch.full((max(need, need_fwd),), 255, dtype=torch.uint8, device="cuda")
    o, lse = torch.empty_like(q), torch.empty((3, 8, 1), device="cuda")
    stream = torch.cuda.current_stream().cuda_stream

    def shared(ptr, size):
        return lib.fn("decode_shared", sfx)(
            q.data_ptr(), c.t_k.data_ptr(), c.t_v.data_ptr(), o.data_ptr(), lse.data_ptr(),
            c.t_prefix.data_ptr(), c.t_table.data_ptr(), c.t_lens.data_ptr(), 3, 8, 2, 200, 16,
            c.max_pages, 64, 0.125, ptr, size, stream)

    def forward(ptr, size):
        return lib.fn("forward_paged", sfx)(
            q.data_ptr(), c.t_k.data_ptr(), c.t_v.data_ptr(), o.data_ptr(), lse.data_ptr(),
            c.t_table.data_ptr(), c.t_lens.data_ptr(), starts.data_ptr(), 3, 3, 8, 2, 16,
            c.max_pages, 64, 0.125, True, ptr, size, stream)

    # The forward reads whole sequences from the block table: put the prefix there as well.
    c.t_table[:, :200 // 16] = c.t_prefix[:200 // 16]
    page = 200 // 16
    for b in range(3):
        own = int(c.t_table[b, page])
        c.t_k[own, :200 % 16] = c.t_k[int(c.t_prefix[page]), :200 % 16]
        c.t_v[own, :200 % 16] = c.t_v[int(c.t_prefix[page]), :200 % 16]
    want = None
    for call, size in ((shared, need), (forward, need_fwd)):
        results = []
        for ptr, given in ((None, 0), (ws.data_ptr(), size)):
            o.fill_(7.0)
            assert call(ptr, given) == 0
            torch.cuda.synchronize()
            results.append((o.clone(), lse.clone()))
        assert all(torch.equal(a, b) for a, b in zip(*results))
        assert call(ws.data_ptr(), 256) == cuflash_attn.OUT_OF_MEMORY
        assert call(ws.data_ptr() + 16, size) == cuflash_attn.INVALID_DIMENSION
        if want is not None:
            assert float((want.float() - results[0][0].float()).abs().max()) <= \
                8 * HALF_STEP[dtype] * 6
        want = results[0][0]


@pytest.mark.gpu
def test_captured_without_a_workspace(torch_gpu, lib):
    """Through the C ABI: the forward runs in one chunk, the shared decode is refused, and the capture
    goes on."""
    torch = torch_gpu
    c = PagedCase("bfloat16", 128, 8, 2, 16, prefix=64, lens=[2000, 100])
    q = torch.randn((2, 8, 128), device="cuda").bfloat16()
    o, lse = torch.zeros_like(q), torch.zeros((2, 8), device="cuda")
    starts = c.ints([0, 1, 2])
    c.t_table[:, :4] = c.t_prefix
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        stream = torch.cuda.current_stream().cuda_stream
        status = lib.fn("decode_shared", "bf16")(
            q.data_ptr(), c.t_k.data_ptr(), c.t_v.data_ptr(), o.data_ptr(), lse.data_ptr(),
            c.t_prefix.data_ptr(), c.t_table.data_ptr(), c.t_lens.data_ptr(), 2, 8, 2, 64, 16,
            c.max_pages, 128, 0.1, None, 0, stream)
        assert status == cuflash_attn.OUT_OF_MEMORY
        status = lib.fn("forward_paged", "bf16")(
            q.data_ptr(), c.t_k.data_ptr(), c.t_v.data_ptr(), o.data_ptr(), lse.data_ptr(),
            c.t_table.data_ptr(), c.t_lens.data_ptr(), starts.data_ptr(), 2, 2, 8, 2, 16,
            c.max_pages, 128, 128 ** -0.5, True, None, 0, stream)
        assert status == 0
    for rep in range(3):
        print(f"[captured without workspace] replay {rep}", flush=True)
        q.normal_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = o.clone(), lse.clone()
        c.check(synth.to_numpy(q), [1, 1], True, synth.to_numpy(got[0]), synth.to_numpy(got[1]))


@pytest.mark.gpu
def test_two_streams_at_once(torch_gpu):
    """Calls on two streams share nothing."""
    torch = torch_gpu
    cases, streams, got, want = [], [], [], []
    for seed in (1, 2):
        c = PagedCase("float16", 64, 16, 4, 16, prefix=500, lens=[3000 + 7 * seed, 600, 501, 900],
                      seed=seed)
        q = torch.randn((4, 16, 1, 64), device="cuda").half()
        cases.append((c, q))
        streams.append(torch.cuda.Stream())

    def call(c, q, stream=None):
        return cuflash_attn.flash_attention_decode_shared(q, c.t_k, c.t_v, c.t_prefix, 500,
                                                          c.t_table, c.t_lens, stream=stream)

    want = [call(*x) for x in cases]
    torch.cuda.synchronize()
    for _ in range(20):
        got.append([call(*x, stream=s) for x, s in zip(cases, streams)])
    torch.cuda.synchronize()
    for pair in got:
        for (o, lse), (wo, wl) in zip(pair, want):
            assert torch.equal(o, wo) and torch.equal(lse, wl)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [2, 90])
def test_cache_past_32_bit_offsets(torch_gpu, tokens):
    """Pages more than 2^32 elements into the cache: append, forward (few and many rows) and shared
    decode read and write there what they do at its start."""
    torch = torch_gpu
    page, kv_heads, d, heads = 64, 8, 128, 32
    pages = (1 << 32) // (page * kv_heads * d) + 16
    shape = (pages, page, kv_heads, d)
    k, v = (torch.empty(shape, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    n = 5 * page - 7
    x = torch.randn((n, 2, kv_heads, d), device="cuda").bfloat16()
    q = torch.randn((tokens, heads, d), device="cuda").bfloat16()
    ints = lambda y: torch.tensor(y, dtype=torch.int32, device="cuda")  # noqa: E731
    lens, results = ints([n]), []
    for first in (0, pages - 5):
        table = ints([list(range(first, first + 5))])
        cuflash_attn.flash_attention_append_paged(x[:, 0], x[:, 1], k, v, table, lens,
                                                  ints([0, n]))
        assert torch.equal(k[first:first + 5].reshape(-1, kv_heads, d)[:n], x[:, 0])
        assert torch.equal(v[first:first + 5].reshape(-1, kv_heads, d)[:n], x[:, 1])
        r = list(cuflash_attn.flash_attention_forward_paged(q, k, v, table, lens,
                                                            ints([0, tokens]), causal=True))
        b = min(tokens, 40)
        both = table.expand(b, 5).contiguous()
        r += cuflash_attn.flash_attention_decode_shared(
            q[:b].unsqueeze(2), k, v, table[0, :3].contiguous(), 3 * page, both,
            lens.expand(b).contiguous())
        results.append(r)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(*results))
    del k, v
    torch.cuda.empty_cache()


@pytest.mark.gpu
def test_captured_step(torch_gpu):
    """A server's captured step: append, then both attentions, replayed as the sequences grow. The graph's
    cache and the eager one stay the same bit for bit, and so do the outputs."""
    torch = torch_gpu
    c = PagedCase("bfloat16", 128, 16, 4, 16, prefix=200, lens=[230, 900, 205, 411], capacity=1024)
    c.t_table[:, :12] = c.t_prefix[:12]
    spare = torch.full((60,) + tuple(c.t_k.shape[1:]), float("nan"), device="cuda", dtype=c.t_k.dtype)
    caches = [[torch.cat([x, spare]) for x in (c.t_k, c.t_v)] for _ in range(2)]
    pages = c.t_k.shape[0]
    for b in range(4):  # rows to grow into, and each sequence's own copy of the page the prefix ends in
        have = -(-c.lens[b] // 16)
        c.t_table[b, have:have + 2] = torch.arange(pages + 10 * b, pages + 10 * b + 2)
        for k, v in caches:
            own, shared = int(c.t_table[b, 12]), int(c.t_prefix[12])
            k[own, :8], v[own, :8] = k[shared, :8], v[shared, :8]
    lens, starts = c.t_lens.clone(), c.ints([0, 1, 2, 3, 4])
    qkv = torch.randn((4, 24, 128), device="cuda").bfloat16()
    angle = torch.arange(1024, device="cuda")[:, None] * 1e4 ** (-torch.arange(64, device="cuda") / 64)
    cos, sin = angle.cos().contiguous(), angle.sin().contiguous()

    def step(k, v):
        q = cuflash_attn.flash_attention_append_paged(
            qkv[:, 16:20], qkv[:, 20:], k, v, c.t_table, lens, q=qkv[:, :16], cos=cos, sin=sin)
        return (q, *cuflash_attn.flash_attention_forward_paged(q, k, v, c.t_table, lens, starts,
                                                               causal=True),
                *cuflash_attn.flash_attention_decode_shared(q.unsqueeze(2), k, v, c.t_prefix, 200,
                                                            c.t_table, lens))

    graph = torch.cuda.CUDAGraph()
    lens += 1
    with torch.cuda.graph(graph):
        out = step(*caches[0])
    torch.cuda.synchronize()
    for rep in range(4):
        print(f"[captured step] replay {rep}", flush=True)
        qkv.normal_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in out]
        want = step(*caches[1])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), rep
        assert bool(torch.isfinite(got[1].float()).all() and torch.isfinite(got[3].float()).all())
        # One query per sequence: both attentions see the same keys.
        off = (got[1].float() - got[3][:, :, 0].float()).abs().max()
        assert float(off) <= 8 * HALF_STEP["bfloat16"] * 6
        for a, b in zip(*caches):
            assert torch.equal(a.view(torch.int16), b.view(torch.int16)), rep
        lens += 1
