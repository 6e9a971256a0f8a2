"""The paged-cache operators in plain numpy, in float64: what the GPU tests compare with."""

from __future__ import annotations

import numpy as np

# Half a step of the type relative to the value, and the smallest half step.
HALF_STEP = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
TINY = {"float32": 2.0 ** -150, "float16": 2.0 ** -25, "bfloat16": 2.0 ** -134}


def rotate(x, pos, cos, sin, interleaved):
    """x [T, heads, D] rotated by rows pos of cos, sin [., R / 2], and the magnitudes |x1 cos| +
    |x2 sin| that the rounding of the products goes by (0 where nothing is rotated)."""
    y = x.astype(np.float64)
    size = np.zeros_like(y)
    half = cos.shape[1]
    one = np.arange(half) * (2 if interleaved else 1)
    two = one + (1 if interleaved else half)
    c, s = (t[pos].astype(np.float64)[:, None, :] for t in (cos, sin))
    a, b = y[..., one].copy(), y[..., two].copy()
    y[..., one], y[..., two] = a * c - b * s, b * c + a * s
    size[..., one], size[..., two] = abs(a * c) + abs(b * s), abs(b * c) + abs(a * s)
    return y, size


def positions(seq_lens, starts):
    """[(token, sequence, position)] of the packed tokens."""
    out = []
    for b, n in enumerate(seq_lens):
        for t in range(starts[b], starts[b + 1]):
            out.append((t, b, n - (starts[b + 1] - t)))
    return out


def rotated_bound(dtype, value, size):
    """How far a rotated element may be off: one product is rounded to float32, then the fused sum
    (for 16-bit types; it is the output's own rounding in float32), then the output."""
    e = 2.0 ** -24 * size
    if dtype != "float32":
        e = e + 2.0 ** -24 * (abs(value) + e)
    return e + HALF_STEP[dtype] * (abs(value) + e) + TINY[dtype]


def attention(q, k, v, scale, limits):
    """One key/value head in float64: q [rows, D], k, v [n, D]; row r sees the keys below limits[r].
    -> O, L and what their bounds go by: sum of p |v| per element, the largest |score| and |q||k|
    of a row."""
    q, k, v = (x.astype(np.float64) for x in (q, k, v))
    rows, n = len(q), len(k)
    o, lse = np.zeros((rows, v.shape[1])), np.full(rows, -np.inf)
    size, top, prod = np.zeros_like(o), np.zeros(rows), np.zeros(rows)
    if n == 0:
        return o, lse, size, top, prod
    s = q @ k.T * scale
    hidden = np.arange(n)[None, :] >= np.asarray(limits)[:, None]
    some = ~hidden.all(1)
    top[some] = np.where(hidden, 0.0, abs(s)).max(1)[some]
    prod[some] = np.where(hidden, 0.0, abs(q) @ abs(k).T * scale).max(1)[some]
    s = np.where(hidden, -np.inf, s)
    with np.errstate(invalid="ignore"):
        m = s.max(1)
        some &= m > -np.inf
        p = np.exp(s - np.where(some, m, 0.0)[:, None])
    p[~some] = 0.0
    l = p.sum(1)
    lse[some] = m[some] + np.log(l[some])
    p[some] /= l[some, None]
    o, size = p @ v, p @ abs(v)
    return o, lse, size, top, prod


def attention_bounds(dtype, d, n, o, lse, size, top, prod, v_abs):
    """Bounds on |O - o| and |L - lse|, from the arithmetic: scores are float32 sums of d products
    (each of the d additions rounds: d 2^-24 of the largest sum of magnitudes, `prod`); the exponent's
    argument, in units of log 2, is rounded twice and its exponential and logarithm are good to 2^-22;
    sums over n keys, by blocks, lose at most n 2^-24; P is rounded to the inputs' type before P V
    (half a step, or the type's smallest half step against a sum of at least 1) and the output once."""
    eps = (d * 2.0 ** -24 * prod + 2.0 ** -22 * (3.0 + 1.45 * (top + abs(lse))))
    eps = np.where(np.isfinite(eps), eps, 0.0)
    l_bound = eps + n * 2.0 ** -24
    rel = np.expm1(2.0 * eps) + 2 * n * 2.0 ** -24
    half = 0.0 if dtype == "float32" else HALF_STEP[dtype]
    tiny = 0.0 if dtype == "float32" else 2.0 ** 8 * TINY[dtype] * v_abs
    o_bound = (half + rel)[:, None] * size * (1 + rel[:, None]) + tiny
    return o_bound + HALF_STEP[dtype] * (abs(o) + o_bound) + TINY[dtype], l_bound


class PagedCase:
    """Sequences in a shuffled paged cache, on the host and on the GPU. Rows that no key has and the
    page that unused table entries name hold NaN. `prefix` keys are the same pages for all of them."""

    def __init__(self, dtype, d, heads, kv_heads, page, lens, prefix=0, capacity=None, seed=1,
                 std=1.0, device="cuda"):
        import torch

        from cuflash_attn import synth

        self.dtype, self.d, self.heads, self.kv_heads, self.page = dtype, d, heads, kv_heads, page
        self.lens, self.prefix = list(lens), prefix
        B = len(lens)
        first = prefix // page
        longest = max(1, max(max(lens), prefix) if capacity is None else capacity)
        self.max_pages = -(-longest // page)
        prefix_pages = -(-prefix // page)
        own = [max(0, -(-min(n, self.max_pages * page) // page) - first) if n > prefix else 0
               for n in lens]
        pages = prefix_pages + sum(own) + 1
        rng = np.random.default_rng(seed)
        order = rng.permutation(pages)
        poison = order[-1]
        self.prefix_table, at = order[:prefix_pages], prefix_pages
        self.table = np.full((B, self.max_pages), poison)
        for b in range(B):
            self.table[b, first:first + own[b]] = order[at:at + own[b]]
            at += own[b]
        shape = (pages, page, kv_heads, d)
        k, v = (synth.round_to(synth.normal(seed + s, shape, std), dtype) for s in (1, 2))
        # Keys and values of each sequence, [n, kv_heads, d].
        used = np.zeros(shape[:2], dtype=bool)
        self.keys, self.values = [], []
        for b, n in enumerate(lens):
            n = min(max(n, 0), self.max_pages * page)
            j = np.arange(n)
            pg = np.where(j < prefix, 0, self.table[b, j // page]) if n else j
            if prefix and n:
                pg = np.where(j < prefix, self.prefix_table[np.minimum(j, prefix - 1) // page], pg)
            used[pg, j % page] = True
            self.keys.append((pg, j % page))
        if prefix:
            j = np.arange(prefix)
            used[self.prefix_table[j // page], j % page] = True
        k[~used], v[~used] = np.nan, np.nan
        self.k, self.v = k, v
        self.t_k, self.t_v = (synth.to_torch(x, dtype, device) for x in (k, v))
        ints = lambda x: torch.tensor(np.asarray(x).tolist(), dtype=torch.int32,  # noqa: E731
                                      device=device)
        self.ints = ints
        self.t_table, self.t_lens = ints(self.table), ints(self.lens)
        self.t_prefix = ints(self.prefix_table) if prefix else None

    def sequence(self, b):
        """Keys and values of sequence b, [n, kv_heads, d]."""
        pg, row = self.keys[b]
        return self.k[pg, row], self.v[pg, row]

    def check(self, q, new, causal, o, lse, scale=None):
        """Compares O [T, heads, d] and L [T, heads] of packed queries q, new[b] of sequence b."""
        scale = self.d ** -0.5 if scale is None else scale
        group, t0 = self.heads // self.kv_heads, 0
        for b, n in enumerate(new):
            keys, values = self.sequence(b)
            limits = [max(0, len(keys) - n + i + 1) if causal else len(keys) for i in range(n)]
            for h in range(self.kv_heads):
                at = (slice(t0, t0 + n), slice(h * group, (h + 1) * group))
                x = q[at].reshape(n * group, self.d)
                want = attention(x, keys[:, h], values[:, h], scale, np.repeat(limits, group))
                v_abs = abs(values[:, h]).sum(0) if len(keys) else 0.0
                o_bound, l_bound = attention_bounds(self.dtype, self.d, len(keys), *want, v_abs)
                got_o, got_l = o[at].reshape(n * group, self.d), lse[at].reshape(n * group)
                where = f"sequence {b}, key/value head {h}"
                off = abs(got_o - want[0]) - o_bound
                assert (off <= 0).all(), (where, off.max(), np.argwhere(~(off <= 0))[:4])
                none = np.isneginf(want[1])
                assert np.array_equal(np.isneginf(got_l), none), where
                off = abs(got_l[~none] - want[1][~none]) - l_bound[~none]
                assert (off <= 0).all(), (where, "L", off.max())
            t0 += n
