"""An 8-bit paged cache in plain numpy (include/cuflash/paged_cache_q8.h): codes, exponents and values,
and sequences in such a cache. What attention over it gives is paged_reference.py's, on the values."""

from __future__ import annotations

import numpy as np

from paged_reference import attention, attention_bounds

TOP = {"int8": 127.0, "e4m3": 448.0}


def most_exponent(code, dtype):
    if dtype == "float16":
        return 9 if code == "int8" else 7
    return 121 if code == "int8" else 119


def _e4m3_table():
    c = np.arange(256)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e > 0, (8.0 + m) * 2.0 ** (e - 10.0), m * 2.0 ** -9)
    v[(c & 127) == 127] = np.nan
    return np.where(c & 128, -v, v)


E4M3 = _e4m3_table()


def code_values(codes, code):
    """What codes (uint8 bytes) are as numbers, float64."""
    return codes.view(np.int8).astype(np.float64) if code == "int8" else E4M3[codes]


def values(codes, exps, code):
    """codes [..., D] uint8 with exponents [...] uint8, float64."""
    with np.errstate(over="ignore"):
        f = np.where(exps == 255, np.nan, 2.0 ** (exps.astype(np.float64) - 127.0))
    return code_values(codes, code) * f[..., None]


def quantise(x, code, dtype):
    """Codes and exponents of rows x [..., D] float32. Everything is exact but the codes' rounding."""
    x = np.ascontiguousarray(x, dtype=np.float32)
    amax = abs(x).max(-1).astype(np.float64)
    number = np.isfinite(amax)
    amax = np.where(number, amax, 0.0)
    top = TOP[code]
    with np.errstate(divide="ignore"):
        e = np.where(amax > 0, np.ceil(np.log2(amax / top)), -1000.0)
    e = np.where(amax > top * 2.0 ** e, e + 1, e)  # the logarithm is rounded
    e = np.where((amax > 0) & (amax <= top * 2.0 ** (e - 1)), e - 1, e)
    e = np.clip(e, -100, most_exponent(code, dtype))
    with np.errstate(invalid="ignore", over="ignore"):
        y = np.clip(x.astype(np.float64) * 2.0 ** -e[..., None], -top, top)
    y[~number] = 0.0
    if code == "int8":
        codes = np.rint(y).astype(np.int8).view(np.uint8)
    else:
        # The nearest of the codes from 0 up, an even one where two are as near.
        up = E4M3[:127]
        mag = abs(y)
        hi = np.clip(np.searchsorted(up, mag), 1, 126)
        lo = hi - 1
        a, b = mag - up[lo], up[hi] - mag
        pick = np.where(a < b, lo, np.where(b < a, hi, np.where(lo % 2 == 0, lo, hi)))
        codes = (pick | np.where(np.signbit(y), 128, 0)).astype(np.uint8)
        codes[~number] = 0x7F
    return codes, np.where(number, e + 127, 255).astype(np.uint8)


def rotate32(x, pos, cos, sin, interleaved):
    """x [T, heads, D] float32 rotated by rows pos of cos, sin, every operation rounded to float32."""
    y = x.astype(np.float32).copy()
    half = cos.shape[1]
    one = np.arange(half) * (2 if interleaved else 1)
    two = one + (1 if interleaved else half)
    c, s = (t[pos][:, None, :] for t in (cos, sin))
    a, b = y[..., one].copy(), y[..., two].copy()
    y[..., one] = a * c - b * s
    y[..., two] = b * c + a * s
    return y


def torch_cache(codes, code, device="cuda"):
    import torch

    t = torch.from_numpy(np.ascontiguousarray(codes).view(np.int8)).to(device)
    return t if code == "int8" else t.view(torch.float8_e4m3fn)


class Q8Case:
    """Sequences in a shuffled 8-bit cache, on the host and on the GPU. Rows that no key has and the page
    that unused table entries name hold NaN: x = 255 and, for e4m3, NaN codes."""

    def __init__(self, dtype, code, d, heads, kv_heads, page, lens, capacity=None, seed=1, std=1.0):
        import torch

        from cuflash_attn import synth

        self.dtype, self.code, self.d, self.page = dtype, code, d, page
        self.heads, self.kv_heads, self.lens = heads, kv_heads, list(lens)
        B = len(lens)
        longest = max(1, max(lens) if capacity is None else capacity)
        self.max_pages = -(-longest // page)
        cap = self.max_pages * page
        own = [-(-min(max(n, 0), cap) // page) for n in lens]
        pages = sum(own) + 1
        rng = np.random.default_rng(seed)
        order = rng.permutation(pages)
        self.unused = order[-1]
        self.table = np.full((B, self.max_pages), self.unused)
        at = 0
        for b in range(B):
            self.table[b, :own[b]] = order[at:at + own[b]]
            at += own[b]
        shape = (pages, page, kv_heads, d)
        used = np.zeros(shape[:2], dtype=bool)
        self.places = []
        for b, n in enumerate(lens):
            j = np.arange(min(max(n, 0), cap))
            pg = self.table[b, j // page]
            used[pg, j % page] = True
            self.places.append((pg, j % page))
        self.codes, self.exps = [], []
        for s in (1, 2):
            c, e = quantise(synth.normal(seed + s, shape, std), code, dtype)
            c[~used] = 0x7F
            e[~used] = 255
            self.codes.append(c)
            self.exps.append(e)
        ints = lambda x: torch.tensor(np.asarray(x).tolist(), dtype=torch.int32,  # noqa: E731
                                      device="cuda")
        self.ints = ints
        self.t_table, self.t_lens = ints(self.table), ints(self.lens)
        self.upload()

    def upload(self):
        import torch

        self.t_k, self.t_v = (torch_cache(c, self.code) for c in self.codes)
        self.t_kx, self.t_vx = (torch.from_numpy(e.transpose(0, 2, 1).copy()).cuda()
                                for e in self.exps)
        self.cache = (self.t_k, self.t_v, self.t_kx, self.t_vx)

    def sequence(self, b):
        """Keys and values of sequence b, [n, kv_heads, d] float64."""
        pg, row = self.places[b]
        return tuple(values(c[pg, row], e[pg, row], self.code)
                     for c, e in zip(self.codes, self.exps))

    def check(self, q, new, causal, o, lse, scale=None, only=None):
        """Compares O [T, heads, d] and L [T, heads] of packed queries q, new[b] of sequence b. A float
        query takes part in three pieces, so three times as many products are summed."""
        scale = self.d ** -0.5 if scale is None else scale
        group, t0 = self.heads // self.kv_heads, 0
        times = 3 if self.dtype == "float32" else 1
        for b, n in enumerate(new):
            if only is not None and b not in only:
                t0 += n
                continue
            keys, vals = self.sequence(b)
            limits = [max(0, len(keys) - n + i + 1) if causal else len(keys) for i in range(n)]
            for h in range(self.kv_heads):
                at = (slice(t0, t0 + n), slice(h * group, (h + 1) * group))
                x = q[at].reshape(n * group, self.d)
                want = attention(x, keys[:, h], vals[:, h], scale, np.repeat(limits, group))
                v_abs = abs(vals[:, h]).sum(0) if len(keys) else 0.0
                o_bound, l_bound = attention_bounds(self.dtype, times * self.d, times * len(keys),
                                                    *want, v_abs)
                got_o, got_l = o[at].reshape(n * group, self.d), lse[at].reshape(n * group)
                where = f"sequence {b}, key/value head {h}"
                off = abs(got_o - want[0]) - o_bound
                assert (off <= 0).all(), (where, off.max(), np.argwhere(~(off <= 0))[:4])
                none = np.isneginf(want[1])
                assert np.array_equal(np.isneginf(got_l), none), where
                off = abs(got_l[~none] - want[1][~none]) - l_bound[~none]
                assert (off <= 0).all(), (where, "L", off.max())
            t0 += n
