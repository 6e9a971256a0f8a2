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
