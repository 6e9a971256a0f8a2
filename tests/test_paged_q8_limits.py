"""The largest attentions over an 8-bit paged cache: those with more tiles than the cut into waves has room for are
refused before any GPU call, the others are cut without passing 32 bits."""

from __future__ import annotations

import pytest

from cuflash_attn import INVALID_DIMENSION
from test_host_rules import run_program
from test_paged_cache import _call
from test_paged_cache_q8 import DECODE, FORWARD, SFX


@pytest.mark.parametrize("sfx", SFX)
@pytest.mark.parametrize("code", [0, 1])
@pytest.mark.parametrize("d", [32, 64, 128])
def test_too_many_tiles_are_refused(lib, sfx, code, d):
    many = (1 << 30) + 1
    one = dict(heads=1, kv_heads=1, page=2048, max_pages=1, d=d, code=code)
    assert _call(lib, "decode_paged_q8", sfx, DECODE, batch=many, **one) == INVALID_DIMENSION
    assert _call(lib, "forward_paged_q8", sfx, FORWARD, batch=many, tokens=many,
                 **one) == INVALID_DIMENSION
    assert _call(lib, "forward_paged_q8", sfx, FORWARD, batch=(1 << 31) - 63, tokens=5,
                 **one) == INVALID_DIMENSION


def test_tiles_that_fit_and_those_that_do_not(tmp_path):
    run_program("test_paged_q8_limits", tmp_path)


def test_starts_that_decrease_stay_in_bounds(tmp_path):
    """Also where the sum over all sequences passes 32 bits."""
    run_program("test_paged_q8_disorder", tmp_path, 300, 1)
