"""The cuts of the paged attentions (cuflash-attn_amd/csrc/paged_plan.hpp) on the host, beyond the launches
of test_paged_cache.py."""

from __future__ import annotations

from test_host_rules import run_program


def test_every_shape_up_to_the_key_limit(tmp_path):
    """The shapes of all engines, lengths up to 2^31 - 1024, more than 96 query heads over a key/value
    head (tests/cpp/test_paged_limits.cpp)."""
    run_program("test_paged_limits", tmp_path, 300, 1)
