"""The cuts of the paged attentions (cuflash-attn_amd/csrc/paged_plan.hpp) on the host, beyond the launches
of test_paged_cache.py."""

from __future__ import annotations

from test_host_rules import run_program


def test_shared_cut_up_to_the_key_limit(tmp_path):
    """Lengths up to 2^31 - 1024 (tests/cpp/test_paged_limits.cpp)."""
    run_program("test_paged_limits", tmp_path, 300, 1)
