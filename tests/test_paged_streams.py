"""The stream argument of the paged attentions' tensor helpers: what is captured is that stream, whichever
is torch's current one."""

from __future__ import annotations

import contextlib

import pytest

import cuflash_attn
from paged_reference import PagedCase


class _Sizes:
    """A library whose workspace sizes are 512."""

    def fn(self, kind, sfx):
        assert kind.endswith("_workspace") and sfx == "f32"
        return lambda *sizes: 512


@pytest.mark.parametrize("current,stream,captured,given", [
    ("main", None, "main", True), ("main", None, "side", False),
    ("main", "side", "side", True), ("main", "side", "main", False)])
def test_workspace_where_the_calls_stream_is_captured(monkeypatch, current, stream, captured, given):
    import torch

    at = [current]

    @contextlib.contextmanager
    def on(s):
        at.append(s)
        yield
        at.pop()

    monkeypatch.setattr(torch.cuda, "stream", on)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: at[-1] == captured)
    ptr, size, keep = cuflash_attn._captured_workspace(_Sizes(), "decode_shared", torch.zeros(1),
                                                       stream, 4, 8, 2, 64)
    assert (ptr, size) == ((keep.data_ptr(), 512) if given else (None, 0))
    assert at == [current]


@pytest.mark.gpu
def test_captured_stream_is_not_the_current_one(torch_gpu, lib):
    """The three operators captured through `stream`, another stream being current: with a workspace, so
    in the same chunks as the eager calls."""
    torch = torch_gpu
    c = PagedCase("bfloat16", 128, 8, 2, 16, prefix=208, lens=[3000, 230, 209], capacity=3008)
    c.t_table[:, :13] = c.t_prefix[:13]
    starts = c.ints([0, 1, 2, 3])
    x = torch.empty((3, 12, 128), device="cuda", dtype=torch.bfloat16)

    def step(stream=None):
        q = cuflash_attn.flash_attention_append_paged(x[:, 8:10], x[:, 10:], c.t_k, c.t_v, c.t_table,
                                                      c.t_lens, q=x[:, :8], stream=stream)
        return [q, *cuflash_attn.flash_attention_forward_paged(
            q, c.t_k, c.t_v, c.t_table, c.t_lens, starts, causal=True, stream=stream),
            *cuflash_attn.flash_attention_decode_shared(
                q.unsqueeze(2), c.t_k, c.t_v, c.t_prefix, 208, c.t_table, c.t_lens, stream=stream)]

    x.normal_()
    step()
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = torch.cuda.current_stream()
        with torch.cuda.stream(other):
            out = step(captured)
    torch.cuda.synchronize()
    for rep in range(3):
        print(f"[another stream current] replay {rep}", flush=True)
        x.normal_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [y.clone() for y in out]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), rep
