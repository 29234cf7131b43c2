"""Calls of the paged cache and its operators as a program makes them on the GPU."""

import pytest
import torch

import kiln
import paged_reference as ref

pytestmark = pytest.mark.gpu


def gen(seed=0):
    return torch.Generator().manual_seed(seed)


def test_the_cache_refuses_to_be_captured():
    cache = kiln.PagedCache(1, 6, 16, 2, 8, dtype=torch.float32)
    a = cache.open()
    k = torch.randn(1, 1, 20, 2, 8, generator=gen()).cuda()
    cache.append([a], k, k)
    table, lengths = cache.batch([a])
    p = ref.problem(gen(1), batch=1, draft=3, heads=2, kv=2, dim=8, lengths=(20,), device="cuda")
    args = (p["q"], p["k"], p["v"], cache.k[0], cache.v[0], table, lengths, p["parents"])
    want = kiln.tree_attention(*args)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = kiln.tree_attention(*args)
        for call in (lambda: cache.append([a], k, k), lambda: cache.batch([a]), cache.compact):
            with pytest.raises(RuntimeError, match="captured"):
                call()
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(out, want)
    cache.append([a], k, k)
    assert cache.length(a) == 40


def test_a_device_without_a_number_is_the_current_one():
    cache = kiln.PagedCache(1, 6, 16, 2, 8, device="cuda")
    assert cache.device == cache.k.device == torch.device("cuda", torch.cuda.current_device())
    a = cache.open()
    table, lengths = cache.batch([a])
    assert table.device == lengths.device == cache.device
