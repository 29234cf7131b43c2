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


@pytest.mark.parametrize("cache,act", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.float16, torch.float16)])
def test_append_and_copies_in_a_graph(cache, act):
    """Replays write the tokens, and copy the pages, that the operands name at the replay; the eager calls' bits."""
    g = gen(2)
    layers, pages, kv, page, dim, batch, n = 2, 20, 3, 16, 40, 3, 9
    pools = [torch.randn(layers, pages, kv, page, dim, generator=g).to(cache).cuda() for _ in range(2)]
    pools.append(torch.zeros(layers, pages, kv, dim, device="cuda"))
    k, v = (torch.zeros(layers, batch, n, kv, dim, dtype=act, device="cuda") for _ in range(2))
    table = torch.arange(12, dtype=torch.int32).view(3, 4).cuda()
    lengths, rows = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros(3, 6, dtype=torch.int32, device="cuda")

    def step(k_pages, v_pages, means):
        kiln.cache_append(k, v, k_pages, v_pages, table, lengths, rows=rows, k_means=means)
        kiln.copy_pages([k_pages, v_pages, means.unsqueeze(-2)], [0, 4, 8], [15, 16, 17])

    step(*[t.clone() for t in pools])
    mine, graphs = [t.clone() for t in pools], []
    for _ in range(2):     # two graphs over the same pools
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            step(*mine)
    for a, b in zip(mine, pools):
        a.copy_(b)
    for turn in range(4):
        for t in (k, v):
            t.copy_(torch.randn(t.shape, generator=g))
        lengths.copy_(torch.tensor([turn * 5, 11 + turn, 40 - turn], dtype=torch.int32))
        rows.copy_(torch.randint(-1, n, (3, 6), generator=g))
        graphs[turn % 2].replay()
        step(*pools)
        assert all(torch.equal(a, b) for a, b in zip(mine, pools))


def test_calls_from_several_threads():
    """Each thread on a stream of its own, the same and other forms of calls at once."""
    import threading

    problems = [ref.problem(gen(i), batch=2, draft=1 + i % 3, lengths=(900, 40 * i), cache=torch.bfloat16, device="cuda")
                for i in range(4)]
    means = [p["k_pages"].float().mean(2) for p in problems]

    def step(i):
        p = problems[i]
        sel = kiln.select_pages(p["q"], means[i], p["table"], p["lengths"], page_size=16, pages=5)
        return kiln.tree_attention(**p), sel, kiln.selected_attention(**p, selected=sel)

    want = [step(i) for i in range(4)]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    for j in (i, (i + 1) % 4):
                        got = step(j)
                        torch.cuda.current_stream().synchronize()
                        if not all(torch.equal(a, b) for a, b in zip(got, want[j])):
                            wrong.append((i, j))
        except Exception as error:      # (an exception in a thread would go unseen)
            wrong.append(error)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
