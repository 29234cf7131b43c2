"""verify_tokens on the GPU against its definition in 64 bits, and the whole
decoding step. Whole numbers, compared for equality (test_verify.py says why
they can be)."""

import math

import pytest
import torch

import kiln
import packed_reference as ref
import test_verify
from kiln.hip import lib as kl

pytestmark = pytest.mark.gpu


def gen(seed=0):
    return torch.Generator().manual_seed(seed)


def workspace(batch, n, vocab, type=kl.TYPE_F32):
    """Bytes of a call's workspace: where there are some, the first sums are a launch of their own."""
    size = kl.ctypes.c_size_t()
    kl.check(kl.load().kh_verify_workspace_bytes(kl.Verify(batch, n, vocab, type), size), "")
    return size.value


def check(p):
    got = kiln.verify_tokens(**p)
    for a, b in zip(got, ref.verify(**{k: None if t is None else t.cpu() for k, t in p.items()})):
        assert a.dtype == torch.int32 and a.tolist() == b
    return got


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tree", [True, False], ids=["tree", "chain"])
@pytest.mark.parametrize("probs", [True, False], ids=["probs", "sampled"])
@pytest.mark.parametrize("batch,n,vocab", [(1, 1, 1), (1, 5, 50257), (3, 2, 1023), (6, 7, 1025), (5, 40, 300), (2, 256, 4099),
                                           (300, 3, 2500), (4, 9, 7)])
def test_sizes(dtype, tree, probs, batch, n, vocab):
    p = ref.drafted(gen(n), batch, n, vocab, dtype, tree, probs, device="cuda")
    check(p)
    check(dict(p, tokens=p["tokens"].to(torch.int32), uniforms=p["uniforms"].double()))


# More than 65536 tokens: the first sums of few sequences are a launch of their own.
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tree", [True, False], ids=["tree", "chain"])
@pytest.mark.parametrize("probs", [True, False], ids=["probs", "sampled"])
@pytest.mark.parametrize("batch,n,vocab", [(1, 1, 65537), (3, 7, 70001), (2, 5, 128000)])
def test_first_sums_beforehand(dtype, tree, probs, batch, n, vocab):
    assert workspace(batch, n, vocab)
    p = ref.drafted(gen(n), batch, n, vocab, dtype, tree, probs, device="cuda")
    check(p)
    check(dict(p, tokens=p["tokens"].to(torch.int32), uniforms=p["uniforms"].double()))


@pytest.mark.parametrize("probs", [True, False], ids=["probs", "sampled"])
def test_large_vocabulary(probs):
    # more stretches than are kept: longer ones
    for vocab in (2 ** 20 + 5, 3 * 2 ** 20 + 1):
        check(ref.drafted(gen(1), 2, 3, vocab, probs=probs, device="cuda"))


def test_refused_often():
    # a draft that knows little: refusals one after another, under one token and along the path
    for batch in (4, 260):
        p = ref.drafted(gen(2), batch, 30, 700, noise=3.0, device="cuda")
        counts = check(p)[1]
        assert 1 <= int(counts.max()) < 30


def test_refused_often_beside_the_first_sums():
    # several refusals under one token, and tokens kept after a refusal, behind sums that were made beforehand
    p = ref.drafted(gen(2), 4, 30, 70001, noise=3.0, device="cuda")
    assert workspace(4, 30, 70001)
    counts = check(p)[1]
    assert 1 <= int(counts.max()) < 30
    # the root's children 1 to 4 are refused, 5 is kept; 6 and 7, its own, too are refused and kept
    p["parents"][0] = torch.tensor([-1, 0, 0, 0, 0, 0, 5, 5] + [7] * 22)
    p["uniforms"][0, 1:5], p["uniforms"][0, 6] = 1.0, 1.0
    p["uniforms"][0, 5], p["uniforms"][0, 7], p["uniforms"][0, 8:] = 0.0, 0.0, 1.0
    for i, up in ((5, 0), (7, 5)):        # (something is left of these)
        p["tokens"][0, i] = (p["target"][0, up] - 3 * p["draft"][0, up]).argmax()
    for i, up in ((1, 0), (2, 0), (3, 0), (4, 0), (6, 5)):
        p["tokens"][0, i] = p["draft"][0, up].argmax()
        p["draft"][0, up, p["tokens"][0, i]] += p["target"][0, up, p["tokens"][0, i]]
    rows, counts, _ = check(p)
    assert rows[0].tolist()[:3] == [0, 5, 7]


def test_unused_and_odd_tokens_beside_the_first_sums():
    for probs in (True, False):
        p = ref.drafted(gen(3), 5, 6, 70001, probs=probs, device="cuda")
        p["parents"] = torch.tensor([[-2, 0, 0, 1, 2, 3], [-1, -1, -1, 0, 1, 2], [-1, 1, 5, 0, -7, 3], [0, 0, 0, 0, 0, 0], [-1, 0, 0, 0, 0, 0]],
                                    dtype=torch.int32, device="cuda")
        p["tokens"][4] = torch.tensor([0, -1, 70001, 2 ** 40, 3, 3])
        counts = check(p)[1]
        assert counts[0] == 0 and counts[3] == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_odd_probabilities_beside_the_first_sums(dtype):
    for probs in (True, False):
        p = ref.drafted(gen(4), 7, 4, 70001, dtype, probs=probs, tree=False, device="cuda")
        p["target"][0] = 0.0
        p["target"][1, :, ::2] = math.nan
        p["target"][2, :, 3] = math.inf
        p["target"][3] *= -1.0
        p["target"][4] = p["target"][4] * 0
        p["target"][4, :, 69999] = 1.0
        p["uniforms"][5] = torch.tensor([1.0, 0.0, math.nan, -3.0])
        p["uniforms"][6] = 1.0 - 2.0 ** -24
        if probs:
            p["draft"][1, :, 5] = math.nan
            p["draft"][6] = p["target"][6]
            p["uniforms"][6] = 1.0
        assert check(p)[2].tolist()[0] == -1


def test_unused_and_odd_tokens():
    for probs in (True, False):
        p = ref.drafted(gen(3), 5, 6, 20, probs=probs, device="cuda")
        p["parents"] = torch.tensor([[-2, 0, 0, 1, 2, 3], [-1, -1, -1, 0, 1, 2], [-1, 1, 5, 0, -7, 3], [0, 0, 0, 0, 0, 0], [-1, 0, 0, 0, 0, 0]],
                                    dtype=torch.int32, device="cuda")
        p["tokens"][4] = torch.tensor([0, -1, 20, 2 ** 40, 3, 3])
        check(p)


def test_odd_probabilities():
    for probs in (True, False):
        p = ref.drafted(gen(4), 7, 4, 3000, probs=probs, tree=False, device="cuda")
        p["target"][0] = 0.0
        p["target"][1, :, ::2] = math.nan
        p["target"][2, :, 3] = math.inf
        p["target"][3] *= -1.0
        p["target"][4] = p["target"][4] * 0
        p["target"][4, :, 2999] = 1.0
        p["uniforms"][5] = torch.tensor([1.0, 0.0, math.nan, -3.0])
        p["uniforms"][6] = 1.0 - 2.0 ** -24
        if probs:
            p["draft"][1, :, 5] = math.nan
            p["draft"][6] = p["target"][6]
            p["uniforms"][6] = 1.0
        check(p)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("vocab", [40, 3000])
def test_draft_probabilities_that_count_as_nothing(dtype, vocab):
    for seed in range(3):
        p = ref.drafted(gen(seed), 6, 9, vocab, dtype, noise=2.0, device="cuda")
        odd, want = test_verify.odd_drafts(p)
        check(want)
        assert [t.tolist() for t in kiln.verify_tokens(**odd)] == [t.tolist() for t in kiln.verify_tokens(**want)]


def test_strides_and_odd_places():
    p = ref.drafted(gen(6), 3, 5, 1717, torch.bfloat16, device="cuda")
    want = [t.tolist() for t in kiln.verify_tokens(**p)]
    wide = torch.full((3, 5, 1720), math.nan, dtype=torch.bfloat16, device="cuda")   # rows at odd elements, NaN behind them
    wide[..., 1:1718] = p["target"]
    flat = torch.full((p["draft"].numel() + 1,), math.nan, dtype=torch.bfloat16, device="cuda")
    flat[1:] = p["draft"].flatten()
    q = dict(p, tokens=p["tokens"].t().contiguous().t(), target=wide[..., 1:1718], draft=flat[1:].view(3, 5, 1717),
             uniforms=torch.stack([p["uniforms"]] * 2, -1)[..., 0])
    assert [t.tolist() for t in kiln.verify_tokens(**q)] == want


@pytest.mark.parametrize("probs", [True, False], ids=["probs", "sampled"])
def test_rows_past_32_bits(probs):
    """A second sequence's rows more than 2^31 elements behind the first one's."""
    p = ref.drafted(gen(7), 2, 4, 2050, torch.bfloat16, probs=probs, device="cuda")
    want = [t.tolist() for t in kiln.verify_tokens(**p)]
    far = 2 ** 31 + 64
    for name in ("target", "draft"):
        if p[name] is not None:
            rows = torch.empty(far + 4 * 2050, dtype=torch.bfloat16, device="cuda").as_strided((2, 4, 2050), (far, 2050, 1))
            p[name] = rows.copy_(p[name])
    assert [t.tolist() for t in kiln.verify_tokens(**p)] == want


def test_graph_and_streams():
    p = ref.drafted(gen(7), 4, 6, 5000, device="cuda")
    more = [ref.drafted(gen(8 + i), 4, 6, 5000, device="cuda") for i in range(4)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kiln.verify_tokens(**p)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = kiln.verify_tokens(**p)
        second = kiln.verify_tokens(**dict(p, draft=None))    # (its own workspace)
    for q in more:
        for name, t in p.items():
            t.copy_(q[name])
        graph.replay()
        eager, eager2 = kiln.verify_tokens(**p), kiln.verify_tokens(**dict(p, draft=None))
        torch.cuda.synchronize()
        for a, b, c in zip(out, eager, ref.verify(**q)):
            assert a.tolist() == b.tolist() == c
        assert all(torch.equal(a, b) for a, b in zip(second, eager2))


def test_graph_with_workspaces():
    # two calls with a workspace each in one graph, and a second graph of one call: nothing is shared
    sizes = (4, 6, 70001)
    assert workspace(*sizes)
    p, q = (ref.drafted(gen(i), *sizes, device="cuda") for i in (7, 17))
    more = [ref.drafted(gen(8 + i), *sizes, device="cuda") for i in range(3)]
    kiln.verify_tokens(**p)
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    with torch.cuda.graph(graphs[0]):
        first = kiln.verify_tokens(**p)
        second = kiln.verify_tokens(**dict(p, draft=None))
    with torch.cuda.graph(graphs[1]):
        third = kiln.verify_tokens(**q)
    for x in more:
        for name, t in p.items():
            t.copy_(x[name])
        graphs[0].replay()
        graphs[1].replay()
        eager = kiln.verify_tokens(**p), kiln.verify_tokens(**dict(p, draft=None)), kiln.verify_tokens(**q)
        torch.cuda.synchronize()
        for got, want in zip((first, second, third), eager):
            assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert [t.tolist() for t in first] == list(ref.verify(**x))
    assert [t.tolist() for t in third] == list(ref.verify(**{k: t.cpu() for k, t in q.items()}))


def test_as_an_operator_of_torch():
    p = ref.drafted(gen(9), 2, 4, 100, device="cuda")
    with torch.utils.flop_counter.FlopCounterMode(display=False):
        got = kiln.verify_tokens(**p)
    for a, b in zip(got, kiln.verify_tokens(**p)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("packed", [True, False], ids=["fp4", "bf16"])
def test_decoding_steps(packed):
    # draft, attend, verify, append, let go of pages: what the cache then holds is the kept tokens, and what a
    # later step attends to is them
    g = gen(10)
    seqs, n, kv, dim, vocab, window, sinks = 3, 7, 2, 64, 50, 40, 3
    cache = kiln.PagedCache(2, 40, 16, kv, dim, dtype=torch.float4_e2m1fn_x2 if packed else torch.bfloat16, device="cuda")
    ids = [cache.open() for _ in range(seqs)]
    stored = (lambda t: ref.rounded(t)) if packed else (lambda t: t.bfloat16().double())
    held = [(torch.zeros(2, 0, kv, dim, dtype=torch.float64),) * 2 for _ in ids]
    for step in range(25):
        p = ref.drafted(g, seqs, n, vocab, device="cuda")
        q, (k, v) = torch.randn(seqs, n, 4, dim, generator=g), (torch.randn(2, seqs, n, kv, dim, generator=g) for _ in "kv")
        table, lengths = cache.batch(ids)
        for layer in range(2):
            got = kiln.tree_attention(q.cuda(), k[layer].cuda(), v[layer].cuda(), cache.k[layer], cache.v[layer], table, lengths,
                                      p["parents"], window=window, sinks=sinks)
            for s in range(seqs):
                mine = [t[layer] for t in held[s]]
                for i, path in enumerate(ref.paths(p["parents"][s].tolist(), n)):
                    kk, vv = (torch.cat([a, stored(b[layer, s, path])]) for a, b in zip(mine, (k, v)))
                    at = torch.arange(len(kk))
                    seen = (at < sinks) | (at > len(kk) - 1 - window)
                    for h in range(4):
                        w = torch.softmax(kk[seen, h // 2] @ q[s, i, h].double() / 8.0, 0)
                        torch.testing.assert_close(got[s, i, h].cpu().double(), w @ vv[seen, h // 2], rtol=0, atol=1e-4)
        rows, counts, after = check(p)
        rows = [r[:c] for r, c in zip(rows.tolist(), counts.tolist())]
        cache.append(ids, k.cuda(), v.cuda(), rows=rows)
        for s, path in enumerate(rows):
            held[s] = tuple(torch.cat([a, stored(t[:, s, path])], 1) for a, t in zip(held[s], (k, v)))
            cache.release(ids[s], window=window, sinks=sinks)
        assert [cache.length(s) for s in ids] == [t[0].shape[1] for t in held]
    assert min(map(cache.length, ids)) > window + sinks + 16
    assert cache.free_pages >= 40 - seqs * (1 + -(-window // 16) + 1)
