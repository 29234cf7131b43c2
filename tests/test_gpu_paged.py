"""The paged cache's operators on the GPU against their definitions in 64 bits.

Tolerances. A result is a weighted mean of values: with weights off by a
relative e_w each and values exact, it is off by at most 2 e_w times the
largest |value| (numerator and denominator). A score off by e_s moves its
weight by a relative e_s. fp32 work: scores of |s| < 32 (normal inputs, dim
256) in products whose sums round once a product at 2^-24 of their partial
sums, which 64 of random sign keep under 2^-18; so e_s < 2^-18, weights and
their sums add under 2^-20, and the mean's own sums another 2^-18 of the
largest value (|v| < 6): 2 * 6 * 2^-17 < 1e-4 at the worst, for any element.
A 16-bit result adds half a step of itself, and one pass over 16-bit weights
half a step of each weight, 2 * 6 * eps / 2 at the worst; random signs of the
weights' roundings keep it far below.
"""

import math

import pytest
import torch

import kiln
import paged_reference as ref

pytestmark = pytest.mark.gpu

TYPES = [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.float16, torch.float32),
         (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16)]
IDS = ["fp32", "bf16-cache", "fp16-cache", "bf16", "fp16"]


def tolerance(act):
    if act == torch.float32:
        return dict(rtol=0.0, atol=1e-4)
    half = torch.finfo(act).eps / 2
    return dict(rtol=half, atol=1e-4 + 2 * 6 * half)


def gen(seed=0):
    return torch.Generator().manual_seed(seed)


def check(p, parents="parents", **more):
    got = kiln.tree_attention(**p, **more)
    want = ref.attention(**{k: v for k, v in p.items()}, **more)
    assert got.dtype == p["q"].dtype and got.shape == p["q"].shape
    torch.testing.assert_close(got.double().cpu(), want, equal_nan=True, **tolerance(got.dtype))
    return got


@pytest.mark.parametrize("cache,act", TYPES, ids=IDS)
@pytest.mark.parametrize("dim", [8, 64, 80, 128, 200, 256])
@pytest.mark.parametrize("heads,kv,draft", [(2, 2, 1), (4, 1, 5), (6, 2, 33)])
def test_types_heads_dims(cache, act, dim, heads, kv, draft):
    check(ref.problem(gen(dim), draft=draft, heads=heads, kv=kv, dim=dim, cache=cache, act=act, device="cuda"))


@pytest.mark.parametrize("cache,act", TYPES, ids=IDS)
@pytest.mark.parametrize("page", [16, 32, 128, 1024])
@pytest.mark.parametrize("lengths", [(0, 0), (1, 0), (15, 16), (31, 33), (129, 1000), (2049, 5)], ids=str)
def test_lengths_and_pages(cache, act, page, lengths):
    check(ref.problem(gen(page), lengths=lengths, page=page, cache=cache, act=act, device="cuda"))


@pytest.mark.parametrize("draft", [1, 2, 31, 32, 33, 64, 100, 256])
@pytest.mark.parametrize("tree", [True, False], ids=["tree", "chain"])
def test_drafts(draft, tree):
    check(ref.problem(gen(draft), draft=draft, heads=3, kv=1, tree=tree, lengths=(50, 0), cache=torch.bfloat16, device="cuda"))
    check(ref.problem(gen(draft), draft=draft, heads=8, kv=1, tree=tree, lengths=(50, 3), cache=torch.float16,
                      act=torch.float16, dim=128, device="cuda"))


@pytest.mark.parametrize("cache,act", TYPES, ids=IDS)
def test_long_and_ragged(cache, act):
    # ranges that end inside an item, and many items in one range
    lengths = (5000, 0, 1, 700, 33, 2600, 64, 16)
    check(ref.problem(gen(1), batch=8, draft=2, heads=4, kv=2, lengths=lengths, cache=cache, act=act, device="cuda"))
    check(ref.problem(gen(2), batch=40, draft=1, heads=2, kv=1, lengths=[7 * i for i in range(40)], cache=cache,
                      act=act, device="cuda"))


@pytest.mark.parametrize("cache,act", TYPES, ids=IDS)
@pytest.mark.parametrize("tree", [True, False], ids=["tree", "chain"])
def test_picked_pages(cache, act, tree):
    p = ref.problem(gen(3), batch=3, draft=5, heads=6, kv=2, lengths=(300, 0, 41), cache=cache, act=act, tree=tree,
                    device="cuda")
    means = p["k_pages"].float().mean(2)
    for top in (1, 2, 7, 30):
        sel = kiln.select_pages(p["q"], means, p["table"], p["lengths"], page_size=16, pages=top)
        want = ref.select(p["q"], means, p["table"], p["lengths"], 16, top)
        assert torch.equal(sel.cpu(), want)
        got = kiln.selected_attention(**p, selected=sel)
        torch.testing.assert_close(got.double().cpu(), ref.attention(**p, selected=want), **tolerance(act))


def test_unused_rows_are_zeros():
    p = ref.problem(gen(4), draft=40, lengths=(20, 0), cache=torch.bfloat16, device="cuda")
    p["parents"][0, 7] = 9          # follows a later token
    p["parents"][0, 20] = -5
    p["parents"][1, 0] = 0          # follows itself: every token of the sequence that leads to it is unused
    for t in (p["k"], p["v"]):
        t[0, 7] = math.nan
        t[1, 0] = math.inf
    got = check(p)
    assert (got[0, 7] == 0).all() and (got[0, 20] == 0).all() and (got[1, 0] == 0).all()


@pytest.mark.parametrize("cache,act", TYPES, ids=IDS)
def test_what_is_masked_does_not_reach(cache, act):
    p = ref.problem(gen(5), draft=6, lengths=(37, 16), cache=cache, act=act, spare=3, device="cuda")
    used = torch.zeros(len(p["k_pages"]), 16, dtype=torch.bool)
    for s, n in enumerate((37, 16)):
        for t in range(n):
            used[p["table"][s, t // 16].cpu(), t % 16] = True
    for pages in (p["k_pages"], p["v_pages"]):
        pages[(~used).nonzero(as_tuple=True)[0].cuda(), :, (~used).nonzero(as_tuple=True)[1].cuda()] = math.nan
    p["parents"] = torch.tensor([[-1, 0, 0, 1, 2, 4], [-1, -1, -1, -1, -1, -1]], dtype=torch.int32, device="cuda")
    p["v"][0, 1, 0, 3] = math.inf      # reaches tokens 1 and 3 of the first sequence alone
    p["v"][0, 4, 1] = math.nan         # tokens 4, 5
    p["k"][1, 2] = math.nan            # token 2 of the second
    got = check(p)
    assert torch.isfinite(got[0, [0, 2]]).all() and torch.isfinite(got[1, [0, 1, 3, 4, 5]]).all()


@pytest.mark.parametrize("cache,act", TYPES, ids=IDS)
def test_scores_far_apart(cache, act):
    # a weight of one and others of zero; large scores of both signs
    p = ref.problem(gen(6), lengths=(70, 33), cache=cache, act=act, device="cuda")
    p["q"] *= 30
    got = kiln.tree_attention(**p)
    want = ref.attention(**p)
    # scores up to 2^10: half a step of one is 2^-14, a weight's relative error; times 2 * 6
    tol = dict(rtol=torch.finfo(act).eps / 2, atol=2 * 6 * (2 ** -13 + (0 if act == torch.float32 else torch.finfo(act).eps / 2)))
    torch.testing.assert_close(got.double().cpu(), want, **tol)


def test_tables_that_name_no_page():
    p = ref.problem(gen(7), lengths=(100, 64), cache=torch.float16, device="cuda")
    p["table"][0, 2] = -1
    p["table"][0, 3] = len(p["k_pages"])
    p["table"][1, 0] = 2 ** 31 - 1
    check(p)
    p["lengths"][0] = 10 ** 6        # beyond the table: what the table has
    p["lengths"][1] = -3
    check(p)


def test_lists_that_do_not_ascend():
    p = ref.problem(gen(8), draft=1, heads=2, kv=1, lengths=(200, 90), device="cuda")
    sel = torch.tensor([[3, 3, 1, 5, 4, 99, -1, 2], [0, -1, 0, 5, 6, 5, 5, 7]], dtype=torch.int32, device="cuda")
    sel = sel.view(2, 1, 1, 8)
    got = kiln.selected_attention(**p, selected=sel)
    torch.testing.assert_close(got.double().cpu(), ref.attention(**p, selected=sel), **tolerance(torch.float32))


def test_select_ties_and_odd_scores():
    g = gen(9)
    q = torch.randn(1, 2, 4, 64, generator=g).cuda()
    means = torch.randn(600, 2, 64, generator=g).cuda()
    table = torch.randint(0, 40, (1, 600), generator=g).to(torch.int32).cuda()   # pages named many times: ties
    means[3, 0] = math.nan
    means[4, 1] = math.inf
    means[5] = -math.inf
    means[7] = 0.0
    table[0, 11] = -1
    for length in (1, 16, 17, 600 * 16, 599 * 16 + 1, 5000):
        lengths = torch.tensor([length], dtype=torch.int32, device="cuda")
        for top in (1, 3, 64, 599, 601):
            got = kiln.select_pages(q, means, table, lengths, page_size=16, pages=top)
            assert torch.equal(got.cpu(), ref.select(q, means, table, lengths, 16, top)), (length, top)


@pytest.mark.parametrize("cache,act", TYPES + [(torch.float32, torch.float16), (torch.float16, torch.bfloat16)])
@pytest.mark.parametrize("layers,dim,page", [(1, 64, 16), (3, 80, 32), (2, 256, 64), (1, 8, 1024)])
def test_append(cache, act, layers, dim, page):
    g = gen(dim)
    batch, n, kv, pages = 4, 45, 3, 24
    k_pages = torch.randn(layers, pages, kv, page, dim, generator=g).to(cache).cuda()
    v_pages = torch.randn(layers, pages, kv, page, dim, generator=g).to(cache).cuda()
    means = torch.randn(layers, pages, kv, dim, generator=g).cuda()
    table = torch.randperm(pages, generator=g).to(torch.int32).view(4, 6).cuda()
    table[3, 1] = -1
    lengths = torch.tensor([0, page - 1, 2 * page + 3, page - 5], dtype=torch.int32, device="cuda")
    k = torch.randn(layers, batch, n, kv, dim, generator=g).to(act).cuda()
    v = torch.randn(layers, batch, n, kv, dim, generator=g).to(act).cuda()
    rows = torch.full((batch, 20), -1, dtype=torch.int32)
    rows[0] = torch.arange(20) * 2
    rows[1, :7] = torch.tensor([3, 3, 44, 0, 1, -1, 9])     # ends at the sixth
    rows[3, :9] = torch.arange(9)
    for r in (None, rows.cuda()):
        mine = [t.clone() for t in (k_pages, v_pages, means)]
        kiln.cache_append(k, v, mine[0], mine[1], table, lengths, rows=r, k_means=mine[2])
        want = ref.append(k, v, k_pages, v_pages, table, lengths, r, means)
        assert torch.equal(mine[0].cpu(), want[0]) and torch.equal(mine[1].cpu(), want[1])
        # sums of at most 1024 values below 6 in fp32: each addition off by 2^-24 of a sum below 2^8
        torch.testing.assert_close(mine[2].double().cpu(), want[2], rtol=0, atol=1024 * 2 ** -16 / page * 2 ** -8 + 1e-5)
        without = [t.clone() for t in (k_pages, v_pages)]
        kiln.cache_append(k, v, *without, table, lengths, rows=r)
        assert torch.equal(without[0].cpu(), want[0]) and torch.equal(without[1].cpu(), want[1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.int8])
@pytest.mark.parametrize("shape", [(1, 9, 1, 16, 8), (3, 700, 2, 16, 64), (2, 40, 3, 64, 128)])
def test_copy_pages(dtype, shape):
    g = gen(1)
    pool = torch.randint(-100, 100, shape, generator=g).to(dtype).cuda()
    flat = torch.randint(-100, 100, (shape[1], 4), generator=g).to(torch.int32).cuda()
    order = torch.randperm(shape[1], generator=g).tolist()
    half = shape[1] // 2
    source, target = order[:half], order[half:2 * half]
    want, want_flat = pool.clone(), flat.clone()
    want[:, target] = pool[:, source]
    want_flat[target] = flat[source]
    kiln.copy_pages([pool, flat], source, target)
    assert torch.equal(pool, want) and torch.equal(flat, want_flat)


def test_strided_operands():
    g = gen(2)
    p = ref.problem(g, batch=2, draft=3, heads=4, kv=2, lengths=(40, 17), cache=torch.bfloat16, device="cuda")
    # token-major pages, seen as head-major
    for name in ("k_pages", "v_pages"):
        p[name] = p[name].transpose(1, 2).contiguous().transpose(1, 2)
    check(p)
    # every second page of a larger pool, columns of a wider table, rows that are no views of 16 bytes
    wide = torch.randn(2 * len(p["k_pages"]), *p["k_pages"].shape[1:], generator=g).to(torch.bfloat16).cuda()
    wide[::2] = p["k_pages"]
    p["k_pages"] = wide[::2]
    p["table"] = torch.cat([p["table"], p["table"]], 1)[:, :p["table"].shape[1]]
    q = torch.randn(2, 3, 4, 65, generator=g).cuda()
    p["q"] = q[..., 1:]
    p["k"] = p["k"].transpose(1, 2).contiguous().transpose(1, 2)
    p["v"] = p["v"].expand_as(p["v"])
    p["parents"] = p["parents"].t().contiguous().t()
    check(p)


def test_other_streams_and_graphs():
    p = ref.problem(gen(3), batch=3, draft=2, lengths=(900, 40, 0), cache=torch.bfloat16, device="cuda")
    want = kiln.tree_attention(**p)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = kiln.tree_attention(**p)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    # two graphs captured over the same operands, replayed around eager work
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(kiln.tree_attention(**p))
        graphs.append(g)
    for turn in range(4):
        p["q"].copy_(torch.randn(p["q"].shape, generator=gen(10 + turn)))
        p["lengths"].copy_(torch.tensor([900 - 200 * turn, 40 + turn, turn], dtype=torch.int32))
        want = kiln.tree_attention(**p)
        for g, out in zip(graphs, outs):
            out.zero_()
            g.replay()
            assert torch.equal(out, want)
    # same inputs, same bits
    assert all(torch.equal(kiln.tree_attention(**p), want) for _ in range(3))


def test_select_and_attend_in_a_graph():
    p = ref.problem(gen(4), batch=2, draft=3, heads=4, kv=2, lengths=(400, 90), cache=torch.float16, device="cuda")
    means = p["k_pages"].float().mean(2)

    def step():
        sel = kiln.select_pages(p["q"], means, p["table"], p["lengths"], page_size=16, pages=5)
        return kiln.selected_attention(**p, selected=sel), sel

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, sel = step()
    for turn in range(3):
        p["q"].copy_(torch.randn(p["q"].shape, generator=gen(20 + turn)))
        want = step()
        graph.replay()
        assert torch.equal(out, want[0]) and torch.equal(sel, want[1])


def test_past_32_bits():
    # pages beyond 2^31 elements
    kv, page, dim = 8, 128, 128
    pages = 2 ** 31 // (kv * page * dim) + 40
    p = ref.problem(gen(5), batch=1, draft=1, heads=8, kv=kv, dim=dim, page=page, lengths=(300,), cache=torch.bfloat16)
    far = pages - 1 - torch.arange(3)
    for name in ("k_pages", "v_pages"):
        big = torch.zeros(pages, kv, page, dim, dtype=torch.bfloat16, device="cuda")
        big[far.cuda()] = p[name][p["table"][0].long()].cuda()
        p[name] = big
    p["table"] = far.to(torch.int32).view(1, 3)
    p = {k: v.cuda() for k, v in p.items()}
    small = dict(p, k_pages=p["k_pages"][far.cuda()], v_pages=p["v_pages"][far.cuda()],
                 table=torch.arange(3, dtype=torch.int32, device="cuda").view(1, 3))
    assert torch.equal(kiln.tree_attention(**p), kiln.tree_attention(**small))
    k = torch.randn(1, 5, kv, dim, device="cuda")
    kiln.cache_append(k, k, p["k_pages"], p["v_pages"], p["table"], p["lengths"])
    assert torch.equal(p["k_pages"][far[2].item(), :, 44:49], k[0].transpose(0, 1).bfloat16())
    kiln.copy_pages([p["k_pages"]], [pages - 3], [0])
    assert torch.equal(p["k_pages"][0], p["k_pages"][pages - 3])


# -- a run of them together --------------------------------------------------------------------------


def small_stack(layers=2, d=64, nh=4):
    from models.transformer import Stack, gpt2_init_

    return gpt2_init_(Stack(layers, d, nh, 16), seed=0, std=0.1).eval()


def rows_of(stack, xs):
    """The stack over whole sequences without a cache, in 64 bits: every row's result."""
    import copy

    out = []
    for x in xs:
        model = copy.deepcopy(stack).double().cpu()
        for b in model.blocks:
            b.mask = torch.full((len(x), len(x)), -math.inf, dtype=torch.float64).triu(1)
        with torch.no_grad():
            out.append(model(x.double().cpu()))
    return out


@pytest.mark.parametrize("flags", [{}, dict(cuda_graphs=False), dict(fusion=False), dict(debug=True)], ids=str)
@pytest.mark.parametrize("top", [None, 64])
def test_decoding_with_drafted_trees(flags, top):
    """Two sequences grow by the accepted paths of drafted trees; every drafted
    row's result is that of the whole sequence along its path. The cache is
    fp32, so the tolerance is that of compiled fp32 stacks (1e-4, 1e-4 behind a
    LayerNorm of rows of size one); 64 pages are all there are."""
    from models.decoder import CachedStack

    stack = small_stack()
    g = gen(8)
    tokens, d = 5, 64
    cache = kiln.PagedCache(2, 40, 16, 4, 16, dtype=torch.float32, means=True)
    seqs = [cache.open(), cache.open()]
    prefix = [torch.zeros(0, d), torch.zeros(0, d)]
    compiled = None
    for step in range(12):
        x = torch.randn(2, tokens, d, generator=g)
        back = 1 + (torch.randn(2, tokens, generator=g).abs() * 2).long()
        parents = (torch.arange(tokens) - back).clamp(min=-1).to(torch.int32)
        table, lengths = cache.batch(seqs, columns=8)
        args = (x.view(-1, d).cuda(), cache.k, cache.v, table, lengths, parents.cuda()) + ((cache.means,) if top else ())
        if compiled is None:
            # (the examples' rows lie where the model is; the cache lies where it is)
            compiled = kiln.compile(CachedStack(stack, tokens, top), (args[0].cpu(), *args[1:]), device="cuda", **flags)
            assert not compiled.report.lowering["cuda_graphs"]     # the cache is read in place
        y, *kv = compiled(*args)
        paths = []
        for s in range(2):
            path, _ = ref.see(parents[s].tolist(), tokens)
            for i in range(tokens):
                rows = torch.cat([prefix[s], x[s, path[i]]])
                want = rows_of(stack, [rows])[0][-1]
                torch.testing.assert_close(y[s * tokens + i].double().cpu(), want, rtol=1e-4, atol=1e-4)
            accepted = path[int(torch.randint(tokens, (1,), generator=g))].nonzero()[:, 0].tolist()
            paths.append(accepted)
            prefix[s] = torch.cat([prefix[s], x[s, accepted]])
        cache.append(seqs, torch.stack(kv[:2]), torch.stack(kv[2:]), rows=paths)
        if step == 5:      # the second sequence goes on from a copy of the first
            cache.free(seqs[1])
            seqs[1], = cache.fork(seqs[0])
            prefix[1] = prefix[0]
        if step == 8:
            cache.compact()
    assert cache.length(seqs[0]) == len(prefix[0])


@pytest.mark.parametrize("cache,precision,tol", [
    (torch.bfloat16, "fp32", 1e-4), (torch.float16, "fp32", 1e-4),
    # bf16 products: half a step of 2^-8 in q, the weights and each product's operands, some ten of them in a row
    (torch.bfloat16, "bf16", 10 * 2 ** -8)])
def test_compiled_block_precisions(cache, precision, tol):
    from models.decoder import CachedBlock

    stack = small_stack(1, 128, 2)
    p = ref.problem(gen(9), batch=3, draft=4, heads=2, kv=2, dim=64, lengths=(500, 33, 0), cache=cache, device="cuda")
    x = torch.randn(12, 128, generator=gen(10)).cuda()
    args = (x, p["k_pages"], p["v_pages"], p["table"], p["lengths"], p["parents"])
    got = kiln.compile(CachedBlock(stack.blocks[0], 4), (x.cpu(), *args[1:]), device="cuda", matmul_precision=precision)(*args)[0]
    from test_paged import block_reference

    want = block_reference(stack.blocks[0].cpu(), x.cpu(), *[t.cpu() for t in args[1:]], 4)[0]
    torch.testing.assert_close(got.double().cpu(), want, rtol=tol, atol=tol)


def test_compiled_block_in_a_callers_graph():
    from models.decoder import CachedBlock

    block = small_stack(1).blocks[0]
    p = ref.problem(gen(11), batch=2, draft=3, heads=4, kv=4, dim=16, lengths=(90, 20), cache=torch.bfloat16, device="cuda")
    args = (torch.randn(6, 64, device="cuda"), p["k_pages"], p["v_pages"], p["table"], p["lengths"], p["parents"])
    compiled = kiln.compile(CachedBlock(block, 3), (args[0].cpu(), *args[1:]), device="cuda")
    compiled(*args)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = compiled(*args)
    for turn in range(4):
        args[0].copy_(torch.randn(6, 64, generator=gen(turn)))
        args[4].copy_(torch.tensor([90 - turn * 30, turn], dtype=torch.int32))
        want = compiled(*args)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_torch_compile_backend(monkeypatch):
    from models.decoder import CachedBlock

    monkeypatch.setenv("KILN_STRICT", "1")
    block = small_stack(1).blocks[0].cuda()
    p = ref.problem(gen(12), batch=2, draft=3, heads=4, kv=4, dim=16, lengths=(90, 20), cache=torch.float16, device="cuda")
    args = (torch.randn(6, 64, device="cuda"), p["k_pages"], p["v_pages"], p["table"], p["lengths"], p["parents"])
    model = CachedBlock(block, 3)
    before = kiln.stats["compiled"]
    with torch.no_grad():
        got = torch.compile(model, backend=kiln.backend, dynamic=False)(*args)
        want = model(*args)          # the operators as functions, torch's other kernels
    assert kiln.stats["compiled"] > before
    for a, b in zip(got, want):
        torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-5)


def test_another_cards_tensors_are_refused():
    p = ref.problem(gen(13), device="cuda")
    with pytest.raises(ValueError):
        kiln.tree_attention(**dict(p, table=p["table"].cpu()))
    with pytest.raises(NotImplementedError):
        kiln.tree_attention(**{k: v.cpu() for k, v in p.items()})


@pytest.mark.parametrize("cache,act", TYPES[1:], ids=IDS[1:])
@pytest.mark.parametrize("dim,group", [(64, 1), (80, 2), (128, 1), (128, 4)])
def test_many_rows(cache, act, dim, group):
    # 48 rows of an item and more share tiles: one block, two, several; ranges and whole items
    draft = 70
    for lengths, page in (((1100, 0), 16), ((63, 130), 128)):
        p = ref.problem(gen(group), draft=draft, heads=group * 2, kv=2, dim=dim, lengths=lengths, page=page, cache=cache,
                        act=act, device="cuda")
        used = torch.zeros(len(p["k_pages"]), page, dtype=torch.bool)
        for s, n in enumerate(lengths):
            for t in range(n):
                used[p["table"][s, t // page].cpu(), t % page] = True
        at = [x.cuda() for x in (~used).nonzero(as_tuple=True)]
        for pages in (p["k_pages"], p["v_pages"]):
            pages[at[0], :, at[1]] = math.nan      # a page's unwritten slots
        p["parents"][0, 40] = 50                    # unused
        p["v"][1, 33, 0, 5] = -math.inf
        p["v"][1, 66, 1] = math.nan
        check(p)
        p["parents"] = None
        check({k: v for k, v in p.items() if k != "parents"})


@pytest.mark.parametrize("heads", [96, 320])
def test_many_heads_of_a_picked_page(heads):
    p = ref.problem(gen(14), draft=2, heads=heads, kv=1, lengths=(700, 90), cache=torch.float16, act=torch.float16, dim=128,
                    device="cuda")
    sel = torch.tensor([[0, 3, 4, -1], [1, 2, 5, 43]], dtype=torch.int32, device="cuda").view(1, 2, 1, 4).expand(2, 2, 1, 4)
    got = kiln.selected_attention(**p, selected=sel)
    torch.testing.assert_close(got.double().cpu(), ref.attention(**p, selected=sel.cpu()), **tolerance(torch.float16))


def test_many_sequences():
    p = ref.problem(gen(15), batch=1500, draft=1, heads=1, kv=1, lengths=[i % 40 for i in range(1500)], cache=torch.bfloat16,
                    columns=200, device="cuda")
    check(p)
