"""The paged cache on the CPU: refusals, the book-keeping of kiln.PagedCache,
the way from a model to a plan, and the meaning of the operators
(KILN_HIP_INTERPRET=1: the library's CPU meaning) against their definitions.

Tolerance of the CPU meaning: it works in 64 bits and rounds its fp32 or 16-bit
result once, so half a step of the result; a compiled block adds the fp32
rounding of its other kernels' results, held to the 1e-4 / 1e-5 of the GPU
tests."""

import random

import numpy as np
import pytest
import torch

import kiln
import paged_reference as ref
from kiln.frontend.fx_import import Unsupported, import_exported
from kiln.hip import lib as kl
from kiln.ir import interpret, parse, verify
from models.decoder import CachedBlock, CachedStack
from models.transformer import Block, Stack, gpt2_init_


@pytest.fixture()
def interpreting(monkeypatch):
    monkeypatch.setenv("KILN_HIP_INTERPRET", "1")


def gen(seed=0):
    return torch.Generator().manual_seed(seed)


TYPES = [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.float16, torch.float16)]


@pytest.mark.parametrize("cache,act", TYPES)
def test_meaning(interpreting, cache, act):
    p = ref.problem(gen(), batch=3, draft=7, heads=6, kv=2, lengths=(70, 0, 33), cache=cache, act=act)
    p["parents"][0, 3] = 5     # unused, and what follows it
    p["table"][0, 1] = 99      # no such page
    means = p["k_pages"].float().mean(2)
    tol = dict(rtol=torch.finfo(act).eps / 2, atol=1e-7 if act == torch.float32 else 2 ** -25)
    torch.testing.assert_close(kiln.tree_attention(**p).double(), ref.attention(**p), **tol)
    torch.testing.assert_close(kiln.tree_attention(**dict(p, parents=None), scale=0.3).double(),
                               ref.attention(**dict(p, parents=None), scale=0.3), **tol)
    for top in (1, 3, 9):
        sel = kiln.select_pages(p["q"], means, p["table"], p["lengths"], page_size=16, pages=top)
        assert torch.equal(sel, ref.select(p["q"], means, p["table"], p["lengths"], 16, top))
        torch.testing.assert_close(kiln.selected_attention(**p, selected=sel).double(),
                                   ref.attention(**p, selected=sel), **tol)


@pytest.mark.parametrize("cache,act", TYPES)
def test_append_meaning(interpreting, cache, act):
    g = gen(1)
    k_pages = torch.randn(2, 9, 3, 16, 8, generator=g).to(cache)
    v_pages = torch.randn(2, 9, 3, 16, 8, generator=g).to(cache)
    means = torch.randn(2, 9, 3, 8, generator=g)
    table = torch.tensor([[4, 2, -1], [0, 7, 8]], dtype=torch.int32)
    lengths = torch.tensor([14, 31], dtype=torch.int32)
    k, v = (torch.randn(2, 2, 21, 3, 8, generator=g).to(act) for _ in range(2))
    rows = torch.tensor([[0, 2, 2, 20, 5], [9, 1, -1, 3, 4]], dtype=torch.int32)
    for r in (None, rows):
        want = ref.append(k, v, k_pages, v_pages, table, lengths, r, means)
        got = [t.clone() for t in (k_pages, v_pages, means)]
        kiln.cache_append(k, v, got[0], got[1], table, lengths, rows=r, k_means=got[2])
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        torch.testing.assert_close(got[2].double(), want[2], rtol=2 ** -24, atol=0)


# -- refusals -----------------------------------------------------------------------------------


def operands(**more):
    return ref.problem(gen(), **more)


@pytest.mark.parametrize("change,error", [
    (dict(q=torch.zeros(2, 3, 4, 64, dtype=torch.bfloat16)), TypeError),       # 16-bit q over fp32 pages
    (dict(q=torch.zeros(2, 3, 4, 64, dtype=torch.float64)), TypeError),
    (dict(q=torch.zeros(2, 3, 4, 32)), ValueError),
    (dict(q=torch.zeros(2, 3, 64)), ValueError),
    (dict(q=torch.zeros(2, 3, 3, 64)), ValueError),                             # 3 heads over 2
    (dict(k=torch.zeros(2, 2, 2, 64)), ValueError),
    (dict(v=torch.zeros(2, 3, 2, 64, dtype=torch.float16)), TypeError),
    (dict(v_pages=torch.zeros(1, 2, 16, 64)), ValueError),
    (dict(table=torch.zeros(2, 3, dtype=torch.int64)), TypeError),
    (dict(table=torch.zeros(1, 3, dtype=torch.int32)), ValueError),
    (dict(table=None), ValueError),
    (dict(lengths=torch.zeros(3, dtype=torch.int32)), ValueError),
    (dict(lengths=torch.zeros(2)), TypeError),
    (dict(parents=torch.zeros(2, 2, dtype=torch.int32)), ValueError),
    (dict(q=torch.zeros(2, 3, 4, 64, requires_grad=True)), NotImplementedError),
])
def test_refusals_of_attention(interpreting, change, error):
    with pytest.raises(error):
        kiln.tree_attention(**dict(operands(), **change))


def test_refusals_of_sizes(interpreting):
    for sizes in (dict(dim=12), dict(dim=10), dict(dim=12, cache=torch.float16), dict(dim=20, cache=torch.bfloat16, act=torch.bfloat16),
                  dict(dim=264), dict(page=8, lengths=(20, 9)), dict(page=48, lengths=(20, 9)),
                  dict(draft=257), dict(page=2048, lengths=(20, 9))):
        with pytest.raises(NotImplementedError):
            kiln.tree_attention(**operands(**sizes))
    for dim in (4, 10, 260):
        pages, k = torch.zeros(4, 2, 16, dim, dtype=torch.float16), torch.zeros(1, 3, 2, dim)
        with pytest.raises(NotImplementedError):
            kiln.cache_append(k, k, pages, pages.clone(), torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))
        with pytest.raises(NotImplementedError):
            kiln.select_pages(k, pages.float().mean(2), torch.zeros(1, 2, dtype=torch.int32),
                              torch.zeros(1, dtype=torch.int32), page_size=16, pages=1)
    p = operands()
    with pytest.raises(ValueError):    # token rows that do not lie together
        kiln.tree_attention(**dict(p, k_pages=p["k_pages"].transpose(2, 3).contiguous().transpose(2, 3)))
    with pytest.raises(ValueError):    # pages that do not start at 16 bytes
        flat = torch.zeros(p["k_pages"].numel() + 1)
        kiln.tree_attention(**dict(p, k_pages=flat[1:].view(p["k_pages"].shape)))
    with pytest.raises(ValueError):
        kiln.selected_attention(**p, selected=torch.zeros(2, 3, 4, 1, dtype=torch.int32))
    with pytest.raises(TypeError):
        kiln.selected_attention(**p, selected=None)
    with pytest.raises(ValueError):
        kiln.select_pages(p["q"], torch.zeros(5, 2, 64), p["table"], p["lengths"], page_size=16, pages=0)
    with pytest.raises(TypeError):
        kiln.select_pages(p["q"], torch.zeros(5, 2, 64, dtype=torch.float64), p["table"], p["lengths"], page_size=16, pages=1)


def test_no_cpu_path():
    with pytest.raises(NotImplementedError):
        kiln.tree_attention(**operands())
    with pytest.raises(NotImplementedError):
        kiln.copy_pages([torch.zeros(4, 8)], [0], [1])


def test_empty_calls(interpreting):
    p = operands()
    none = {n: t[:0] if n not in ("k_pages", "v_pages") else t for n, t in p.items()}
    assert kiln.tree_attention(**none).shape == (0, 3, 4, 64)
    no_tokens = dict(p, q=p["q"][:, :0], k=p["k"][:, :0], v=p["v"][:, :0], parents=p["parents"][:, :0])
    assert kiln.tree_attention(**no_tokens).shape == (2, 0, 4, 64)
    no_columns = dict(p, table=p["table"][:, :0])
    torch.testing.assert_close(kiln.tree_attention(**no_columns).double(), ref.attention(**no_columns))


def test_refusals_of_append_and_copy(interpreting):
    k_pages = torch.zeros(4, 2, 16, 8)
    k = torch.zeros(1, 3, 2, 8)
    table, lengths = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    for args, more, error in (
            ((k, k[:, :2], k_pages, k_pages, table, lengths), {}, ValueError),
            ((k, k.half(), k_pages, k_pages, table, lengths), {}, TypeError),
            ((k, k, k_pages, k_pages[:3], table, lengths), {}, ValueError),
            ((k, k, k_pages, k_pages, table, lengths.long()), {}, TypeError),
            ((k, k, k_pages, k_pages, table, lengths), dict(rows=torch.zeros(2, 3, dtype=torch.int32)), ValueError),
            ((k, k, k_pages, k_pages, table, lengths), dict(k_means=torch.zeros(4, 2, 16)), ValueError),
            ((k.unsqueeze(0), k, k_pages, k_pages, table, lengths), {}, ValueError)):
        with pytest.raises(error):
            kiln.cache_append(*args, **more)
    pool = torch.arange(40.0).view(10, 4)
    for source, target in (([0], [0]), ([0, 1], [2, 2]), ([0, 1], [1, 2]), ([10], [0]), ([0], [-1])):
        with pytest.raises(ValueError):
            kiln.copy_pages([pool], source, target)
    with pytest.raises(ValueError):
        kiln.copy_pages([pool], [0, 1], [2])
    with pytest.raises(ValueError):
        kiln.copy_pages([pool, pool[:5]], [0], [1])
    with pytest.raises(ValueError):
        kiln.copy_pages([pool.t()], [0], [1])
    with pytest.raises(TypeError):
        kiln.copy_pages([pool], ["a"], [1])
    with pytest.raises(ValueError):
        kiln.copy_pages([pool], [2 ** 32], [1])
    assert torch.equal(pool, torch.arange(40.0).view(10, 4))
    kiln.copy_pages([pool], [1, 3, 1], [0, 2, 9])
    assert torch.equal(pool[[0, 2, 9]], torch.arange(40.0).view(10, 4)[[1, 3, 1]])


# -- kiln.PagedCache ---------------------------------------------------------------------------------


class Model:
    """What the cache should hold: per sequence a list of (k, v) tokens."""

    def __init__(self):
        self.tokens = {}


def content(cache, seq):
    n, ps = cache.length(seq), cache.page_size
    if not n:
        return cache.k[:, 0, :, :0], cache.v[:, 0, :, :0]
    pages = list(cache.pages_of(seq))
    k, v = (t[:, pages].permute(0, 2, 1, 3, 4).flatten(2, 3)[:, :, :n] for t in (cache.k, cache.v))
    return k, v     # [layers, heads, tokens, dim]


def consistent(cache):
    refs = [0] * cache.pages
    for seq, pages in cache._pages.items():
        assert len(pages) == -(-cache._length[seq] // cache.page_size)
        for p in pages:
            refs[p] += 1
    assert refs == cache._refs
    assert sorted(cache._free) == [p for p in range(cache.pages) if not refs[p]]


@pytest.mark.parametrize("seed", range(6))
def test_cache_keeps_what_it_is_given(interpreting, seed):
    rng, g = random.Random(seed), gen(seed)
    cache = kiln.PagedCache(2, 24, 16, 2, 8, dtype=torch.bfloat16, means=True)
    held = {}
    for step in range(60):
        seqs = list(held)
        what = rng.choice(["open", "append", "append", "append", "fork", "free", "truncate", "compact"])
        if what == "open" and len(seqs) < 6:
            held[cache.open()] = (torch.zeros(2, 2, 0, 8), torch.zeros(2, 2, 0, 8))
        elif what == "append" and seqs:
            some = rng.sample(seqs, rng.randint(1, len(seqs)))
            n = rng.randint(1, 20)
            k, v = (torch.randn(2, len(some), n, 2, 8, generator=g) for _ in range(2))
            rows = None if rng.random() < 0.5 else [sorted(rng.sample(range(n), rng.randint(0, n))) for _ in some]
            before = (cache.k.clone(), dict(cache._length), {s: cache.pages_of(s) for s in seqs}, cache.free_pages)
            try:
                cache.append(some, k, v, rows=rows)
            except MemoryError:
                assert torch.equal(cache.k, before[0]) and cache._length == before[1]
                assert {s: cache.pages_of(s) for s in seqs} == before[2] and cache.free_pages == before[3]
                consistent(cache)
                cache.free(some[0])
                del held[some[0]]
                continue
            for i, s in enumerate(some):
                path = list(range(n)) if rows is None else rows[i]
                held[s] = tuple(torch.cat([old, t[:, i, path].transpose(1, 2).bfloat16().float()], 2)
                                for old, t in zip(held[s], (k, v)))
        elif what == "fork" and seqs:
            s = rng.choice(seqs)
            for new in cache.fork(s, rng.randint(0, 2)):
                held[new] = held[s]
        elif what == "free" and seqs:
            s = rng.choice(seqs)
            cache.free(s)
            del held[s]
        elif what == "truncate" and seqs:
            s = rng.choice(seqs)
            n = rng.randint(0, cache.length(s))
            cache.truncate(s, n)
            held[s] = tuple(t[:, :, :n] for t in held[s])
        elif what == "compact":
            used = cache.compact()
            assert used == cache.pages - cache.free_pages
            assert all(p < used for s in held for p in cache.pages_of(s))
        consistent(cache)
        for s, want in held.items():
            for got, w in zip(content(cache, s), want):
                assert torch.equal(got.float(), w)
            # the means of full pages (a truncated page's is stale until the next append, and is not read)
            for j, p in enumerate(cache.pages_of(s)[:cache.length(s) // 16]):
                torch.testing.assert_close(cache.means[:, p], cache.k[:, p].float().mean(2), rtol=1e-5, atol=1e-6)
    table, lengths = cache.batch(list(held))
    assert table.dtype == lengths.dtype == torch.int32 and lengths.tolist() == [cache.length(s) for s in held]
    for row, s in zip(table.tolist(), held):
        assert tuple(x for x in row if x >= 0) == cache.pages_of(s)


def test_cache_refusals(interpreting):
    for bad, error in ((dict(page_size=24), NotImplementedError), (dict(dim=12), NotImplementedError), (dict(pages=0), ValueError),
                       (dict(dtype=torch.float64), TypeError)):
        with pytest.raises(error):
            kiln.PagedCache(**dict(dict(layers=1, pages=4, page_size=16, kv_heads=2, dim=8), **bad))
    cache = kiln.PagedCache(1, 4, 16, 2, 8, dtype=torch.float32)
    a = cache.open()
    k = torch.zeros(1, 1, 5, 2, 8)
    for call in (lambda: cache.append([a, a], k, k), lambda: cache.append([a], k, k, rows=[[5]]),
                 lambda: cache.append([a], k, k, rows=[[0], [1]]), lambda: cache.append([a], k[0], k[0]),
                 lambda: cache.free(7), lambda: cache.truncate(a, 1), lambda: cache.batch([a, 9]),
                 lambda: cache.fork(a, -1)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(MemoryError):
        cache.append([a], k.expand(1, 1, 5, 2, 8).repeat(1, 1, 14, 1, 1), k.repeat(1, 1, 14, 1, 1))
    assert cache.free_pages == 4 and cache.length(a) == 0
    cache.free(a)
    with pytest.raises(ValueError):
        cache.length(a)


# -- through kiln.compile -----------------------------------------------------------------------------------


def block_operands(seed=0, seqs=2, tokens=3, d=64, nh=4, cache=torch.bfloat16, lengths=(40, 17)):
    p = ref.problem(gen(seed), batch=seqs, draft=tokens, heads=nh, kv=nh, dim=d // nh, lengths=lengths, cache=cache)
    x = torch.randn(seqs * tokens, d, generator=gen(seed + 1))
    return x, p["k_pages"], p["v_pages"], p["table"], p["lengths"], p["parents"]


def block_reference(block, x, k_pages, v_pages, table, lengths, parents, tokens, top=None, k_means=None):
    """The cached block in 64 bits."""
    b = block.double()
    x = x.double()
    shape = (len(x) // tokens, tokens, b.nh, x.shape[1] // b.nh)
    with torch.no_grad():
        q, k, v = (y.view(shape) for y in b.c_attn(b.ln1(x)).split(x.shape[1], 1))
        sel = None if top is None else ref.select(q, k_means, table, lengths, k_pages.shape[2], top)
        # (keys are rounded to the cache's type from fp32 values)
        y = ref.attention(q, k.float(), v.float(), k_pages, v_pages, table, lengths, parents, sel)
        x = x + b.c_proj(y.reshape(x.shape))
        out = x + b.proj(torch.nn.functional.gelu(b.fc(b.ln2(x)), approximate="tanh"))
    block.float()
    return out, k, v


@pytest.mark.parametrize("cache", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("fusion", [True, False], ids=["fused", "unfused"])
def test_compiled_block(interpreting, cache, fusion):
    block = gpt2_init_(Block(64, 4, 16), seed=0).eval()
    args = block_operands(cache=cache)
    compiled = kiln.compile(CachedBlock(block, 3), args, device="cuda", fusion=fusion)
    assert compiled.report.lowering["families"]["paged"] == 1
    for got, want in zip(compiled(*args), block_reference(block, *args, 3)):
        torch.testing.assert_close(got.double(), want, rtol=1e-4, atol=1e-5)
    # the cache is read in place, at each call anew
    args[1].mul_(-0.5)
    args[4][0] = 31
    torch.testing.assert_close(compiled(*args)[0].double(), block_reference(block, *args, 3)[0], rtol=1e-4, atol=1e-5)


def test_compiled_block_with_picked_pages(interpreting):
    block = gpt2_init_(Block(64, 4, 16), seed=1).eval()
    args = block_operands(lengths=(90, 33))
    means = args[1].float().mean(2)
    compiled = kiln.compile(CachedBlock(block, 3, top=2), (*args, means), device="cuda")
    assert compiled.report.lowering["families"]["paged"] == 2
    for got, want in zip(compiled(*args, means), block_reference(block, *args, 3, 2, means)):
        torch.testing.assert_close(got.double(), want, rtol=1e-4, atol=1e-5)


def test_compiled_stack_reads_layers_of_one_pool(interpreting):
    stack = gpt2_init_(Stack(2, 64, 4, 16), seed=2).eval()
    x, k_pages, v_pages, table, lengths, parents = block_operands()
    k_pages, v_pages = (torch.stack([t, t.flip(0)]) for t in (k_pages, v_pages))
    model = CachedStack(stack, 3)
    compiled = kiln.compile(model, (x, k_pages, v_pages, table, lengths, parents), device="cuda")
    y, *kv = compiled(x, k_pages, v_pages, table, lengths, parents)
    h, want_kv = x, []
    for i, b in enumerate(stack.blocks):
        h, k, v = block_reference(b, h.float(), k_pages[i], v_pages[i], table, lengths, parents, 3)
        want_kv.append((k, v))
    want = torch.nn.functional.layer_norm(h, (64,), stack.ln_f.weight.double(), stack.ln_f.bias.double())
    torch.testing.assert_close(y.double(), want.detach(), rtol=1e-4, atol=1e-4)   # (LayerNorm of small rows)


def test_list_of_pages_as_a_result(interpreting):
    x = torch.randn(2, 3, 4, 64, generator=gen())
    p = operands(lengths=(100, 40))
    means = p["k_pages"].mean(2)

    def fn(q, means, table, lengths):
        return kiln.select_pages(q * 2.0, means, table, lengths, page_size=16, pages=3)

    compiled = kiln.compile(fn, (x, means, p["table"], p["lengths"]), device="cuda")
    got = compiled(x, means, p["table"], p["lengths"])
    assert got.dtype == torch.int32
    assert torch.equal(got, ref.select(x * 2, means, p["table"], p["lengths"], 16, 3))


def imported(model, args):
    return import_exported(torch.export.export(model, args).run_decompositions())


@pytest.mark.parametrize("top", [None, 2])
def test_graph_text_and_meaning(top):
    block = gpt2_init_(Block(32, 2, 16), seed=3).eval()
    args = block_operands(d=32, nh=2)
    args += (args[1].float().mean(2),) if top else ()
    g = imported(CachedBlock(block, 3, top), args)
    verify(g)
    again = parse(str(g))
    assert str(again) == str(g)
    out = interpret(g, *[t.float().numpy() if t.dtype == torch.bfloat16 else t.numpy() for t in args])
    want = block_reference(block, *args[:6], 3, top, args[6] if top else None)
    np.testing.assert_allclose(out[0], want[0].numpy(), rtol=1e-4, atol=1e-5)


def test_calls_that_a_plan_refuses(interpreting):
    block = gpt2_init_(Block(64, 4, 16), seed=0).eval()
    args = list(block_operands())
    compiled = kiln.compile(CachedBlock(block, 3), tuple(args), device="cuda")
    for i, bad in ((1, args[1].float()), (3, args[3].long()), (1, args[1].transpose(2, 3).contiguous().transpose(2, 3)),
                   (1, args[1][:-1])):
        with pytest.raises(ValueError):
            compiled(*args[:i], bad, *args[i + 1:])


def test_models_that_are_refused():
    block = Block(64, 4, 16).eval()
    args = block_operands()

    class Holds(torch.nn.Module):     # the cache as buffers would be frozen into the plan
        def __init__(self):
            super().__init__()
            self.inner = CachedBlock(block, 3)
            self.register_buffer("pages", args[1].float())

        def forward(self, x, table, lengths, parents):
            return self.inner(x, self.pages, self.pages, table, lengths, parents)

    with pytest.raises(Unsupported):
        imported(Holds(), (args[0], *args[3:]))

    class Sixteen(torch.nn.Module):   # bf16 activations
        def forward(self, q, k_pages, table, lengths):
            return kiln.tree_attention(q, q, q, k_pages, k_pages, table, lengths)

    with pytest.raises(Unsupported):
        imported(Sixteen(), (torch.zeros(2, 3, 4, 16, dtype=torch.bfloat16), *args[1:2], *args[3:5]))

    class Adds(torch.nn.Module):      # arithmetic on the pages
        def forward(self, q, k_pages, table, lengths):
            return kiln.tree_attention(q, q, q, k_pages + k_pages, k_pages, table, lengths)

    with pytest.raises(Unsupported):
        imported(Adds(), (torch.zeros(2, 3, 4, 16), *args[1:2], *args[3:5]))

    class Appends(torch.nn.Module):
        def forward(self, k, k_pages, table, lengths):
            kiln.cache_append(k, k, k_pages, k_pages, table, lengths)
            return k

    with pytest.raises(Exception, match="between"):
        imported(Appends(), (torch.zeros(2, 3, 4, 16), *args[1:2], *args[3:5]))
    # without such operators nothing has changed
    with pytest.raises(Unsupported, match="only float32"):
        imported(torch.nn.ReLU(), (torch.zeros(3, dtype=torch.float16),))


# -- the C entries -----------------------------------------------------------------------------------------


def test_c_entries_refuse(interpreting):
    lib = kl.load()
    op = kl.Paged()
    assert lib.kh_paged_run(None, None, 0, None) == kl.ERR_INVALID
    assert lib.kh_paged_run(op, None, 0, None) == kl.ERR_INVALID
    assert lib.kh_cache_append(None, None) == kl.ERR_INVALID
    assert lib.kh_cache_copy(None, 1, 4, None, None, 0, None) == kl.ERR_INVALID
    launch = kl.LaunchDesc()
    launch.family = kl.FAM_PAGED
    launch.variant = 9
    handle = kl.ctypes.c_void_p()
    assert lib.kh_plan_create(kl.ctypes.byref(launch), 1, kl.ctypes.byref(handle)) == kl.ERR_INVALID
    launch.variant = kl.PAGED_ATTENTION
    launch.n_refs = 8
    launch.cfg[4] = 11
    assert lib.kh_plan_create(kl.ctypes.byref(launch), 1, kl.ctypes.byref(handle)) == kl.ERR_INVALID


def test_strides_past_32_bits_are_refused(interpreting):
    op = kl.Paged(kl.PAGED_ATTENTION, 1, 1, 1, 1, 64, 1024, 4, 2, 0, kl.TYPE_F32, kl.TYPE_F32, 0, 1.0)
    size = kl.ctypes.c_size_t()
    lib = kl.load()
    assert lib.kh_paged_workspace_bytes(op, size) == kl.OK
    op.kp_t = 2 ** 20
    assert lib.kh_paged_workspace_bytes(op, size) == kl.ERR_UNSUPPORTED
    op.kp_t, op.k_n = 0, 2 ** 24
    assert lib.kh_paged_workspace_bytes(op, size) == kl.ERR_UNSUPPORTED
    op.k_n, op.pages = 0, 2 ** 27
    assert lib.kh_paged_workspace_bytes(op, size) == kl.ERR_UNSUPPORTED
    op.pages, op.batch, op.width = 4, 4096, 2 ** 20
    assert lib.kh_paged_workspace_bytes(op, size) == kl.ERR_UNSUPPORTED


def test_a_cache_whose_append_fails_is_as_before(interpreting, monkeypatch):
    from kiln.hip import paged

    cache = kiln.PagedCache(1, 6, 16, 2, 8, dtype=torch.float32)
    a = cache.open()
    k = torch.randn(1, 1, 20, 2, 8)
    cache.append([a], k, k)
    b, = cache.fork(a)

    def fails(*args, **more):
        raise RuntimeError("a launch failed")

    for name in ("copy_pages", "cache_append"):
        with monkeypatch.context() as m:
            m.setattr(paged, name, fails)
            with pytest.raises(RuntimeError):
                cache.append([b], k, k)
        consistent(cache)
        assert cache.length(b) == 20 and cache.pages_of(b) == cache.pages_of(a) and cache.free_pages == 4
    cache.append([b], k, k)
    consistent(cache)
    assert torch.equal(content(cache, b)[0][:, :, :20], content(cache, a)[0])
