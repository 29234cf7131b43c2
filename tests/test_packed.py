"""The 4-bit cache, dense reads and windows on the CPU: the meaning of the
operators (KILN_HIP_INTERPRET=1: the library's CPU meaning) against their
definitions, refusals, and kiln.PagedCache over 4-bit pages.

What 4 bits hold is exact in both, so pages, codes and values are compared for
equality; the CPU meaning of attention works in 64 bits and rounds its result
once: half a step of it, and 2^-24 of the largest value for what exp and the
sums differ by."""

import math
import random

import numpy as np
import pytest
import torch

import kiln
import packed_reference as ref
from kiln.frontend.fx_import import Unsupported, import_exported
from kiln.hip import lib as kl
from kiln.ir import interpret, parse, verify
from models.decoder import CachedBlock
from models.transformer import Block, gpt2_init_

FP4 = torch.float4_e2m1fn_x2


@pytest.fixture()
def interpreting(monkeypatch):
    monkeypatch.setenv("KILN_HIP_INTERPRET", "1")


def gen(seed=0):
    return torch.Generator().manual_seed(seed)


def half(act):
    return dict(rtol=torch.finfo(act).eps / 2, atol=12 * 2 ** -24)


def blocks():
    """Rows of 32 with every code, ties, the borders of a scale, the smallest and the largest, zeros, signs."""
    g = gen(3)
    rows = [torch.randn(32, generator=g) * 10.0 ** (i - 12) for i in range(26)]
    grid = torch.tensor([0, .25, .5, .75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 6.999])
    both = torch.cat([grid, -grid])
    rows += [both, both * 2.0 ** 100, both * 2.0 ** -100, both * 2.0 ** -124, both * 2.0 ** -130, torch.nextafter(both, both * 2),
             torch.nextafter(both, both * 0), torch.zeros(32), -torch.zeros(32)]
    for top in (7.0, 6.9999995, 3.5, 4.0, torch.finfo(torch.float32).max, 2.0 ** -126, 2.0 ** -149, 1.75 * 2.0 ** -124):
        row = torch.linspace(-0.9, 0.9, 32) * top
        row[7] = top
        rows.append(row)
    return torch.stack(rows)


@pytest.mark.parametrize("act", [torch.float32, torch.bfloat16, torch.float16])
def test_blocks(interpreting, act):
    x = blocks().to(act)
    n = len(x)
    k = x.view(1, n, 1, 32)
    kp, vp = (torch.zeros(-(-n // 16), 1, 16, 17, dtype=torch.uint8) for _ in "kv")
    table = torch.arange(len(kp), dtype=torch.int32)[None]
    zero = torch.zeros(1, dtype=torch.int32)
    kiln.cache_append(k, k.flip(1), kp, vp, table, zero)
    got_k, got_v = kiln.cache_read(kp, vp, table, zero, zero + n, tokens=n, dtype=torch.float32)
    want = ref.rounded(x)
    # (fp32 activations may be past fp16's range: infinite there, a NaN block)
    assert torch.equal(got_k.double().view(n, 32).nan_to_num(nan=99.0), want.nan_to_num(nan=99.0))
    assert torch.equal(got_v.double().view(n, 32).flip(0).nan_to_num(nan=99.0), want.nan_to_num(nan=99.0))


def test_half_a_step():
    # 1/6 of the block's largest at the most: half a step of the top binade is 1, of a largest of 6 (below 7: 1/7 beyond)
    x = blocks()
    x = x[(x.abs().amax(1) > 2.0 ** -120) & torch.isfinite(x).all(1)]
    assert bool(((ref.rounded(x) - x.double()).abs() <= x.double().abs().amax(1, keepdim=True) / 3.5).all())


@pytest.mark.parametrize("dim,page", [(32, 16), (96, 32), (256, 16)])
def test_append_and_read(interpreting, dim, page):
    g = gen(dim)
    k_pages, v_pages = (ref.fast_pack(torch.randn(2, 9, 3, page, dim, generator=g), keys) for keys in (True, False))
    means = torch.randn(2, 9, 3, dim, generator=g)
    table = torch.tensor([[4, 2, -1], [0, 7, 8], [1, 3, 99]], dtype=torch.int32)
    lengths = torch.tensor([page - 2, 2 * page - 1, 5], dtype=torch.int32)
    k, v = (torch.randn(2, 3, 21, 3, dim, generator=g) for _ in range(2))
    rows = torch.tensor([[0, 2, 2, 20, 5], [9, 1, -1, 3, 4], [-1, 0, 0, 0, 0]], dtype=torch.int32)
    for r in (None, rows):
        want = ref.append(k, v, k_pages, v_pages, table, lengths, r, means)
        got = [t.clone() for t in (k_pages, v_pages, means)]
        kiln.cache_append(k, v, got[0], got[1], table, lengths, rows=r, k_means=got[2])
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        torch.testing.assert_close(got[2].double(), want[2], rtol=2 ** -24, atol=0)
    starts = torch.tensor([0, -3, page + 1], dtype=torch.int32)
    ends = torch.tensor([page + 3, 10 ** 6, page + 9], dtype=torch.int32)
    for dtype in (None, torch.float32, torch.float16):
        got = kiln.cache_read(k_pages, v_pages, table, starts, ends, tokens=3 * page + 7, dtype=dtype)
        for a, b in zip(got, ref.read(k_pages, v_pages, table, starts, ends, 3 * page + 7)):
            assert a.dtype == (dtype or torch.bfloat16) and torch.equal(a.double(), b)
    one = kiln.cache_read(k_pages[1], v_pages[1], table, starts, ends, tokens=5)
    assert torch.equal(one[0], kiln.cache_read(k_pages, v_pages, table, starts, ends, tokens=5)[0][1])


def test_reads_as_a_sequence_grows(interpreting, monkeypatch):
    # one kept form, whatever the number of tokens: a long-lived program's reads push no other operator's out
    from kiln.hip import paged

    monkeypatch.setattr(paged, "_forms", {})
    p = ref.problem(gen(6), cache=torch.bfloat16, lengths=(40, 17))
    starts = torch.zeros(2, dtype=torch.int32)
    pages = p["k_pages"], p["v_pages"]
    want = ref.read(*(t[None] for t in pages), p["table"], starts, p["lengths"], 45)
    for n in [*range(1, 46), 0, 7]:
        got = kiln.cache_read(*pages, p["table"], starts, p["lengths"], tokens=n)
        assert all(torch.equal(a.double(), b[0, :, :n]) for a, b in zip(got, want))
    assert len(paged._forms) == 1
    for n in (-1, 2 ** 31):
        with pytest.raises(ValueError):
            kiln.cache_read(*pages, p["table"], starts, p["lengths"], tokens=n)


@pytest.mark.parametrize("cache", [torch.float32, torch.bfloat16, torch.float16])
def test_read_of_other_types(interpreting, cache):
    g = gen(5)
    k_pages, v_pages = (torch.randn(2, 9, 3, 16, 40, generator=g).to(cache) for _ in "kv")
    table = torch.tensor([[4, 2, -1], [0, 7, 8]], dtype=torch.int32)
    starts, ends = torch.tensor([3, 0], dtype=torch.int32), torch.tensor([40, 17], dtype=torch.int32)
    for dtype in (None, torch.float32, torch.bfloat16, torch.float16):
        got = kiln.cache_read(k_pages, v_pages, table, starts, ends, tokens=50, dtype=dtype)
        for a, b in zip(got, ref.read(k_pages, v_pages, table, starts, ends, 50)):
            assert torch.equal(a, b.to(dtype or cache))


ACTS = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dim", [32, 64, 96])
def test_attention_meaning(interpreting, act, dim):
    p = ref.problem(gen(), act=act, batch=3, draft=7, heads=6, kv=2, lengths=(70, 0, 33), dim=dim)
    p["parents"][0, 3] = 5     # unused, and what follows it
    p["table"][0, 1] = 99      # no such page
    torch.testing.assert_close(kiln.tree_attention(**p).double(), ref.attention(**p), **half(act))
    for window, sinks in ((1, 0), (3, 0), (5, 2), (40, 17), (1000, 3)):
        more = dict(window=window, sinks=sinks)
        torch.testing.assert_close(kiln.tree_attention(**p, **more).double(), ref.attention(**p, **more), **half(act))
        chain = dict(p, parents=None, **more)
        torch.testing.assert_close(kiln.tree_attention(**chain).double(), ref.attention(**chain), **half(act))
    sel = torch.tensor([[0, 2, 4], [1, 1, 3]], dtype=torch.int32).expand(3, 7, 2, 3).contiguous()
    torch.testing.assert_close(kiln.selected_attention(**p, selected=sel).double(), ref.attention(**p, selected=sel), **half(act))


@pytest.mark.parametrize("cache,act", [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.float16, torch.float16)])
def test_window_meaning(interpreting, cache, act):
    p = ref.problem(gen(2), cache=cache, act=act, batch=3, draft=9, heads=4, kv=2, lengths=(70, 0, 33))
    for window, sinks in ((1, 0), (1, 100), (4, 1), (17, 0), (33, 20), (2 ** 31 - 1, 2 ** 31 - 1)):
        more = dict(window=window, sinks=sinks)
        torch.testing.assert_close(kiln.tree_attention(**p, **more).double(), ref.attention(**p, **more), **half(act))
    whole = kiln.tree_attention(**p)
    assert torch.equal(kiln.tree_attention(**p, window=80), whole)      # (a window that holds everything)


# -- refusals -----------------------------------------------------------------------------------


def test_refusals(interpreting):
    p = ref.problem(gen())
    for change, more, error in (
            (dict(k_pages=p["k_pages"][..., :33].contiguous(), v_pages=p["v_pages"][..., :33].contiguous()), {}, ValueError),
            (dict(k_pages=p["k_pages"][..., :0], v_pages=p["v_pages"][..., :0]), {}, ValueError),
            (dict(q=p["q"].double()), {}, TypeError),
            (dict(k=p["k"].half()), {}, TypeError),
            (dict(v_pages=p["v_pages"].float()), {}, TypeError),
            (dict(k_pages=p["k_pages"].transpose(2, 3).contiguous().transpose(2, 3)), {}, ValueError),
            ({}, dict(window=0), ValueError),
            ({}, dict(window=-1), ValueError),
            ({}, dict(sinks=4), ValueError),
            ({}, dict(window=4, sinks=-1), ValueError),
            ({}, dict(window=2.5), TypeError),
            ({}, dict(window=3, sinks=1.0), TypeError),
            ({}, dict(window=2 ** 31), ValueError)):
        with pytest.raises(error):
            kiln.tree_attention(**dict(p, **change), **more)
    with pytest.raises(NotImplementedError):     # 288 dimensions
        kiln.tree_attention(**ref.problem(gen(), dim=288))
    with pytest.raises(ValueError):
        torch.ops.kiln.paged_attention(*[p[n] for n in ("q", "k", "v", "k_pages", "v_pages", "table", "lengths", "parents")],
                                       torch.zeros(2, 3, 2, 1, dtype=torch.int32), 1.0, 4, 0)
    zero = torch.zeros(2, dtype=torch.int32)
    read = dict(k_pages=p["k_pages"], v_pages=p["v_pages"], table=p["table"], starts=zero, ends=zero + 4, tokens=4)
    for change, error in ((dict(tokens=-1), ValueError), (dict(dtype=torch.float64), TypeError), (dict(dtype=torch.uint8), TypeError),
                          (dict(starts=zero.long()), TypeError), (dict(ends=zero[:1]), ValueError), (dict(table=None), ValueError),
                          (dict(v_pages=p["v_pages"][:1]), ValueError), (dict(k_pages=None), TypeError),
                          (dict(k_pages=p["k_pages"][:, :, :15], v_pages=p["v_pages"][:, :, :15]), (ValueError, NotImplementedError))):
        with pytest.raises(error):
            kiln.cache_read(**dict(read, **change))
    with pytest.raises(NotImplementedError):
        kiln.cache_read(**dict(read, k_pages=torch.zeros(2, 1, 16, 64, requires_grad=True), v_pages=torch.zeros(2, 1, 16, 64)))
    assert kiln.cache_read(**dict(read, tokens=0))[0].shape == (2, 0, 2, 64)
    with pytest.raises(NotImplementedError):     # 48 dimensions: no block ends there
        kiln.PagedCache(1, 4, 16, 1, 48, dtype=FP4)


@pytest.mark.parametrize("cache,act", [(0, 0), (1, 0), (1, 1), (2, 2)], ids=["fp32", "bf16-fp32", "bf16", "fp16"])
def test_limits_of_other_caches(interpreting, cache, act):
    # 32-bit counts of tiles: keys / 32 and 10 more a sequence, times the kv heads and their row blocks. What ranges
    # over 4-bit pages count beside their tiles narrows 4-bit calls alone.
    lib, size = kl.load(), kl.ctypes.c_size_t()

    def of(cache, act, tokens, batch=4096, heads=32, kv_heads=8, variant=kl.PAGED_ATTENTION):
        op = kl.Paged(variant, batch, 1, heads, kv_heads, 128, 64, 1000, tokens // 64, 0, cache, act, 0, 1.0)
        return lib.kh_paged_workspace_bytes(op, size)

    # (keys / 32 + 10) * 4096 * 8 <= (2^31 - 1) / 2: up to 32757 tiles
    assert of(cache, act, 32757 // 2 * 64) == kl.OK
    assert of(cache, act, 32757 // 2 * 64 + 64) == kl.ERR_UNSUPPORTED
    assert of(kl.TYPE_MX4, act, 32757 // 2 * 64) == kl.ERR_UNSUPPORTED
    assert of(kl.TYPE_MX4, act, (32757 - 12) // 2 * 64) == kl.OK
    # (keys / 32 + 9) * batch <= 2^31 - 1
    for tokens, want in ((524278 * 32, kl.OK), (524280 * 32, kl.ERR_UNSUPPORTED)):
        assert of(kl.TYPE_F32, act, tokens, batch=4096, heads=1, kv_heads=1, variant=kl.PAGED_SELECT) == want


def test_transforms_are_refused(interpreting):
    from torch.autograd import forward_ad

    p = ref.problem(gen(), cache=torch.float32)
    zero = torch.zeros(2, dtype=torch.int32)
    read = dict(k_pages=p["k_pages"], v_pages=p["v_pages"], table=p["table"], starts=zero, ends=zero + 4, tokens=4)
    kiln.cache_read(**read)                # (the form of a call that is known does not pass either)
    for name in ("k_pages", "table", "ends"):
        with pytest.raises(RuntimeError):
            torch.vmap(lambda t: kiln.cache_read(**dict(read, **{name: t})))(torch.stack([read[name]] * 2))
    with pytest.raises(NotImplementedError):
        torch.func.jvp(lambda t: kiln.cache_read(**dict(read, k_pages=t))[0], (p["k_pages"],), (p["k_pages"],))
    with forward_ad.dual_level(), pytest.raises(NotImplementedError):
        kiln.cache_read(**dict(read, v_pages=forward_ad.make_dual(p["v_pages"], p["v_pages"])))
    with pytest.raises(NotImplementedError):
        torch.func.grad(lambda t: kiln.cache_read(**dict(read, k_pages=t))[0].sum())(p["k_pages"])


def test_no_cpu_path():
    p = ref.problem(gen())
    with pytest.raises(NotImplementedError):
        kiln.tree_attention(**p, window=4)
    with pytest.raises(NotImplementedError):
        kiln.cache_read(p["k_pages"], p["v_pages"], p["table"], p["lengths"], p["lengths"], tokens=3)


# -- kiln.PagedCache ---------------------------------------------------------------------------------


def test_packed_cache_keeps_what_it_is_given(interpreting):
    rng, g = random.Random(1), gen(1)
    cache = kiln.PagedCache(2, 24, 16, 2, 32, dtype=FP4, means=True)
    assert cache.k.dtype == torch.uint8 and cache.k.shape == (2, 24, 2, 16, 17)
    held = {}
    for step in range(30):
        seqs = list(held)
        what = rng.choice(["open", "append", "append", "fork", "truncate", "compact"])
        if what == "open" and len(seqs) < 4:
            held[cache.open()] = (torch.zeros(2, 0, 2, 32), torch.zeros(2, 0, 2, 32))
        elif what == "append" and seqs:
            some = rng.sample(seqs, rng.randint(1, len(seqs)))
            k, v = (torch.randn(2, len(some), 3, 2, 32, generator=g) for _ in range(2))
            cache.append(some, k, v)
            for i, s in enumerate(some):
                held[s] = tuple(torch.cat([old, ref.rounded(t[:, i]).float()], 1) for old, t in zip(held[s], (k, v)))
        elif what == "fork" and seqs and len(seqs) < 6:
            s = rng.choice(seqs)
            held[cache.fork(s)[0]] = held[s]
        elif what == "truncate" and seqs:
            s = rng.choice(seqs)
            n = rng.randint(0, cache.length(s))
            cache.truncate(s, n)
            held[s] = tuple(t[:, :n] for t in held[s])
        elif what == "compact":
            cache.compact()
        if held:
            for got, i in zip(cache.read(list(held), dtype=torch.float32), (0, 1)):
                for j, s in enumerate(held):
                    assert torch.equal(got[:, j, :cache.length(s)], held[s][i])
                    assert not got[:, j, cache.length(s):].any()
    # into another cache, of another type
    seqs = list(held)
    other = kiln.PagedCache(2, 24, 32, 2, 32, dtype=torch.bfloat16)
    there = [other.open() for _ in seqs]
    k, v = cache.read(seqs)
    other.append(there, k, v, rows=[list(range(cache.length(s))) for s in seqs])
    for a, b in zip(other.read(there), (k, v)):
        assert torch.equal(a, b)


def test_release(interpreting):
    cache = kiln.PagedCache(1, 12, 16, 1, 32, dtype=torch.float32)
    a = cache.open()
    k = torch.randn(1, 1, 100, 1, 32, generator=gen(8))
    cache.append([a], k, k)
    whole = cache.read([a])[0]
    cache.release(a, window=101)                  # everything is in it
    assert cache.free_pages == 5 and -1 not in cache.pages_of(a)
    cache.release(a, window=40, sinks=17)         # keys 61 .. and 0 .. 16 are seen: page 2 alone is not
    assert [p < 0 for p in cache.pages_of(a)] == [False, False, True, False, False, False, False] and cache.free_pages == 6
    assert cache.length(a) == 100
    got = cache.read([a])[0]
    assert torch.equal(got[:, :, :32], whole[:, :, :32]) and not got[:, :, 32:48].any() and torch.equal(got[:, :, 48:], whole[:, :, 48:])
    q = torch.randn(1, 3, 2, 32, generator=gen(9))
    new = torch.randn(1, 3, 1, 32, generator=gen(10))
    fresh = kiln.PagedCache(1, 12, 16, 1, 32, dtype=torch.float32)
    b = fresh.open()
    fresh.append([b], k, k)
    for more in (dict(window=40, sinks=17), dict(window=3)):
        out = [kiln.tree_attention(q, new, new, c.k[0], c.v[0], *c.batch([s]), **more) for c, s in ((cache, a), (fresh, b))]
        assert torch.equal(*out)
    (c,) = cache.fork(a)                          # shares what is left
    cache.release(c, window=20)
    assert [p < 0 for p in cache.pages_of(c)] == [True] * 5 + [False, False] and cache.free_pages == 6
    for length in (1, 99):
        with pytest.raises(ValueError):
            cache.truncate(a, length)
    cache.append([a], k[:, :, :30], k[:, :, :30])
    cache.truncate(a, 100)
    cache.append([a, c], k[:, :, :2].expand(1, 2, 2, 1, 32), k[:, :, :2].expand(1, 2, 2, 1, 32))
    assert cache.length(a) == cache.length(c) == 102
    assert torch.equal(cache.read([a])[0][:, :, 100:], k[:, :, :2])
    used = cache.compact()
    assert used == 12 - cache.free_pages and all(p < used for s in (a, c) for p in cache.pages_of(s))
    assert torch.equal(cache.read([a])[0][:, :, 48:100], whole[:, :, 48:])
    cache.free(a)
    cache.truncate(c, 0)
    assert cache.free_pages == 12 and cache.read([c])[0].shape[2] == 0
    cache.append([c], k, k)                       # (anew: nothing of it is gone)
    cache.truncate(c, 3)
    for window, sinks in ((0, 0), (-1, 0), (3, -1)):
        with pytest.raises(ValueError):
            cache.release(c, window=window, sinks=sinks)
    with pytest.raises(ValueError):
        cache.release(99, window=3)
    cache.release(c, window=1)
    assert cache.free_pages == 11                 # (the last page has room)


# -- through kiln.compile -----------------------------------------------------------------------------------


class WindowBlock(CachedBlock):
    """The cached block whose attention has a window."""

    def __init__(self, block, tokens, window=None, sinks=0):
        super().__init__(block, tokens)
        self.window, self.sinks = window, sinks

    def attend(self, x, k_pages, v_pages, table, lengths, parents, k_means):
        b = self.block
        split = (len(x) // self.tokens, self.tokens, b.nh, x.shape[-1] // b.nh)
        q, k, v = (y.view(split) for y in b.c_attn(b.ln1(x)).split(x.shape[-1], dim=1))
        y = kiln.tree_attention(q, k, v, k_pages, v_pages, table, lengths, parents, window=self.window, sinks=self.sinks)
        return x + b.c_proj(y.reshape(x.shape)), k, v


def block_operands(cache=torch.uint8, seed=0, seqs=2, tokens=3, d=64, nh=2, lengths=(40, 17)):
    p = ref.problem(gen(seed), cache=cache, batch=seqs, draft=tokens, heads=nh, kv=nh, dim=d // nh, lengths=lengths)
    x = torch.randn(seqs * tokens, d, generator=gen(seed + 1))
    return x, p["k_pages"], p["v_pages"], p["table"], p["lengths"], p["parents"]


def block_reference(block, x, k_pages, v_pages, table, lengths, parents, tokens, **more):
    """(the block's result, its keys and values) in 64 bits. (4-bit blocks have steps: a comparison is one only where
    the keys and values round alike, steps_agree.)"""
    b = block.double()
    x = x.cpu().double()
    shape = (len(x) // tokens, tokens, b.nh, x.shape[1] // b.nh)
    with torch.no_grad():
        q, k, v = (y.view(shape) for y in b.c_attn(b.ln1(x)).split(x.shape[1], 1))
        y = ref.attention(q, k.float(), v.float(), k_pages, v_pages, table, lengths, parents, **more)
        x = x + b.c_proj(y.reshape(x.shape))
        out = x + b.proj(torch.nn.functional.gelu(b.fc(b.ln2(x)), approximate="tanh"))
    block.float()
    return out, k, v


def steps_agree(got, want):
    """Whether fp32 keys or values round to 4 bits as their 64-bit ones do."""
    return torch.equal(ref.rounded(got.cpu().float()), ref.rounded(want.float()))


@pytest.mark.parametrize("cache", [torch.uint8, torch.float32, torch.bfloat16])
@pytest.mark.parametrize("window,sinks", [(None, 0), (20, 3), (2, 0)])
def test_compiled_block(interpreting, cache, window, sinks):
    block = gpt2_init_(Block(64, 2, 16), seed=0).eval()
    args = block_operands(cache=cache)
    model = WindowBlock(block, 3, window, sinks)
    compiled = kiln.compile(model, args, device="cuda")
    assert compiled.report.lowering["families"]["paged"] == 1
    got, want = compiled(*args), block_reference(block, *args, 3, window=window, sinks=sinks)
    assert cache != torch.uint8 or all(steps_agree(a, b) for a, b in zip(got[1:], want[1:]))
    for a, b in zip(got, want):
        torch.testing.assert_close(a.double(), b, rtol=1e-4, atol=1e-5)
    args[4][0] = 31       # the cache is read in place, at each call anew
    torch.testing.assert_close(compiled(*args)[0].double(), block_reference(block, *args, 3, window=window, sinks=sinks)[0], rtol=1e-4, atol=1e-5)


@pytest.mark.parametrize("window,sinks", [(None, 0), (5, 2)])
def test_graph_text_and_meaning(window, sinks):
    block = gpt2_init_(Block(64, 2, 16), seed=3).eval()
    args = block_operands()
    g = import_exported(torch.export.export(WindowBlock(block, 3, window, sinks), args).run_decompositions())
    verify(g)
    assert str(parse(str(g))) == str(g)
    out = interpret(g, *[t.numpy() for t in args])
    want = block_reference(block, *args, 3, window=window, sinks=sinks)
    assert all(steps_agree(torch.tensor(a), b) for a, b in zip(out[1:], want[1:]))
    np.testing.assert_allclose(out[0], want[0].numpy(), rtol=1e-4, atol=1e-5)


class Views(torch.nn.Module):
    """Attention over what a view makes of the pages."""

    def __init__(self, view):
        super().__init__()
        self.view = view

    def forward(self, q, k, v, k_pages, v_pages, table, lengths):
        return kiln.tree_attention(q, k, v, self.view(k_pages), self.view(v_pages), table, lengths)


def view_operands(dim, make):
    p = ref.problem(gen(21), dim=64, lengths=(40, 17))
    q, k, v = (p[name][..., :dim].contiguous() for name in ("q", "k", "v"))
    return q, k, v, make(p["k_pages"]), make(p["v_pages"]), p["table"], p["lengths"]


@pytest.mark.parametrize("view,make", [
    (lambda x: x[1], lambda x: torch.stack([x.flip(0), x])),              # a layer
    (lambda x: x[1:], lambda x: torch.cat([x[:1], x])),                   # pages
    (lambda x: x[:, 1:3], lambda x: torch.cat([x, x], 1)),                # heads
    (lambda x: x[:, :, :16], lambda x: torch.cat([x, x], 2)),             # whole tokens, in a block all the same
    (lambda x: x.view(-1, 2, 16, 34), lambda x: x.reshape(-1))])
def test_views_of_pages_in_a_model(interpreting, view, make):
    args = view_operands(64, make)
    got = kiln.compile(Views(view), args, device="cuda")(*args)
    want = ref.attention(*args[:3], *(view(t).contiguous() for t in args[3:5]), *args[5:])
    torch.testing.assert_close(got.double(), want, rtol=1e-4, atol=1e-5)


@pytest.mark.parametrize("view,make,dim", [
    (lambda x: x[..., :17], lambda x: x, 32),                             # the first half of each token's bytes
    (lambda x: x[:, :, ::2], lambda x: x.repeat_interleave(2, 2), 64),    # every other token's
    (lambda x: x.transpose(1, 2), lambda x: x.transpose(1, 2).contiguous(), 64)])
def test_views_that_part_a_heads_bytes(interpreting, view, make, dim):
    # 4-bit pages of a head are one block of bytes: no view of it is another page
    args = view_operands(dim, make)
    with pytest.raises(NotImplementedError, match="4-bit pages of a head"):
        kiln.compile(Views(view), args, device="cuda")


def test_models_that_are_refused():
    args = block_operands()

    class Adds(torch.nn.Module):      # arithmetic on the pages' bytes
        def forward(self, q, k_pages, table, lengths):
            return kiln.tree_attention(q, q, q, k_pages + k_pages, k_pages, table, lengths)

    class Verifies(torch.nn.Module):  # between steps, not in them
        def forward(self, q, k_pages, table, lengths):
            y = kiln.tree_attention(q, q, q, k_pages, k_pages, table, lengths)
            return kiln.verify_tokens(table, y[:, :, 0].softmax(-1), y[:, :, 0, 0])[0]

    q = torch.zeros(2, 3, 2, 32)
    for model in (Adds(), Verifies()):
        with pytest.raises(Unsupported):
            import_exported(torch.export.export(model, (q, *args[1:2], *args[3:5])).run_decompositions())
