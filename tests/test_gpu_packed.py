"""The 4-bit cache, dense reads and windows on the GPU against their definitions
in 64 bits.

Pages, codes and dense values are compared for equality. Attention: the bounds
of test_gpu_paged.py, whose scores and weights are made the same way: values of
4-bit pages are bf16 ones, at most 6 times the largest of a block's new tokens
here (|v| < 6 of normal inputs), and products of fp32 activations take three
bf16 parts, of fp16 ones two (16 bits of q, which has 11, and of the weights):
1e-4 for fp32, and half a step of the result and of each weight more for 16-bit
activations."""

import math

import pytest
import torch

import kiln
import packed_reference as ref
import test_packed

pytestmark = pytest.mark.gpu

ACTS = [torch.float32, torch.bfloat16, torch.float16]
CACHES = [(torch.uint8, a) for a in ACTS] + [(torch.float32, torch.float32), (torch.bfloat16, torch.float32),
                                             (torch.float16, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16)]
IDS = ["fp4-fp32", "fp4-bf16", "fp4-fp16", "fp32", "bf16-fp32", "fp16-fp32", "bf16", "fp16"]


def gen(seed=0):
    return torch.Generator().manual_seed(seed)


def tolerance(act):
    if act == torch.float32:
        return dict(rtol=0.0, atol=1e-4)
    half = torch.finfo(act).eps / 2
    return dict(rtol=half, atol=1e-4 + 2 * 6 * half)


def check(p, selected=None, **more):
    if selected is None:
        got = kiln.tree_attention(**p, **more)
    else:
        got = kiln.selected_attention(**p, selected=selected)
        more = dict(selected=selected)
    want = ref.attention(**p, **more)
    assert got.dtype == p["q"].dtype and got.shape == p["q"].shape
    torch.testing.assert_close(got.double().cpu(), want, equal_nan=True, **tolerance(got.dtype))
    return got


@pytest.mark.parametrize("act", ACTS)
def test_blocks(act):
    x = test_packed.blocks().to(act)
    n = len(x)
    k = x.view(1, n, 1, 32).cuda()
    kp, vp = (torch.zeros(-(-n // 16), 1, 16, 17, dtype=torch.uint8, device="cuda") for _ in "kv")
    table = torch.arange(len(kp), dtype=torch.int32, device="cuda")[None]
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    kiln.cache_append(k, k.flip(1), kp, vp, table, zero)
    want = torch.zeros(len(kp) * 16, 32, dtype=act)
    want[:n] = x
    assert torch.equal(kp[:, 0].cpu().flatten()[:n // 16 * 272], ref.pack(want.view(-1, 16, 32), True).flatten()[:n // 16 * 272])
    got_k, got_v = kiln.cache_read(kp, vp, table, zero, zero + n, tokens=n, dtype=torch.float32)
    want = ref.rounded(x)
    assert torch.equal(got_k.cpu().double().view(n, 32).nan_to_num(nan=99.0), want.nan_to_num(nan=99.0))
    assert torch.equal(got_v.cpu().double().view(n, 32).flip(0).nan_to_num(nan=99.0), want.nan_to_num(nan=99.0))


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("layers,dim,page", [(1, 32, 16), (3, 96, 32), (2, 256, 64), (1, 64, 1024)])
def test_append_and_read(act, layers, dim, page):
    g = gen(dim)
    batch, n, kv, pages = 4, 45, 3, 24
    k_pages, v_pages = (torch.cat([ref.fast_pack(torch.randn(pages, kv, page, dim, generator=g), keys)[None] for _ in range(layers)])
                        .cuda() for keys in (True, False))
    means = torch.randn(layers, pages, kv, dim, generator=g).cuda()
    table = torch.randperm(pages, generator=g).to(torch.int32).view(4, 6).cuda()
    table[3, 1] = -1
    lengths = torch.tensor([0, page - 1, 2 * page + 3, page - 5], dtype=torch.int32, device="cuda")
    k = torch.randn(layers, batch, n, kv, dim, generator=g).to(act).cuda()
    v = torch.randn(layers, batch, n, kv, dim, generator=g).to(act).cuda()
    k[0, 0, 2, 1, 5] = math.inf
    v[0, 1, 3, 0, 31] = math.nan
    rows = torch.full((batch, 20), -1, dtype=torch.int32)
    rows[0] = torch.arange(20) * 2
    rows[1, :7] = torch.tensor([3, 3, 44, 0, 1, -1, 9])     # ends at the sixth
    rows[3, :9] = torch.arange(9)
    for r in (None, rows.cuda()):
        mine = [t.clone() for t in (k_pages, v_pages, means)]
        kiln.cache_append(k, v, mine[0], mine[1], table, lengths, rows=r, k_means=mine[2])
        want = ref.append(k, v, k_pages, v_pages, table, lengths, r, means)
        assert torch.equal(mine[0].cpu(), want[0]) and torch.equal(mine[1].cpu(), want[1])
        # sums of at most 1024 values below 8 in fp32: each addition off by 2^-24 of a sum below 2^8
        torch.testing.assert_close(mine[2].double().cpu(), want[2], rtol=0, atol=1024 * 2 ** -16 / page * 2 ** -8 + 1e-5, equal_nan=True)
        without = [t.clone() for t in (k_pages, v_pages)]
        kiln.cache_append(k, v, *without, table, lengths, rows=r)
        assert torch.equal(without[0].cpu(), want[0]) and torch.equal(without[1].cpu(), want[1])
    starts = torch.tensor([0, -3, page + 1, 2 * page - 2], dtype=torch.int32, device="cuda")
    ends = torch.tensor([page + 3, 10 ** 6, page + 9, 5], dtype=torch.int32, device="cuda")
    for dtype in ACTS:
        got = kiln.cache_read(*mine[:2], table, starts, ends, tokens=page + 70, dtype=dtype)
        for a, b in zip(got, ref.read(*mine[:2], table, starts, ends, page + 70)):
            assert torch.equal(a.cpu().nan_to_num(nan=99.0), b.to(dtype).nan_to_num(nan=99.0))


@pytest.mark.parametrize("cache", ACTS)
def test_read_of_other_types(cache):
    g = gen(5)
    k_pages, v_pages = (torch.randn(2, 9, 3, 16, 40, generator=g).to(cache).cuda() for _ in "kv")
    table = torch.tensor([[4, 2, -1], [0, 7, 8]], dtype=torch.int32, device="cuda")
    starts, ends = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([3, 0], [40, 17]))
    for dtype in (None, *ACTS):
        got = kiln.cache_read(k_pages, v_pages, table, starts, ends, tokens=50, dtype=dtype)
        for a, b in zip(got, ref.read(k_pages, v_pages, table, starts, ends, 50)):
            assert torch.equal(a.cpu(), b.to(dtype or cache))


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 160, 256])
@pytest.mark.parametrize("heads,kv,draft", [(2, 2, 1), (4, 1, 5), (6, 2, 33)])
def test_types_heads_dims(act, dim, heads, kv, draft):
    check(ref.problem(gen(dim), act=act, draft=draft, heads=heads, kv=kv, dim=dim, device="cuda"))


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("page", [16, 32, 128, 1024])
@pytest.mark.parametrize("lengths", [(0, 0), (1, 0), (15, 16), (31, 33), (129, 1000), (2049, 5)], ids=str)
def test_lengths_and_pages(act, page, lengths):
    check(ref.problem(gen(page), act=act, lengths=lengths, page=page, device="cuda"))


@pytest.mark.parametrize("draft", [1, 2, 31, 32, 33, 64, 100, 256])
@pytest.mark.parametrize("tree", [True, False], ids=["tree", "chain"])
def test_drafts(draft, tree):
    check(ref.problem(gen(draft), draft=draft, heads=3, kv=1, tree=tree, lengths=(50, 0), device="cuda"))
    check(ref.problem(gen(draft), act=torch.float16, draft=draft, heads=8, kv=1, tree=tree, lengths=(50, 3), dim=128, device="cuda"))


def test_many_tokens_of_wide_heads():
    # the new tokens' own pages in the LDS, at their largest
    for act in ACTS:
        check(ref.problem(gen(13), act=act, draft=256, heads=1, kv=1, dim=256, lengths=(50, 400), device="cuda"))


@pytest.mark.parametrize("act", ACTS)
def test_long_and_ragged(act):
    # ranges that end inside an item, and many items in one range
    lengths = (5000, 0, 1, 700, 33, 2600, 64, 16)
    check(ref.problem(gen(1), act=act, batch=8, draft=2, heads=4, kv=2, lengths=lengths, device="cuda"))
    check(ref.problem(gen(2), act=act, batch=40, draft=1, heads=2, kv=1, lengths=[7 * i for i in range(40)], device="cuda"))
    check(ref.problem(gen(3), act=act, batch=3, draft=20, heads=8, kv=2, dim=128, lengths=(3000, 1111, 2), device="cuda"))


@pytest.mark.parametrize("act", ACTS)
def test_picked_pages(act):
    p = ref.problem(gen(3), act=act, batch=3, draft=5, heads=6, kv=2, lengths=(300, 0, 41), device="cuda")
    means = ref.unpack(p["k_pages"], True).mean(2).float().cuda()
    for top in (1, 7):
        check(p, selected=kiln.select_pages(p["q"], means, p["table"], p["lengths"], page_size=16, pages=top))


@pytest.mark.parametrize("act", ACTS)
def test_what_is_masked_does_not_reach(act):
    for dim in (64, 128, 256):
        p = ref.problem(gen(5), act=act, draft=6, lengths=(37, 16), spare=3, dim=dim, device="cuda")
        for s, n in enumerate((37, 16)):      # slots behind the last token: NaN blocks
            for t in range(n, -(-n // 16) * 16):
                page = int(p["table"][s, t // 16])
                for pages, keys in ((p["k_pages"], True), (p["v_pages"], False)):
                    for d in range(0, dim, 32):
                        at = ref.places(t % 16, d, dim, 16, keys)[1]
                        pages[page].view(2, -1)[:, at] = 253 + t % 3
        p["parents"] = torch.tensor([[-1, 0, 0, 1, 2, 4], [-1, -1, -1, -1, -1, -1]], dtype=torch.int32, device="cuda")
        p["v"][0, 1, 0, 3] = math.inf      # reaches tokens 1 and 3 of the first sequence alone
        p["v"][0, 4, 1] = math.nan         # tokens 4, 5
        p["k"][1, 2] = math.nan            # token 2 of the second
        got = check(p)
        assert torch.isfinite(got[0, [0, 2]]).all() and torch.isfinite(got[1, [0, 1, 3, 4, 5]]).all()
        if dim > 32:
            assert torch.isfinite(got[0, 3, 0, 32:]).all()     # (the other blocks of that value)
        p["v"][0, 1, 0, 3] = 0.0
        at = ref.places(5, 0, dim, 16, False)[1]
        p["v_pages"][int(p["table"][0, 1])].view(2, -1)[:, at] = 255   # a cached value: every row
        assert not torch.isfinite(check(p)[0, :, :, :32]).any()
        at = ref.places(5, 0, dim, 16, True)[1]
        p["k_pages"][int(p["table"][1, 0])].view(2, -1)[0, at] = 255   # a cached key: every row of its heads
        assert not torch.isfinite(check(p)[1, :, :2]).any()


def test_unused_rows_are_zeros():
    p = ref.problem(gen(4), draft=40, lengths=(20, 0), device="cuda")
    p["parents"][0, 7] = 9          # follows a later token
    p["parents"][0, 20] = -5
    p["parents"][1, 0] = 0          # follows itself: every token of the sequence that leads to it is unused
    p["k"][0, 7] = math.nan
    p["v"][1, 0] = math.inf
    for more in (dict(), dict(window=5, sinks=2)):
        got = check(p, **more)
        assert (got[0, 7] == 0).all() and (got[0, 20] == 0).all() and (got[1, 0] == 0).all()


def test_tables_that_name_no_page():
    p = ref.problem(gen(7), lengths=(100, 64), device="cuda")
    p["table"][0, 2] = -1
    p["table"][0, 3] = len(p["k_pages"])
    p["table"][1, 0] = 2 ** 31 - 1
    check(p)
    p["lengths"][0] = 10 ** 6        # beyond the table: what the table has
    p["lengths"][1] = -3
    check(p)
    check(p, window=20, sinks=3)


@pytest.mark.parametrize("act", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 96, 128])
@pytest.mark.parametrize("tree", [True, False], ids=["tree", "chain"])
def test_many_rows_over_long_caches(act, dim, tree):
    # rows that share tiles; with a window, an unused token, NaN in the cache and among the new tokens
    p = ref.problem(gen(14), act=act, batch=2, draft=26, heads=4, kv=1, dim=dim, page=64, lengths=(4700, 4200), tree=tree, device="cuda")
    check(p)
    if tree:
        p["parents"][1, 3] = 3
    p["v"][0, 25] = math.nan
    p["k"][0, 24] = math.inf
    for t in (100, 4300):                  # a value behind the window of every token, and one that some see
        at = ref.places(t % 64, 0, dim, 64, False)[1]
        p["v_pages"][int(p["table"][0, t // 64])].view(1, -1)[:, at] = 255
    got = check(p, window=4097, sinks=33)
    assert torch.isfinite(got[1]).all() and not torch.isfinite(got[0, :, :, :32]).any() and torch.isfinite(got[0, 0, :, 32:]).all()
    for t in (4300,):
        at = ref.places(t % 64, 0, dim, 64, False)[1]
        p["v_pages"][int(p["table"][0, t // 64])].view(1, -1)[:, at] = 127
    first = 4700 - 4200 + 1                # token 0's first key: the others do not see it
    at = ref.places(first % 64, 32, dim, 64, False)[1]
    p["v_pages"][int(p["table"][0, first // 64])].view(1, -1)[:, at] = 255
    if not tree:
        p["v"][0, 25], p["k"][0, 24] = 0.0, 0.0
        got = check(p, window=4200, sinks=33)
        assert not torch.isfinite(got[0, 0, :, 32:64]).any() and torch.isfinite(got[0, 1:]).all() and torch.isfinite(got[0, 0, :, :32]).all()


def shared_cache(batch, draft, heads, kv, dim, page, length, act, spare=3):
    """Sequences of equal length on the same pages, and their cached keys and values in 64 bits, [tokens, kv, dim]."""
    g = gen(length)
    pages = -(-length // page)
    p = dict(q=torch.randn(batch, draft, heads, dim, generator=g).to(act), k=torch.randn(batch, draft, kv, dim, generator=g).to(act),
             v=torch.randn(batch, draft, kv, dim, generator=g).to(act))
    for name, keys in (("k_pages", True), ("v_pages", False)):
        p[name] = ref.fast_pack(torch.empty(pages + spare, kv, page, dim), keys)
    order = torch.randperm(pages + spare, generator=g)[:pages]
    p["table"] = order.to(torch.int32).expand(batch, pages).contiguous()
    p["lengths"] = torch.full((batch,), length, dtype=torch.int32)
    held = [ref.unpack(p[name][order], keys).transpose(1, 2).reshape(-1, kv, dim)[:length] for name, keys in (("k_pages", True), ("v_pages", False))]
    return {name: t.cuda() for name, t in p.items()}, *held


@pytest.mark.parametrize("act", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("more", [{}, dict(window=35000, sinks=300)], ids=["all", "window"])
def test_many_rows_over_ranges_of_many_tiles(act, more):
    # 128 items of 40000 keys on 512 workgroups: ranges of more than the 128 tiles whose pages are looked up at once, and
    # whole numbers of them do not end where items do
    batch, draft, heads, kv, length = 64, 24, 8, 2, 40000
    p, held_k, held_v = shared_cache(batch, draft, heads, kv, 128, 64, length, act)
    for s in (0, 13, 63):                  # a stretch of pages that name none
        p["table"][s, 200:420] = -1
    got = kiln.tree_attention(**p, **more).double().cpu()
    there = torch.arange(length)
    for s, i, h in [(s, i, h) for s in (0, 1, 13, 40, 63) for i in (0, 11, 23) for h in (0, 3, 7)]:
        c = h // (heads // kv)
        seen = torch.ones(length, dtype=torch.bool)
        if s in (0, 13, 63):
            seen &= (there < 200 * 64) | (there >= 420 * 64)
        if more:
            seen &= (there < more["sinks"]) | (there > length + i - more["window"])
        new_k, new_v = (ref.rounded(p[name][s, :i + 1, c].cpu()) for name in ("k", "v"))
        kk, vv = torch.cat([held_k[seen, c], new_k]), torch.cat([held_v[seen, c], new_v])
        want = torch.softmax(kk @ p["q"][s, i, h].double().cpu() / math.sqrt(128), 0) @ vv
        torch.testing.assert_close(got[s, i, h], want, **tolerance(act))


@pytest.mark.parametrize("act", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("more", [{}, dict(window=4200, sinks=20)], ids=["all", "window"])
@pytest.mark.parametrize("tree", [True, False], ids=["tree", "chain"])
def test_blocks_of_many_rows(act, more, tree):
    # 300 rows of a head: two blocks of 128 and one that is not full
    check(ref.problem(gen(16), act=act, batch=2, draft=50, heads=6, kv=1, dim=64, page=64, lengths=(4700, 130), tree=tree, device="cuda"), **more)


@pytest.mark.parametrize("act", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
def test_many_rows_over_picked_pages(act, dim):
    # 104 query heads of one kv head, 70 of 79 pages picked for each token, some lists shorter
    p = ref.problem(gen(17), act=act, batch=2, draft=2, heads=104, kv=1, dim=dim, page=64, lengths=(5000, 4100), device="cuda")
    g, sel = gen(18), torch.full((2, 2, 1, 70), -1, dtype=torch.int32)
    for s, columns in ((0, 79), (1, 65)):
        for i in range(2):
            n = min(70, columns) - 9 * i
            sel[s, i, 0, :n] = torch.randperm(columns, generator=g)[:n].sort().values.to(torch.int32)
    sel[0, 0, 0, 10] = sel[0, 0, 0, 9]     # named twice: counts once
    check(p, selected=sel.cuda())


@pytest.mark.parametrize("draft,heads,lengths,more", [
    (1, 4, (150, 90), {}), (7, 2, (150, 90), {}), (7, 4, (150, 90), dict(window=60, sinks=5)),
    (26, 8, (4300, 4200), {}), (26, 8, (4300, 4200), dict(window=4160, sinks=33))], ids=["one", "few", "window", "wide", "wide-window"])
def test_blocks_that_are_nan(draft, heads, lengths, more):
    # whichever kernel reads them, in whole tiles, the last one and one on a window's edge
    p = ref.problem(gen(15), act=torch.bfloat16, batch=2, draft=draft, heads=heads, kv=2, dim=64, page=64, lengths=lengths, device="cuda")
    for s, n in enumerate(lengths):
        seen = [n - 1, n - 30, n - 50] + ([] if s == 0 else [70 if "window" not in more else n - more["window"] + 1])
        for t in seen:                     # values of one head's second block
            p["v_pages"][int(p["table"][s, t // 64]), 0].view(-1)[ref.places(t % 64, 32, 64, 64, False)[1]] = 255
    page = int(p["table"][1, (lengths[1] - 20) // 64])
    p["k_pages"][page, 1].view(-1)[ref.places((lengths[1] - 20) % 64, 0, 64, 64, True)[1]] = 255
    got = check(p, **more).view(2, draft, 2, heads // 2, 64)
    assert torch.isnan(got[:, :, 0, :, 32:]).all() and torch.isnan(got[1, :, 1]).all()
    assert torch.isfinite(got[:, :, 0, :, :32]).all() and torch.isfinite(got[0, :, 1]).all()


def test_fork_and_compact():
    # pages of 17-byte rows: shared, copied when one of their sequences writes to them, moved to the front of the pool
    g = gen(19)
    cache = kiln.PagedCache(2, 12, 16, 2, 32, dtype=torch.float4_e2m1fn_x2, means=True, device="cuda")
    first = cache.open()

    def tokens(seqs, n):
        k, v = (torch.randn(2, len(seqs), n, 2, 32, generator=g) for _ in "kv")
        cache.append(seqs, k.cuda(), v.cuda())
        for i, s in enumerate(seqs):
            held[s] = tuple(torch.cat([old, ref.rounded(t[:, i])], 1) for old, t in zip(held[s], (k, v)))

    def check_all():
        got = cache.read(list(held), dtype=torch.float32)
        for j, s in enumerate(held):
            n = cache.length(s)
            for t, want in zip(got, held[s]):
                assert torch.equal(t[:, j, :n].double().cpu(), want) and not t[:, j, n:].any()
            for column, page in enumerate(cache.pages_of(s)):
                mean = held[s][0][:, 16 * column:16 * (column + 1)].mean(1)
                torch.testing.assert_close(cache.means[:, page].double().cpu(), mean, rtol=0, atol=16 * 2 ** -24 * 8)

    held = {first: (torch.zeros(2, 0, 2, 32, dtype=torch.float64),) * 2}
    other = cache.open()
    held[other] = held[first]
    tokens([first, other], 39)
    made = cache.fork(first, 2)
    for s in made:
        held[s] = held[first]
    assert cache.free_pages == 6
    tokens([made[0], first], 5)            # both write to a page that three have
    assert cache.free_pages == 4
    check_all()
    cache.free(other)
    del held[other]
    assert cache.compact() == 5 and max(p for s in held for p in cache.pages_of(s)) == 4
    check_all()
    tokens([*made, first], 20)
    check_all()


@pytest.mark.parametrize("cache,act", CACHES, ids=IDS)
@pytest.mark.parametrize("draft,heads,lengths", [(1, 2, (70, 33)), (33, 4, (4300, 200))], ids=["one", "many"])
def test_a_scale_of_zero(cache, act, draft, heads, lengths):
    # every key alike; one whose product with the query is not finite makes the row NaN, and no other
    p = ref.problem(gen(27), cache=cache, act=act, draft=draft, heads=heads, kv=1, dim=64, lengths=lengths, tree=False, device="cuda")
    for more in (dict(), dict(window=50, sinks=3)):
        check(p, scale=0.0, **more)
    p["q"][0, 0, 1, 5] = -math.inf
    page, slot = int(p["table"][1, (lengths[1] - 1) // 16]), (lengths[1] - 1) % 16
    if cache == torch.uint8:
        p["k_pages"][page].view(1, -1)[:, ref.places(slot, 0, 64, 16, True)[1]] = 255
    else:
        p["k_pages"][page, 0, slot, 9] = math.inf
    for more in (dict(), dict(window=50, sinks=3)):
        got = check(p, scale=0.0, **more)
        assert torch.isnan(got[0, 0, 1]).all() and torch.isfinite(got[0, 0, 0]).all() and torch.isnan(got[1]).all()


# -- windows ---------------------------------------------------------------------------------------


@pytest.mark.parametrize("cache,act", CACHES, ids=IDS)
@pytest.mark.parametrize("window,sinks", [(1, 0), (2, 1), (17, 0), (33, 4), (64, 40), (200, 16), (5000, 0)])
def test_windows(cache, act, window, sinks):
    for draft, tree, dim in ((1, False, 64), (7, True, 128), (40, True, 64), (40, False, 128)):
        check(ref.problem(gen(window), cache=cache, act=act, batch=3, draft=draft, heads=4, kv=2, dim=dim, tree=tree,
                          lengths=(430, 0, 61), device="cuda"), window=window, sinks=sinks)


@pytest.mark.parametrize("cache,act", CACHES, ids=IDS)
def test_long_windows(cache, act):
    # ranges, and (many rows) the kernel that shares tiles
    for draft, heads, dim in ((1, 4, 64), (3, 4, 256), (33, 4, 128), (70, 2, 64)):
        check(ref.problem(gen(9), cache=cache, act=act, batch=2, draft=draft, heads=heads, kv=2, dim=dim, page=64,
                          lengths=(6000, 2100), device="cuda"), window=1900, sinks=70)


@pytest.mark.parametrize("cache,act", CACHES, ids=IDS)
@pytest.mark.parametrize("draft,heads", [(6, 4), (33, 4)], ids=["few", "many"])
def test_what_is_behind_the_window_does_not_reach(cache, act, draft, heads):
    # pages that no token sees hold NaN or are not named; a value that only the first tokens still see reaches only them
    p = ref.problem(gen(11), cache=cache, act=act, draft=draft, heads=heads, kv=2, dim=64, lengths=(200, 90), tree=False, device="cuda")
    window, sinks = 50, 5
    first = 200 - window + 1                   # token 0's first key; token 1 does not see it
    spoilt = [(0, t) for t in range(sinks, first)] + [(0, first), (1, 90 - window + 1)]
    for s, t in spoilt:
        page, slot = int(p["table"][s, t // 16]), t % 16
        if cache == torch.uint8:
            for pages, keys in ((p["k_pages"], True), (p["v_pages"], False)):
                for d in (0, 32):
                    pages[page].view(2, -1)[:, ref.places(slot, d, 64, 16, keys)[1]] = 255
        else:
            p["v_pages"][page, :, slot] = math.inf
            p["k_pages"][page, :, slot] = math.nan if t < first - 3 else 0.0
    got = check(p, window=window, sinks=sinks)
    assert torch.isfinite(got[:, 1:]).all() and not torch.isfinite(got[:, 0]).any()
    p["table"][0, 1:(first - 1) // 16] = -1
    assert torch.equal(check(p, window=window, sinks=sinks)[:, 1:], got[:, 1:])


def test_window_of_everything():
    p = ref.problem(gen(12), cache=torch.bfloat16, act=torch.bfloat16, draft=5, lengths=(300, 7), device="cuda")
    assert torch.equal(kiln.tree_attention(**p, window=10 ** 6), kiln.tree_attention(**p))


# -- in graphs, plans and beside other work ------------------------------------------------------------


@pytest.mark.parametrize("precision", ["fp32", "bf16"])
@pytest.mark.parametrize("cache", [torch.uint8, torch.bfloat16])
@pytest.mark.parametrize("window,sinks", [(None, 0), (60, 3)])
def test_compiled_block(precision, cache, window, sinks):
    block = test_packed.gpt2_init_(test_packed.Block(128, 2, 16), seed=0).eval()
    args = test_packed.block_operands(cache=cache, d=128, lengths=(500, 33))
    model = test_packed.WindowBlock(block, 3, window, sinks)
    on_gpu = tuple(t.cuda() for t in args)
    compiled = kiln.compile(model, (args[0], *on_gpu[1:]), device="cuda", matmul_precision=precision)
    got = compiled(*on_gpu)
    if precision == "fp32":
        want = test_packed.block_reference(block, *args, 3, window=window, sinks=sinks)
        assert cache != torch.uint8 or all(test_packed.steps_agree(a, b) for a, b in zip(got[1:], want[1:]))
        for a, b in zip(got, want):
            torch.testing.assert_close(a.double().cpu(), b, rtol=1e-4, atol=1e-5)
    else:
        # the new tokens' keys and values as the plan's bf16 products made them (a 4-bit step may lie between those and
        # the 64-bit ones), the rest of the block in 64 bits
        q = block.double().c_attn(block.ln1(args[0].double())).detach()[:, :128].view(2, 3, 2, 64)
        y = ref.attention(q.float(), got[1].float(), got[2].float(), *args[1:], window=window, sinks=sinks)
        x = args[0].double() + block.c_proj(y.reshape(6, 128))
        want = x + block.proj(torch.nn.functional.gelu(block.fc(block.ln2(x)), approximate="tanh"))
        torch.testing.assert_close(got[0].double().cpu(), want, rtol=2e-2, atol=2e-2)


def test_compiled_block_of_many_rows():
    # fp32 activations rounded to bf16 once, over 4-bit pages: rows that share tiles
    block = test_packed.gpt2_init_(test_packed.Block(128, 2, 16), seed=4).eval()
    args = test_packed.block_operands(d=128, seqs=1, tokens=100, lengths=(4300,))
    on_gpu = tuple(t.cuda() for t in args)
    compiled = kiln.compile(test_packed.WindowBlock(block, 100), (args[0], *on_gpu[1:]), device="cuda", matmul_precision="bf16")
    got = compiled(*on_gpu)
    q = block.double().c_attn(block.ln1(args[0].double())).detach()[:, :128].view(1, 100, 2, 64)
    y = ref.attention(q.float(), got[1].float(), got[2].float(), *args[1:])
    x = args[0].double() + block.c_proj(y.reshape(100, 128))
    want = x + block.proj(torch.nn.functional.gelu(block.fc(block.ln2(x)), approximate="tanh"))
    torch.testing.assert_close(got[0].double().cpu(), want, rtol=2e-2, atol=2e-2)


def test_compiled_block_in_a_callers_graph():
    block = test_packed.gpt2_init_(test_packed.Block(64, 2, 16), seed=1).eval()
    args = test_packed.block_operands()
    on_gpu = tuple(t.cuda() for t in args)
    compiled = kiln.compile(test_packed.WindowBlock(block, 3, 30, 2), (args[0], *on_gpu[1:]), device="cuda")
    compiled(*on_gpu)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = compiled(*on_gpu)
    for turn in range(4):
        on_gpu[0].copy_(torch.randn(6, 64, generator=gen(turn)))
        on_gpu[4].copy_(torch.tensor([40 - turn * 11, turn], dtype=torch.int32))
        want = compiled(*on_gpu)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_torch_compile_backend(monkeypatch):
    monkeypatch.setenv("KILN_STRICT", "1")
    block = test_packed.gpt2_init_(test_packed.Block(64, 2, 16), seed=2).eval().cuda()
    args = tuple(t.cuda() for t in test_packed.block_operands())
    model = test_packed.WindowBlock(block, 3, 30, 2)
    before = kiln.stats["compiled"]
    with torch.no_grad():
        got = torch.compile(model, backend=kiln.backend, dynamic=False)(*args)
        want = model(*args)          # the operators as functions, torch's other kernels
    assert kiln.stats["compiled"] > before
    assert all(test_packed.steps_agree(a, b) for a, b in zip(got[1:], want[1:]))
    for a, b in zip(got, want):
        torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-5)


def test_calls_in_one_graph():
    # ranges with a workspace, whole items, appends and reads: captured together, each with memory of its own
    p = ref.problem(gen(20), act=torch.bfloat16, batch=2, draft=1, heads=8, kv=2, dim=128, page=64, lengths=(9000, 3000), device="cuda")
    q = ref.problem(gen(21), act=torch.float32, batch=2, draft=4, heads=4, kv=2, dim=64, lengths=(90, 5), spare=6, device="cuda")
    zero = torch.zeros(2, dtype=torch.int32, device="cuda")
    out = {}

    def step(pages):
        out["long"] = kiln.tree_attention(**p)
        out["window"] = kiln.tree_attention(**p, window=5000, sinks=4)
        kiln.cache_append(q["k"], q["v"], pages[0], pages[1], q["table"], q["lengths"])
        out["short"] = kiln.tree_attention(q["q"], q["k"], q["v"], *pages, q["table"], q["lengths"], q["parents"])
        out["read"] = torch.stack(kiln.cache_read(*pages, q["table"], zero, q["lengths"], tokens=100))

    mine = [q["k_pages"].clone(), q["v_pages"].clone()]
    step(mine)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(mine)
    captured = dict(out)
    for turn in range(3):
        g = gen(30 + turn)
        p["q"].copy_(torch.randn(p["q"].shape, generator=g))
        q["k"].copy_(torch.randn(q["k"].shape, generator=g))
        q["lengths"].copy_(torch.tensor([80 - turn, 7 + turn], dtype=torch.int32))
        other = [t.clone() for t in mine]
        graph.replay()
        step(other)
        torch.cuda.synchronize()
        for name, t in captured.items():
            assert torch.equal(t.nan_to_num(), out[name].nan_to_num()), name
        assert all(torch.equal(a, b) for a, b in zip(mine, other))


def test_side_stream_and_threads():
    import threading

    p = ref.problem(gen(22), act=torch.bfloat16, batch=2, draft=3, heads=8, kv=2, dim=128, page=64, lengths=(7000, 100), device="cuda")
    want = {w: kiln.tree_attention(**p, window=w) for w in (None, 40, 6000)}
    torch.cuda.synchronize()
    bad = []

    def work(w):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                if not torch.equal(kiln.tree_attention(**p, window=w), want[w]):
                    bad.append(w)
        stream.synchronize()

    threads = [threading.Thread(target=work, args=(w,)) for w in (None, 40, 6000, None)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_other_strides_and_places():
    p = ref.problem(gen(23), act=torch.float16, draft=5, heads=4, kv=2, dim=64, lengths=(40, 17), device="cuda")
    want = kiln.tree_attention(**p, window=20, sinks=3)
    q = dict(p)
    q["q"] = torch.stack([p["q"]] * 2, 2)[:, :, 0]                              # rows apart
    q["k"] = p["k"].transpose(1, 2).contiguous().transpose(1, 2)
    q["v"] = torch.cat([p["v"], p["v"]], -1)[..., :64]
    for name in ("k_pages", "v_pages"):
        both = torch.zeros(len(p[name]), 3, 16, 34, dtype=torch.uint8, device="cuda")   # heads of a wider pool
        both[:, 1:] = p[name]
        q[name] = both[:, 1:]
    q["table"] = torch.stack([p["table"]] * 2, -1)[..., 0]
    q["lengths"] = torch.stack([p["lengths"]] * 2, -1)[:, 0]
    assert torch.equal(kiln.tree_attention(**q, window=20, sinks=3), want)
    layers = torch.stack([q["k_pages"], q["k_pages"]])
    starts = torch.zeros(2, dtype=torch.int32, device="cuda")
    a = kiln.cache_read(layers, layers, q["table"], starts, q["lengths"], tokens=41)
    b = kiln.cache_read(p["k_pages"], p["k_pages"], p["table"], starts, p["lengths"], tokens=41)
    assert all(torch.equal(x[0], y) and torch.equal(x[1], y) for x, y in zip(a, b))


def test_another_cards_tensors_are_refused():
    p = ref.problem(gen(24), device="cuda")
    with pytest.raises(ValueError):
        kiln.tree_attention(**dict(p, table=p["table"].cpu()))
    with pytest.raises(ValueError):
        kiln.cache_read(p["k_pages"], p["v_pages"], p["table"].cpu(), p["lengths"], p["lengths"], tokens=3)


def test_as_operators_of_torch():
    p = ref.problem(gen(25), device="cuda")
    starts = torch.zeros(2, dtype=torch.int32, device="cuda")
    pages = [p["k_pages"].clone(), p["v_pages"].clone()]
    with torch.utils.flop_counter.FlopCounterMode(display=False):
        got = kiln.tree_attention(**p, window=9, sinks=1)
        kiln.cache_append(p["k"], p["v"], *pages, p["table"], p["lengths"])
        k, v = kiln.cache_read(*pages, p["table"], starts, p["lengths"], tokens=30)
    assert torch.equal(got, kiln.tree_attention(**p, window=9, sinks=1))
    kiln.cache_append(p["k"], p["v"], p["k_pages"], p["v_pages"], p["table"], p["lengths"])
    assert torch.equal(pages[0], p["k_pages"]) and torch.equal(pages[1], p["v_pages"])
    assert torch.equal(k, kiln.cache_read(*pages, p["table"], starts, p["lengths"], tokens=30)[0])


@pytest.mark.parametrize("cache,act", [(torch.uint8, torch.bfloat16), (torch.bfloat16, torch.bfloat16)], ids=["fp4", "bf16"])
def test_pools_past_32_bits(cache, act):
    """The last pages of pools of more than 2^32 bytes."""
    p = ref.problem(gen(26), cache=cache, act=act, draft=4, heads=4, kv=2, dim=128, lengths=(40, 17), device="cuda")
    first = 2 ** 32 // p["k_pages"][0].nbytes
    q = dict(p, table=p["table"] + first)
    for name in ("k_pages", "v_pages"):
        q[name] = torch.zeros((first + len(p[name]), *p[name].shape[1:]), dtype=cache, device="cuda")
        q[name][first:] = p[name]
    starts = torch.tensor([3, 0], dtype=torch.int32, device="cuda")
    for more in (dict(), dict(window=20, sinks=3)):
        assert torch.equal(kiln.tree_attention(**q, **more), kiln.tree_attention(**p, **more))
    for x in (p, q):
        kiln.cache_append(x["k"], x["v"], x["k_pages"], x["v_pages"], x["table"], x["lengths"])
    a, b = (kiln.cache_read(x["k_pages"], x["v_pages"], x["table"], starts, x["lengths"] + 4, tokens=50) for x in (p, q))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
