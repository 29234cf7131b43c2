"""The paged cache's attention on the GPU, held to what its arithmetic gives.

Tolerances. fp32 work is off by less than 1e-4 for any element (normal
operands, scores below 32: products' sums 2^-18 a score, which moves a weight
by as much, and the mean's own sums 2^-18 of the largest value, 6). Over 16-bit
activations the weights are two 16-bit parts: the first is their leading 8
(bf16) or 11 (fp16) bits, which leaves less than 2^-7 or 2^-10 of a weight, and
the second is that rest to half a step, 2^-8 or 2^-11 of it. So a weight is off
by less than 2^-15 or 2^-21 of itself, a result by twice that times the largest
value, and by half a step of its own when it is rounded. Nothing of the size of
a result itself is allowed: over 5000 keys that is about 0.02, and a tile of 32
keys that is lost moves it by about 0.002 (the first test below).
"""

import math

import pytest
import torch

import kiln
import paged_reference as ref

TYPES = [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.float16, torch.float32),
         (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16)]
IDS = ["fp32", "bf16-cache", "fp16-cache", "bf16", "fp16"]
WEIGHT = {torch.float32: 0.0, torch.bfloat16: 2 ** -15, torch.float16: 2 ** -21}


def tolerance(act):
    half = 0.0 if act == torch.float32 else torch.finfo(act).eps / 2
    return dict(rtol=half, atol=1e-4 + 2 * 6 * WEIGHT[act])


def gen(seed=0):
    return torch.Generator().manual_seed(seed)


def check(p, **more):
    got = kiln.tree_attention(**p, **more)
    torch.testing.assert_close(got.double().cpu(), ref.attention(**p, **more), equal_nan=True, **tolerance(got.dtype))
    return got


def long_and_ragged(cache, act, device="cpu"):
    lengths = (5000, 0, 1, 700, 33, 2600, 64, 16)
    return ref.problem(gen(1), batch=8, draft=2, heads=4, kv=2, lengths=lengths, cache=cache, act=act, device=device)


@pytest.mark.parametrize("cache,act", TYPES, ids=IDS)
@pytest.mark.parametrize("sequence,first", [(0, 0), (0, 156), (0, 310), (5, 80)])
def test_a_lost_tile_is_seen(cache, act, sequence, first):
    """A tile of the longest sequences that no wave took is outside the tolerance."""
    p = long_and_ragged(cache, act)
    lost = dict(p, table=p["table"].clone())
    lost["table"][sequence, first:first + 2] = -1
    want, got = ref.attention(**p), ref.attention(**lost).to(act).double()
    torch.testing.assert_close(want.to(act).double(), want, **tolerance(act))
    with pytest.raises(AssertionError):
        torch.testing.assert_close(got[sequence], want[sequence], **tolerance(act))


@pytest.mark.gpu
@pytest.mark.parametrize("cache,act", TYPES, ids=IDS)
def test_long_and_ragged(cache, act):
    check(long_and_ragged(cache, act, "cuda"))
    check(ref.problem(gen(2), batch=40, draft=1, heads=2, kv=1, lengths=[7 * i for i in range(40)], cache=cache,
                      act=act, device="cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("cache,act", TYPES, ids=IDS)
@pytest.mark.parametrize("page", [16, 128, 1024])
@pytest.mark.parametrize("dim", [64, 128, 200])
def test_lengths_and_pages(cache, act, page, dim):
    for lengths in ((1, 0), (31, 33), (2049, 129), (4100, 1000)):
        check(ref.problem(gen(page), lengths=lengths, dim=dim, page=page, cache=cache, act=act, device="cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("cache,act", TYPES, ids=IDS)
@pytest.mark.parametrize("dim,group", [(64, 1), (80, 2), (128, 4)])
def test_many_rows(cache, act, dim, group):
    for lengths, page in (((1100, 0), 16), ((3000, 130), 128)):
        check(ref.problem(gen(group), draft=70, heads=group * 2, kv=2, dim=dim, lengths=lengths, page=page, cache=cache,
                          act=act, device="cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("cache,act", TYPES, ids=IDS)
def test_picked_pages(cache, act):
    p = ref.problem(gen(3), batch=3, draft=5, heads=6, kv=2, lengths=(4000, 0, 1041), cache=cache, act=act, device="cuda")
    for top in (3, 100):
        sel = kiln.select_pages(p["q"], p["k_pages"].float().mean(2), p["table"], p["lengths"], page_size=16, pages=top)
        got = kiln.selected_attention(**p, selected=sel)
        torch.testing.assert_close(got.double().cpu(), ref.attention(**p, selected=sel.cpu()), **tolerance(act))


@pytest.mark.gpu
@pytest.mark.parametrize("cache,act", TYPES, ids=IDS)
@pytest.mark.parametrize("scale", [-0.3, 0.0, 0.3])
def test_scales(cache, act, scale):
    """Scores of 0.3 q . k stay below 16, products' sums below 64: the same 2^-18 a score, twice at the most."""
    for draft, heads in ((3, 4), (70, 4)):
        p = ref.problem(gen(4), draft=draft, heads=heads, kv=2, lengths=(300, 41), cache=cache, act=act, device="cuda")
        got = kiln.tree_attention(**p, scale=scale)
        tol = tolerance(act)
        torch.testing.assert_close(got.double().cpu(), ref.attention(**p, scale=scale), rtol=tol["rtol"], atol=2 * tol["atol"])


@pytest.mark.gpu
@pytest.mark.parametrize("cache,act", [TYPES[1], TYPES[4]], ids=[IDS[1], IDS[4]])
def test_many_rows_over_very_long_ranges(cache, act):
    """Sixteen sequences share the pages of the longest: more than 65536 tiles
    of 64 keys for the 512 workgroups, so that one's tiles are more than the
    128 whose places it holds at a time, and items of more than 8192 keys."""
    batch, draft, kv, group, dim, page = 16, 64, 4, 2, 64, 16
    lengths = [70000 - 37 * s for s in range(batch)]
    p = ref.problem(gen(5), batch=1, draft=1, heads=kv, kv=kv, dim=dim, page=page, lengths=lengths[:1], cache=cache, act=act,
                    device="cuda")
    more = ref.problem(gen(6), batch=batch, draft=draft, heads=kv * group, kv=kv, dim=dim, page=page, lengths=[0] * batch,
                       cache=cache, act=act, device="cuda")
    p = dict(more, k_pages=p["k_pages"], v_pages=p["v_pages"], table=p["table"].expand(batch, -1),
             lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    got = kiln.tree_attention(**p)
    # in 64 bits on the GPU, by sequence and head (plain products of contiguous operands)
    at = p["table"][0].long()
    for s in range(0, batch, 3):
        path, used = ref.see(p["parents"][s].tolist(), draft)
        assert all(used)
        for c in range(kv):
            keys, values = (torch.cat([x[at, c].reshape(-1, dim)[:lengths[s]], new[s, :, c].to(cache)]).double()
                            for x, new in ((p["k_pages"], p["k"]), (p["v_pages"], p["v"])))
            for h in range(c * group, (c + 1) * group):
                score = torch.mm(p["q"][s, :, h].double(), keys.t().contiguous()) / math.sqrt(dim)
                score[:, lengths[s]:].masked_fill_(~path.cuda(), -math.inf)
                want = torch.mm(torch.softmax(score, 1), values)
                torch.testing.assert_close(got[s, :, h].double(), want, **tolerance(act))


@pytest.mark.gpu
@pytest.mark.parametrize("cache,act", TYPES, ids=IDS)
@pytest.mark.parametrize("draft,length", [(5, 100), (70, 100), (5, 3000), (70, 3000)])
def test_infinities_that_are_attended_to(cache, act, draft, length):
    """An infinite value makes its dimension infinite in the rows that attend to
    it, a key whose score is -inf has no weight: cached or drafted."""
    p = ref.problem(gen(7), draft=draft, heads=4, kv=2, lengths=(length, 41), cache=cache, act=act, device="cuda")
    page = p["table"][0, 2]
    p["v_pages"][page, 0, 3, 5] = math.inf
    p["v_pages"][page, 1, 7, 11] = -math.inf
    p["q"][0, :, :, 7] = p["q"][0, :, :, 7].abs() + 0.5
    p["k_pages"][page, 1, 9, 7] = -math.inf       # q[7] > 0: a score of -inf
    p["v"][1, 1, 0, 3] = math.inf
    p["q"][1, :, :, 2] = -p["q"][1, :, :, 2].abs() - 0.5
    p["k"][1, 2, 1, 2] = math.inf
    got = check(p)
    assert torch.isinf(got[0]).sum() == 4 * draft
