"""Operators around the paged cache's decoding step, as cases whose speed can be measured.

The paged cache and attention over it are described in ``operators.py`` beside
this file. What is measured here:

  packed   attention of N drafted tokens a sequence over a cache held in 4 bits
  window   the same attention (4-bit pages or others) where a token sees only
           the last `window` tokens up to itself and the first `sinks` of the
           sequence; pages that no token sees any more are not in the pool
  append   new tokens written into 4-bit pages, with the pages' mean keys, and
           the sequences read back as dense keys and values
  verify   drafted tokens, a chain or a tree, kept or refused by the target
           model's probabilities and given random numbers, and the token after

4-bit pages: 32 adjacent dimensions of a token's key or value share a power of
two, 2^(e - 127), e one byte (255: the block is NaN); an element is a sign and
one of 0, .5, 1, 1.5, 2, 3, 4, 6 times it. e is the smallest from 2 on for
which the block's largest rounds to 6 at most. A page of a head holds first the
codes of all its tokens, then their scale bytes, ``[pages, kv heads, page size,
17 dim / 32]`` bytes in all:

  keys     token t, dimension d: code byte t dim/2 + d/2 (the low half where d
           is even), scale byte t dim/32 + d/32
  values   16 tokens together: code byte (t/16) 8 dim + ((t%16)/4 dim/8 + d/8) 16
           + (t%4) 4 + (d%8)/2, scale byte (t/16) dim/2 + ((t%16)/4 dim/32 + d/32) 4 + t%4

A case is a dict: ``kind``, ``batch`` (sequences), ``draft`` (N), ``heads``,
``kv_heads``, ``dim``, ``page``, ``length`` (the longest sequence; the others
are spread below it), ``cache`` and ``act`` (element types), ``window``,
``sinks``, ``layers``; for ``verify`` ``vocab``, ``act`` (the probabilities'
type), ``tree`` and ``probs`` (whether the draft's probabilities are there).

Where ``own`` is false, ``run`` computes in plain torch operations; where it is
true, it calls the framework.
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16, "fp64": torch.float64}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2, "fp4": 17 / 32}
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def kiln():
    if "kiln" not in sys.modules:
        sys.path.insert(0, os.path.abspath("kiln-compiler_amd"))
    import kiln as package

    return package


# -- cases ----------------------------------------------------------------------------------


def listed():
    def attend(name, kind, batch, draft, heads, kv_heads, dim, page, length, cache, act, **more):
        return dict(name=name, kind=kind, batch=batch, draft=draft, heads=heads, kv_heads=kv_heads, dim=dim, page=page,
                    length=length, cache=cache, act=act, **more)

    return [
        # one sequence of the GPT-2 block's heads, one token: the smallest decoding step
        attend("packed one fp32", "packed", 1, 1, 12, 12, 64, 16, 137, "fp4", "fp32"),
        # a serving batch of ragged lengths, one token each, grouped heads
        attend("packed ragged decode bf16", "packed", 32, 1, 32, 8, 128, 64, 8192, "fp4", "bf16"),
        # one long sequence, one token: the cache is split over the whole chip
        attend("packed long bf16", "packed", 1, 1, 32, 8, 128, 64, 131072, "fp4", "bf16"),
        # wide trees over long caches: many rows read each key
        attend("packed wide fp16", "packed", 4, 64, 32, 4, 128, 128, 32768, "fp4", "fp16"),
        # one sequence past its window, one token, in the compiler's own type
        attend("window one fp32", "window", 1, 1, 12, 12, 64, 16, 1000, "fp32", "fp32", window=256, sinks=4),
        # a serving batch deep into long texts: most of each is behind the window
        attend("window far decode bf16", "window", 32, 1, 32, 8, 128, 64, 120000, "bf16", "bf16", window=4096, sinks=4),
        # drafted trees of odd size under a window, 4-bit cache, fp32 activations
        attend("window drafted packed", "window", 16, 27, 32, 8, 128, 64, 9000, "fp4", "fp32", window=1021, sinks=16),
        # one step of a small decoding batch, one layer
        dict(name="append one packed", kind="append", layers=1, batch=4, draft=1, kv_heads=12, dim=64, page=16,
             length=60, cache="fp4", act="fp32"),
        # a piece of several prompts, all layers at once
        dict(name="append prompts packed", kind="append", layers=12, batch=16, draft=256, kv_heads=8, dim=128, page=64,
             length=700, cache="fp4", act="bf16"),
        # one sequence with a short chain from a draft model, over a vocabulary of odd size
        dict(name="verify one chain", kind="verify", batch=1, draft=5, vocab=50257, act="fp32", tree=False, probs=True),
        # a serving batch of chains over a large vocabulary
        dict(name="verify chains", kind="verify", batch=64, draft=8, vocab=128000, act="fp32", tree=False, probs=True),
        # trees of the likeliest continuations, without the draft's probabilities
        dict(name="verify trees", kind="verify", batch=32, draft=27, vocab=50257, act="fp32", tree=True, probs=False),
    ]


def draw(rng):
    """One more case: sizes over the listed ones' range, by their logarithm where it is wide."""
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["packed", "packed", "window", "window", "append", "verify", "verify"])
    if kind == "verify":
        draft = spread(1, 32)
        vocab = spread(200, 130000)
        batch = max(1, min(spread(1, 64), 2 ** 26 // (draft * vocab)))
        return dict(kind="verify", batch=batch, draft=draft, vocab=vocab, act=rng.choice(["fp32", "fp32", "bf16", "fp16"]),
                    tree=rng.random() < 0.5, probs=rng.random() < 0.6)
    kv_heads = rng.choice([1, 2, 4, 8, 12])
    group = rng.choice([1, 1, 2, 4, 7, 8])
    dim = rng.choice([32, 64, 64, 96, 128, 128, 160, 256])
    page = rng.choice([16, 32, 64, 128])
    if kind == "append":
        return dict(kind="append", layers=rng.choice([1, 2, 6, 12]), batch=spread(1, 16), draft=spread(1, 256),
                    kv_heads=rng.choice([1, 2, 4, 8]), dim=min(dim, 128), page=min(page, 64), length=spread(1, 700),
                    cache="fp4", act=rng.choice(["fp32", "bf16", "fp16"]))
    cache, act = rng.choice([("fp4", "fp32"), ("fp4", "bf16"), ("fp4", "fp16")])
    draft = rng.choice([1, 1, 1, spread(2, 64), spread(2, 64)])
    batch = spread(1, 32)
    rows = draft * group
    # cost: cached elements, and cached elements times rows, kept under the largest listed case
    room = max(1, min(2 ** 26, 2 ** 34 // rows) // (batch * kv_heads * dim))
    case = dict(kind=kind, batch=batch, draft=draft, heads=kv_heads * group, kv_heads=kv_heads, dim=dim, page=page,
                length=min(spread(1, 131072), room), cache=cache, act=act)
    if kind == "window":
        case["cache"], case["act"] = rng.choice([(cache, act), ("fp32", "fp32"), ("bf16", "fp32"), ("bf16", "bf16"), ("fp16", "fp16")])
        case["window"] = min(spread(1, 4096), room)
        case["sinks"] = rng.choice([0, 1, 4, 16, 100])
        case["length"] = spread(1, 120000)
    return case


# -- 4-bit blocks ----------------------------------------------------------------------------


def rounded(x):
    """(codes, scale bytes) of x [..., dim] in fp32: uint8 [..., dim] and [..., dim / 32]."""
    blocks = x.unflatten(-1, (-1, 32))
    largest = blocks.abs().amax(-1)
    fraction, power = torch.frexp(largest)                         # largest = fraction 2^power, fraction in [.5, 1)
    e = (power - 3 + 127 + (fraction >= 0.875)).clamp(2, 254)      # largest < 7 2^(e - 127)
    y = (blocks * torch.ldexp(torch.ones_like(largest), 127 - e)[..., None]).abs()
    code = torch.zeros_like(y, dtype=torch.uint8)
    for i in range(7):                                             # a tie goes to the even code
        middle = (LEVELS[i] + LEVELS[i + 1]) / 2
        code += (y > middle) if i % 2 == 0 else (y >= middle)
    code += 8 * torch.signbit(blocks).to(torch.uint8)
    fine = torch.isfinite(largest)
    return torch.where(fine[..., None], code, 0).flatten(-2), torch.where(fine, e, 255).to(torch.uint8)


def values(code, e):
    """What codes [..., dim] with scale bytes [..., dim / 32] stand for, in fp32."""
    levels = torch.tensor(LEVELS, device=code.device)
    x = levels[(code & 7).long()] * torch.where(code >= 8, -1.0, 1.0)
    scale = torch.ldexp(torch.ones(e.shape, device=e.device), e.int() - 127)
    scale = torch.where(e == 255, float("nan"), scale)
    return (x.unflatten(-1, (-1, 32)) * scale[..., None]).flatten(-2)


def packed(code, e, keys):
    """Codes [..., page, dim] and scale bytes [..., page, dim / 32] as pages [..., page, 17 dim / 32]."""
    page, dim = code.shape[-2:]
    both = code[..., ::2] | code[..., 1::2] << 4                   # [..., page, dim / 2]
    if not keys:
        both = both.unflatten(-1, (dim // 8, 4)).unflatten(-3, (page // 16, 4, 4)).transpose(-3, -2)
        e = e.unflatten(-2, (page // 16, 4, 4)).transpose(-2, -1)
        both, e = both.flatten(-5), e.flatten(-4)
    else:
        both, e = both.flatten(-2), e.flatten(-2)
    return torch.cat([both, e], -1).unflatten(-1, (page, 17 * dim // 32)).contiguous()


def unpacked(pages, keys):
    """Pages [..., page, 17 dim / 32] as (codes, scale bytes)."""
    page, dim = pages.shape[-2], pages.shape[-1] // 17 * 32
    flat = pages.flatten(-2)
    both, e = flat[..., :page * dim // 2], flat[..., page * dim // 2:]
    if keys:
        both, e = both.unflatten(-1, (page, dim // 2)), e.unflatten(-1, (page, dim // 32))
    else:
        both = both.unflatten(-1, (page // 16, 4, dim // 8, 4, 4)).transpose(-3, -2).flatten(-2).flatten(-4, -2)
        e = e.unflatten(-1, (page // 16, 4, dim // 32, 4)).transpose(-2, -1).flatten(-4, -2)
    return torch.stack([both & 15, both >> 4], -1).flatten(-2), e


def as_values(pages, keys):
    """fp32 values of pages of any type."""
    return values(*unpacked(pages, keys)) if pages.dtype == torch.uint8 else pages.float()


def as_stored(x, dtype):
    """fp32 values of new tokens as pages of `dtype` hold them."""
    return values(*rounded(x.float())) if dtype == torch.uint8 else x.to(dtype).float()


# -- what a program has in hand ----------------------------------------------------------------


def lengths_of(case):
    """Cached tokens of each sequence: the first has `length`, the others less, some none."""
    n = case["length"]
    return [n if s == 0 else (n * ((s * 37) % 101)) // 100 for s in range(case["batch"])]


def pages_of(tokens, page):
    return -(-tokens // page)


def columns_of(case, length):
    """Columns of the table whose pages hold a token that the new ones may see."""
    page = case["page"]
    if "window" not in case:
        return list(range(pages_of(length, page)))
    first = max(0, length - case["window"] + 1)
    return [c for c in range(pages_of(length, page)) if c * page < case["sinks"] or (c + 1) * page > first]


def random(gen, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype)


def tree_of(gen, batch, draft, root):
    """parents[s, i]: the drafted token that token i follows, -1 for the cached context's end
    (with `root` of token 0 alone)."""
    at = torch.arange(draft, device="cuda")
    back = 1 + (random(gen, batch, draft).abs() * 3).long()      # a few tokens back: branching, mostly deep
    parents = torch.maximum(at - back, torch.full_like(back, 0 if root else -1))
    parents[:, 0] = -1
    return parents.to(torch.int32)


def pool(gen, case, layers, pages, keys):
    """Random pages [layers, pages, kv heads, page size, ...]; some dimensions are larger than others, as a model's are."""
    shape = (layers, pages, case["kv_heads"], case["page"], case["dim"])
    size = torch.exp(0.5 * random(gen, case["kv_heads"], 1, case["dim"]))
    if case["cache"] != "fp4":
        return (random(gen, *shape) * size).to(DTYPES[case["cache"]])
    return torch.stack([packed(*rounded(random(gen, *shape[1:]) * size), keys) for _ in range(layers)])


def prepare_verify(case, gen):
    batch, n, vocab, at = case["batch"], case["draft"], case["vocab"], DTYPES[case["act"]]
    # two models that mostly agree: peaked distributions, the draft's a noisy copy
    target = 3.0 * random(gen, batch, n, vocab)
    draft = target + 0.7 * random(gen, batch, n, vocab)
    target, draft = target.softmax(-1).to(at), draft.softmax(-1).to(at)
    parents = tree_of(gen, batch, n, True) if case["tree"] else None
    up = parents.long().clamp(min=0) if case["tree"] else (torch.arange(n, device="cuda") - 1).clamp(min=0).expand(batch, n)
    if case["probs"]:    # each token drawn from the draft's row of the token it follows
        total = draft.double().cumsum(-1)
        v = torch.rand(batch, n, generator=gen, device="cuda", dtype=torch.float64)
        s = torch.arange(batch, device="cuda")[:, None].expand(batch, n)
        tokens = torch.searchsorted(total[s, up], (v * total[s, up, -1])[..., None], right=True)[..., 0]
    else:                # the j-th child of a token is the j-th likeliest
        place = ((up[:, :, None] == up[:, None, :]) & (torch.ones(n, n, device="cuda").tril(-1) > 0)).sum(-1)
        place = (place - (up == 0).long()).clamp(min=0)              # (token 0 is no child)
        best = draft.topk(min(n + 1, vocab), -1).indices
        s = torch.arange(batch, device="cuda")[:, None].expand(batch, n)
        tokens = best[s, up, place.clamp(max=best.shape[-1] - 1)]
    return dict(kind="verify", tokens=tokens.clamp(max=vocab - 1).to(torch.int32), target=target, parents=parents,
                uniforms=torch.rand(batch, n, generator=gen, device="cuda"), draft=draft if case["probs"] else None)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["kind"] == "verify":
        return prepare_verify(case, gen)
    kind, hkv, d, ps = case["kind"], case["kv_heads"], case["dim"], case["page"]
    at = DTYPES[case["act"]]
    batch, n = case["batch"], case["draft"]
    lens = lengths_of(case)
    new = n if kind == "append" else 0
    columns = [list(range(pages_of(x + new, ps))) if new else columns_of(case, x) for x in lens]
    total = sum(len(c) for c in columns) + 3
    order = torch.randperm(total, generator=gen, device="cuda").tolist()
    table = torch.full((batch, max(1, pages_of(case["length"] + new, ps))), -1, dtype=torch.int32)
    for s, c in enumerate(columns):
        if c:
            table[s, c] = torch.tensor(order[:len(c)], dtype=torch.int32)
            order = order[len(c):]
    state = dict(kind=kind, table=table.cuda(), lengths=torch.tensor(lens, dtype=torch.int32, device="cuda"))
    layers = case.get("layers", 1)
    k, v = pool(gen, case, layers, total, True), pool(gen, case, layers, total, False)
    if kind == "append":
        state["k_pages"], state["v_pages"] = k, v
        state["k_means"] = torch.stack([as_values(layer, True).mean(2) for layer in k])
        state["k"] = random(gen, layers, batch, n, hkv, d, dtype=at)
        state["v"] = random(gen, layers, batch, n, hkv, d, dtype=at)
        state["starts"] = torch.zeros_like(state["lengths"])
        state["ends"] = state["lengths"] + n
        state["most"] = case["length"] + n
        return state
    h = case["heads"]
    # q, k, v as a projection leaves them: side by side in one row a token
    qkv = random(gen, batch, n, (h + 2 * hkv) * d, dtype=at)
    state["q"] = qkv[..., :h * d].view(batch, n, h, d)
    state["k"] = qkv[..., h * d:(h + hkv) * d].view(batch, n, hkv, d)
    state["v"] = qkv[..., (h + hkv) * d:].view(batch, n, hkv, d)
    state["parents"] = tree_of(gen, batch, n, False) if n > 1 else None
    state["k_pages"], state["v_pages"] = k[0], v[0]
    state["window"], state["sinks"] = case.get("window"), case.get("sinks", 0)
    return state


# -- one pass -------------------------------------------------------------------------------------


def ancestors(parents, batch, n, device):
    """[batch, n, n]: token j is token i or one that i follows. Products of the parent matrix with
    itself double the distance covered."""
    eye = torch.eye(n, device=device).expand(batch, n, n)
    if parents is None:
        return torch.ones(n, n, device=device).tril().expand(batch, n, n) > 0
    one = (parents[..., None] == torch.arange(n, device=device)).float()
    reach, step, far = eye, one, 1
    while far < n:
        reach = reach + reach @ step
        step, far = step @ step, 2 * far
    return reach > 0


def softmax_product(scores, ok, v):
    scores = torch.where(ok, scores, float("-inf"))
    e = torch.exp(scores - scores.amax(-1, keepdim=True))
    return (e @ v) / e.sum(-1, keepdim=True)


def plain_attention(q, k, v, k_pages, v_pages, table, lengths, parents, window, sinks):
    batch, n, h, d = q.shape
    hkv, ps = k_pages.shape[1], k_pages.shape[2]
    length = lengths.long()[:, None]
    # the columns of the table that are looked at: all, or the sinks' and those from the window's first on
    if window is None or sinks + window >= table.shape[1] * ps:
        column = torch.arange(table.shape[1], device=q.device).expand(batch, -1)
        fresh = torch.ones_like(column, dtype=torch.bool)
    else:
        few = min(pages_of(sinks, ps), table.shape[1])
        start = (length - window + 1).clamp(min=0) // ps
        column = torch.cat([torch.arange(few, device=q.device).expand(batch, -1),
                            start + torch.arange(pages_of(window, ps) + 1, device=q.device)], 1)
        fresh = torch.arange(column.shape[1], device=q.device) < few
        fresh = fresh | ((column >= few) & (column < table.shape[1]))
    at = table.long().gather(1, column.clamp(max=table.shape[1] - 1))
    place = (column[..., None] * ps + torch.arange(ps, device=q.device)).flatten(1)                    # [S, T]
    here = (fresh & (at >= 0)).repeat_interleave(ps, 1) & (place < length)
    at = at.clamp(min=0)

    def keys(pages, new, of_keys):
        cached = as_values(pages[at], of_keys).permute(0, 2, 1, 3, 4).reshape(batch, hkv, -1, d)
        cached = torch.where(here[:, None, :, None], cached, 0.0)
        return torch.cat([cached, as_stored(new, pages.dtype).transpose(1, 2)], 2)                     # [S, Hkv, T + N, D]

    rows = q.float().view(batch, n, hkv, h // hkv, d).permute(0, 2, 1, 3, 4).reshape(batch, hkv, -1, d)
    scores = (rows @ keys(k_pages, k, True).transpose(2, 3).contiguous()) * (1.0 / math.sqrt(d))
    tree = ancestors(parents, batch, n, q.device)
    ok = torch.cat([here[:, None, :].expand(batch, n, -1), tree], 2)                                    # [S, N, T + N]
    if window is not None:
        mine = length + tree.sum(-1) - 1                                                                # [S, N]
        place = torch.cat([place, mine], 1)[:, None, :]
        ok = ok & ((place < sinks) | (place > mine[..., None] - window))
    ok = ok.repeat_interleave(h // hkv, 1)[:, None]
    out = softmax_product(scores, ok, keys(v_pages, v, False))
    return out.view(batch, hkv, n, h // hkv, d).permute(0, 2, 1, 3, 4).reshape(batch, n, h, d).to(q.dtype)


def plain_append(k, v, k_pages, v_pages, table, lengths, k_means):
    """All tokens of k and v behind the cached ones."""
    n, ps, d = k.shape[2], k_pages.shape[3], k.shape[4]
    length = lengths.long()[:, None]
    column = length // ps + torch.arange((n - 1) // ps + 2, device=k.device)                            # [S, J]
    used = column * ps < length + n
    page = table.long().gather(1, column.clamp(max=table.shape[1] - 1))
    page = torch.where(used, page, page[:, :1])                                                         # (the first again)
    column = torch.where(used, column, column[:, :1])
    row = column[..., None] * ps + torch.arange(ps, device=k.device) - length[..., None]                # [S, J, ps]
    taken = (row >= 0) & (row < n)
    seq = torch.arange(len(k[0]), device=k.device)[:, None, None]
    held = (length + n - column * ps).clamp(1, ps)
    inside = torch.arange(ps, device=k.device) < held[..., None]
    for pages, new, keys in ((k_pages, k, True), (v_pages, v, False)):
        code, e = unpacked(pages[:, page], keys)                                                        # [L, S, J, H, ps, .]
        new_code, new_e = rounded(new.float()[:, seq, row.clamp(0, n - 1)].transpose(4, 3))
        code = torch.where(taken[:, :, None, :, None], new_code, code)
        e = torch.where(taken[:, :, None, :, None], new_e, e)
        pages[:, page] = packed(code, e, keys)
        if keys:
            total = torch.where(inside[:, :, None, :, None], values(code, e), 0.0).sum(4)
            k_means[:, page] = total / held[..., None, None]


def plain_read(k_pages, v_pages, table, starts, ends, most):
    """Tokens starts[s] .. ends[s] as dense bf16 keys and values [L, S, most, H, D], zeros behind them."""
    ps = k_pages.shape[3]
    place = starts.long()[:, None] + torch.arange(most, device=table.device)
    here = place < ends[:, None]
    page = table.long().gather(1, (place // ps).clamp(max=table.shape[1] - 1)).clamp(min=0)
    out = []
    for pages, keys in ((k_pages, True), (v_pages, False)):
        x = as_values(pages, keys).to(torch.bfloat16)[:, page, :, place % ps]                           # [S, most, L, H, D]
        out.append(torch.where(here[..., None, None, None], x, 0.0).permute(2, 0, 1, 3, 4).contiguous())
    return out


def plain_verify(tokens, target, uniforms, parents, draft):
    batch, n, vocab = target.shape
    seq = torch.arange(batch, device=tokens.device)
    parents = (torch.arange(n, device=tokens.device) - 1).expand(batch, n) if parents is None else parents
    tokens, u = tokens.long(), uniforms.double()

    def drawn(weights, u):
        """The first token whose running sum passes u of the whole."""
        run = weights.cumsum(-1)
        return (run <= u[..., None] * run[..., -1:]).sum(-1).clamp(max=vocab - 1)

    now = torch.zeros_like(seq)
    taken = [torch.ones_like(seq, dtype=torch.bool)]
    if draft is None:
        choice = drawn(target.double(), u)
        for i in range(1, n):
            taken.append((parents[:, i] == now) & (choice[seq, now] == tokens[:, i]))
            now = torch.where(taken[-1], i, now)
        after = choice[seq, now]
    else:
        left, whole = target[:, 0].double(), torch.ones(batch, dtype=torch.float64, device=tokens.device)
        for i in range(1, n):
            asked = parents[:, i] == now
            p, q = left[seq, tokens[:, i]], draft[seq, now, tokens[:, i]].double()
            taken.append(asked & (u[:, i] * whole * q < p))
            refused = asked & ~taken[-1]
            rest = torch.clamp(left - whole[:, None] * draft[seq, now].double(), min=0.0)
            left = torch.where(taken[-1][:, None], target[:, i].double(), torch.where(refused[:, None], rest, left))
            whole = torch.where(taken[-1], 1.0, torch.where(refused, rest.sum(-1), whole))
            now = torch.where(taken[-1], i, now)
        empty = left.sum(-1) <= 0
        after = drawn(torch.where(empty[:, None], target[seq, now].double(), left), u[:, 0])
    taken = torch.stack(taken, 1)
    count = taken.sum(1)
    order = torch.where(taken, torch.arange(n, device=tokens.device), n).sort(1).values
    return torch.where(order < n, order, -1).to(torch.int32), count.to(torch.int32), after.to(torch.int32)


def run(state):
    kind = state["kind"]
    if kind == "verify":
        args = [state[x] for x in ("tokens", "target", "uniforms", "parents")]
        if own:
            return kiln().verify_tokens(*args, draft=state["draft"])
        return plain_verify(*args, state["draft"])
    if kind == "append":
        args = [state[x] for x in ("k", "v", "k_pages", "v_pages", "table", "lengths")]
        read = [state[x] for x in ("k_pages", "v_pages", "table", "starts", "ends")]
        if own:
            kiln().cache_append(*args, k_means=state["k_means"])
            k, v = kiln().cache_read(*read, tokens=state["most"])
        else:
            plain_append(*args, state["k_means"])
            k, v = plain_read(*read, state["most"])
        return k, v, state["k_means"]
    args = [state[x] for x in ("q", "k", "v", "k_pages", "v_pages", "table", "lengths", "parents")]
    if own:
        return kiln().tree_attention(*args, window=state["window"], sinks=state["sinks"])
    return plain_attention(*args, state["window"], state["sinks"])


# -- what a pass cannot do without ------------------------------------------------------------------


def work(case):
    batch, n = case["batch"], case["draft"]
    if case["kind"] == "verify":
        # one row of the target's probabilities (and of the draft's) decides the token after
        rows = 2 if case["probs"] else 1
        return {"bytes": batch * (rows * case["vocab"] * BYTES[case["act"]] + 16 * n), "flops": 2 * rows * batch * case["vocab"]}
    hkv, d, ps = case["kv_heads"], case["dim"], case["page"]
    cb, ab = BYTES[case["cache"]], BYTES[case["act"]]
    lens = lengths_of(case)
    if case["kind"] == "append":
        # new tokens read, their codes written; everything read back; the touched pages' means written
        row = case["layers"] * hkv * d
        held = sum(x + n for x in lens)
        touched = sum((x + n - 1) // ps - x // ps + 1 for x in lens)
        return {"bytes": int(row * (2 * batch * n * (ab + cb) + 2 * held * (cb + 2) + touched * 4)), "flops": row * batch * n}
    h = case["heads"]
    seen = sum(min(x, case["window"] - 1 + case["sinks"]) if "window" in case else x for x in lens) * hkv * d
    return {"bytes": int(2 * seen * cb) + batch * n * d * ab * (2 * h + 2 * hkv),
            "flops": 4 * seen * n * (h // hkv) + 2 * batch * n * n * h * d}


# -- the definitions, in 64 bits ---------------------------------------------------------------------


def exact_blocks(x):
    """x [..., dim] as a 4-bit cache holds it, in 64 bits: the nearest level, of two as near the even one."""
    x = x.double().unflatten(-1, (-1, 32))
    top = x.abs().amax(-1, keepdim=True)
    step = torch.full_like(top, 2.0 ** -125)
    while bool((top >= 7 * step).any()):
        step = torch.where(top >= 7 * step, 2 * step, step)
    levels = torch.tensor(LEVELS, dtype=torch.float64, device=x.device)
    far = ((x.abs() / step)[..., None] - levels).abs() + torch.tensor([0, 1e-12] * 4, dtype=torch.float64, device=x.device)
    return (levels[far.argmin(-1)] * step * torch.where(x < 0, -1.0, 1.0)).flatten(-2)


def exact_page(page, keys):
    """[page, 17 dim / 32] bytes of one page of one head, by the layout's formulas."""
    ps, dim = page.shape[0], page.shape[1] // 17 * 32
    flat = page.reshape(-1)
    t, d = torch.arange(ps, device=page.device)[:, None], torch.arange(dim, device=page.device)[None]
    if keys:
        code, scale = t * (dim // 2) + d // 2, t * (dim // 32) + d // 32
    else:
        code = t // 16 * 8 * dim + (t % 16 // 4 * (dim // 8) + d // 8) * 16 + t % 4 * 4 + d % 8 // 2
        scale = t // 16 * (dim // 2) + (t % 16 // 4 * (dim // 32) + d // 32) * 4 + t % 4
    nibble = flat[code].long() >> 4 * (d % 2) & 15
    levels = torch.tensor([*LEVELS, *(-x for x in LEVELS)], dtype=torch.float64, device=page.device)
    return levels[nibble] * 2.0 ** (flat[ps * dim // 2 + scale].double() - 127)


def exact_pages(pages, keys):
    """[pages, page, ...] of one head in 64 bits."""
    if pages.dtype != torch.uint8:
        return pages.double()
    return torch.func.vmap(lambda p: exact_page(p, keys))(pages) if len(pages) else pages.new_zeros(0, 1, 1).double()


def exact_verify(state):
    tokens, u = state["tokens"].tolist(), state["uniforms"].double().tolist()
    batch, n, vocab = state["target"].shape
    follows = [[i - 1 for i in range(n)]] * batch if state["parents"] is None else state["parents"].tolist()
    rows, counts, after = [], [], []

    def drawn(w, u):
        passed = (torch.cumsum(w, 0) > u * w.sum()).nonzero()
        return int(passed[0]) if len(passed) else int(w.nonzero()[-1])

    for s in range(batch):
        path, w, total = [0], state["target"][s, 0].double().cpu(), 1.0
        choice = drawn(w, u[s][0]) if state["draft"] is None else None
        for i in range(1, n):
            at, c = path[-1], tokens[s][i]
            if follows[s][i] != at:
                continue
            if state["draft"] is None:
                if c != choice:
                    continue
            else:
                q = state["draft"][s, at].double().cpu()
                if not u[s][i] * total * float(q[c]) < float(w[c]):
                    w = (w - total * q).clamp(min=0)
                    total = float(w.sum())
                    continue
            path.append(i)
            w, total = state["target"][s, i].double().cpu(), 1.0
            if state["draft"] is None:
                choice = drawn(w, u[s][i])
        if state["draft"] is not None:
            choice = drawn(w if float(w.sum()) > 0 else state["target"][s, path[-1]].double().cpu(), u[s][0])
        rows.append(path + [-1] * (n - len(path)))
        counts.append(len(path))
        after.append(choice)
    return tuple(torch.tensor(x, dtype=torch.int32, device="cuda") for x in (rows, counts, after))


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "verify":
        return exact_verify(state)
    ps, hkv, d = case["page"], case["kv_heads"], case["dim"]
    table, lens, batch, n = state["table"].tolist(), lengths_of(case), case["batch"], case["draft"]
    stored = exact_blocks if case["cache"] == "fp4" else lambda x: x.to(DTYPES[case["cache"]]).double()
    if case["kind"] == "append":
        k, v = (torch.zeros(case["layers"], batch, state["most"], hkv, d, dtype=torch.float64, device="cuda") for _ in "kv")
        means = state["k_means"].double()
        new_k, new_v = stored(state["k"]), stored(state["v"])
        for layer in range(case["layers"]):
            for s, x in enumerate(lens):
                held = table[s][:pages_of(x, ps)]
                for out, pages, new, keys in ((k, state["k_pages"], new_k, True), (v, state["v_pages"], new_v, False)):
                    if x:
                        old = exact_pages(pages[layer, held].flatten(0, 1), keys).view(-1, hkv, ps, d)
                        out[layer, s, :x] = old.transpose(1, 2).flatten(0, 1)[:x]
                    out[layer, s, x:x + n] = new[layer, s]
                for b in range(x // ps, pages_of(x + n, ps)):
                    means[layer, table[s][b]] = k[layer, s, b * ps:min((b + 1) * ps, x + n)].mean(0)
        return k, v, means
    q, parents = state["q"].double(), state["parents"]
    h = case["heads"]
    g = h // hkv
    out = torch.zeros(batch, n, h, d, dtype=torch.float64, device="cuda")
    for s, x in enumerate(lens):
        follows = list(range(-1, n - 1)) if parents is None else parents[s].tolist()
        see, depth = torch.zeros(n, n, dtype=torch.bool), [0] * n
        for i in range(n):
            j = i
            while j >= 0:
                see[i, j] = True
                depth[i] += 1
                j = follows[j]
        mine = x - 1 + torch.tensor(depth)
        columns = columns_of(case, x)
        place = torch.tensor([c * ps + t for c in columns for t in range(ps)], dtype=torch.long)
        kept = (place < x).nonzero()[:, 0]
        place = torch.cat([place[kept], mine])
        ok = torch.cat([torch.ones(n, len(kept), dtype=torch.bool), see], 1)
        if "window" in case:
            ok &= (place < case["sinks"]) | (place > mine[:, None] - case["window"])
        ok, kept = ok.cuda(), kept.cuda()
        held = [table[s][c] for c in columns]
        new_k, new_v = stored(state["k"][s]), stored(state["v"][s])
        for c in range(hkv):
            kk, vv = (exact_pages(state[name][held, c], keys).reshape(-1, d)[kept] if held else q.new_zeros(0, d)
                      for name, keys in (("k_pages", True), ("v_pages", False)))
            kk, vv = torch.cat([kk, new_k[:, c]]), torch.cat([vv, new_v[:, c]])
            for head in range(c * g, (c + 1) * g):
                a = ((q[s, :, head] @ kk.T) / math.sqrt(d)).masked_fill(~ok, -math.inf)
                out[s, :, head] = torch.softmax(a, 1) @ vv
    return out
