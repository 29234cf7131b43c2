"""The operators over a paged key/value cache, as cases whose speed can be measured.

A cache holds the keys and values of many sequences in pages: ``k_pages`` and
``v_pages`` are ``[pages, kv heads, page size, head dim]``, sequence s's token t
lies in page ``table[s, t // page size]`` at slot ``t % page size``, and
``lengths[s]`` tokens of it are there. Four operators work on it:

  tree     attention of N drafted tokens a sequence, each over the whole cache
           and over those drafted tokens that are its ancestors (and itself):
           one token is plain decoding, a chain is a run of tokens
  sparse   the pages a cheap score picks for each drafted token (the sum of a
           group's queries times a page's mean key), then the same attention
           over those pages alone
  append   the accepted drafted tokens' keys and values written behind the
           cached ones, in every layer, and the means of the pages they touch
  copy     whole pages copied within the pool, in every layer (what a fork's
           first write and a compaction do)

A case is a dict: ``kind``, ``batch`` (sequences), ``draft`` (N), ``heads``,
``kv_heads``, ``dim``, ``page``, ``length`` (the longest sequence; the others
are spread below it), ``cache`` and ``act`` (the element types of the pages,
and of q, k, v and the result), ``top`` (pages picked), ``layers``, ``accept``
(tokens appended), ``moved`` (pages copied).

Where ``own`` is false, ``run`` computes in plain torch operations; where it is
true, it calls the framework.
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}


def kiln():
    if "kiln" not in sys.modules:
        sys.path.insert(0, os.path.abspath("kiln-compiler_amd"))
    import kiln as package

    return package


# -- cases ----------------------------------------------------------------------------------


def listed():
    def tree(name, batch, draft, heads, kv_heads, dim, page, length, cache, act):
        return dict(name=name, kind="tree", batch=batch, draft=draft, heads=heads, kv_heads=kv_heads, dim=dim,
                    page=page, length=length, cache=cache, act=act)

    def sparse(name, batch, draft, heads, kv_heads, dim, page, length, cache, act, top):
        return dict(tree(name, batch, draft, heads, kv_heads, dim, page, length, cache, act), kind="sparse", top=top)

    return [
        # one sequence of the GPT-2 block's heads, one token: the smallest decoding step, in the compiler's own type
        tree("tree one fp32", 1, 1, 12, 12, 64, 16, 137, "fp32", "fp32"),
        # the same heads, a drafted tree of odd size per sequence, fp32 activations over a bf16 cache
        tree("tree drafted bf16 cache", 8, 27, 12, 12, 64, 16, 1024, "bf16", "fp32"),
        # a serving batch of ragged lengths, one token each, grouped heads
        tree("tree ragged decode bf16", 32, 1, 32, 8, 128, 64, 8192, "bf16", "bf16"),
        # one long sequence, one token: the cache is split over the whole chip
        tree("tree long bf16 cache", 1, 1, 32, 8, 128, 64, 131072, "bf16", "fp32"),
        # wide trees over long caches: many rows read each key
        tree("tree wide fp16", 4, 64, 32, 4, 128, 128, 32768, "fp16", "fp16"),
        # a short cache where a handful of pages is picked
        sparse("sparse one fp32", 1, 1, 12, 12, 64, 16, 2000, "fp32", "fp32", 8),
        # a serving batch at long lengths, one token each
        sparse("sparse decode bf16", 16, 1, 32, 8, 128, 64, 32768, "bf16", "bf16", 32),
        # drafted trees over very long caches, each token with pages of its own
        sparse("sparse drafted fp16", 2, 13, 32, 8, 128, 128, 131000, "fp16", "fp32", 48),
        # one step of a small decoding batch, one layer
        dict(name="append one bf16", kind="append", layers=1, batch=4, draft=1, accept=1, kv_heads=12, dim=64, page=16,
             length=600, cache="bf16", act="fp32"),
        # the accepted part of drafted trees, all layers at once
        dict(name="append accepted bf16", kind="append", layers=12, batch=64, draft=64, accept=23, kv_heads=8, dim=128,
             page=64, length=4000, cache="bf16", act="bf16"),
        # first writes of three forks of a short sequence
        dict(name="copy forks fp32", kind="copy", layers=1, moved=3, kv_heads=12, dim=64, page=16, pages=64,
             cache="fp32"),
        # a compaction of a large pool
        dict(name="copy compaction bf16", kind="copy", layers=12, moved=301, kv_heads=8, dim=128, page=64, pages=700,
             cache="bf16"),
    ]


def draw(rng):
    """One more case: sizes over the listed ones' range, by their logarithm where it is wide."""
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["tree", "tree", "tree", "sparse", "sparse", "append", "copy"])
    kv_heads = rng.choice([1, 2, 4, 8, 12])
    group = rng.choice([1, 1, 2, 4, 7, 8])
    dim = rng.choice([64, 64, 80, 128, 128, 256])
    page = rng.choice([16, 32, 64, 128])
    cache, act = rng.choice([("fp32", "fp32"), ("bf16", "fp32"), ("fp16", "fp32"), ("bf16", "bf16"), ("fp16", "fp16")])
    if kind == "copy":
        moved = spread(1, 300)
        layers = rng.choice([1, 2, 6, 12])
        return dict(kind="copy", layers=layers, moved=moved, kv_heads=rng.choice([1, 2, 4, 8]), dim=min(dim, 128),
                    page=min(page, 64), pages=2 * moved + rng.randint(1, 90),
                    cache=cache if cache != "fp32" else "bf16")
    if kind == "append":
        draft = spread(1, 64)
        return dict(kind="append", layers=rng.choice([1, 2, 6, 12]), batch=spread(1, 64), draft=draft,
                    accept=rng.randint(1, draft), kv_heads=rng.choice([1, 2, 4, 8]), dim=min(dim, 128),
                    page=min(page, 64), length=spread(1, 4000), cache=cache, act=act)
    # cost: cached elements times rows, kept under the largest listed case
    draft = rng.choice([1, 1, 1, spread(2, 64), spread(2, 64)])
    batch = spread(1, 32)
    length = spread(1, 131072)
    elements = 2 ** 26                                          # keys of one sequence set, all heads
    length = max(1, min(length, elements // (batch * kv_heads * dim)))
    rows = draft * group
    length = max(1, min(length, 2 ** 34 // (batch * kv_heads * dim * rows)))
    case = dict(kind=kind, batch=batch, draft=draft, heads=kv_heads * group, kv_heads=kv_heads, dim=dim, page=page,
                length=length, cache=cache, act=act)
    if kind == "sparse":
        top = rng.randint(1, 48)
        most = 2 ** 27 // (batch * draft * kv_heads * page * dim)   # picked elements
        case["top"] = max(1, min(top, most))
    return case


# -- what a program has in hand ----------------------------------------------------------------


def lengths_of(case):
    """Cached tokens of each sequence: the first has `length`, the others less, some none."""
    n = case["length"]
    return [n if s == 0 else (n * ((s * 37) % 101)) // 100 for s in range(case["batch"])]


def pages_of(tokens, page):
    return -(-tokens // page)


def random(gen, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype)


def tree_of(gen, batch, draft):
    """parents[s, i]: the drafted token that token i follows, -1 for the cached context's end."""
    at = torch.arange(draft, device="cuda")
    back = 1 + (random(gen, batch, draft).abs() * 3).long()      # a few tokens back: branching, mostly deep
    return torch.maximum(at - back, torch.full_like(back, -1)).to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, hkv, d, ps = case["kind"], case["kv_heads"], case["dim"], case["page"]
    ct = DTYPES[case["cache"]]
    if kind == "copy":
        layers, pages, moved = case["layers"], case["pages"], case["moved"]
        k = random(gen, layers, pages, hkv, ps, d, dtype=ct)
        v = random(gen, layers, pages, hkv, ps, d, dtype=ct)
        order = torch.randperm(pages, generator=gen, device="cuda").tolist()
        return dict(kind=kind, k_pages=k, v_pages=v, source=order[:moved], target=order[moved:2 * moved])

    at = DTYPES[case["act"]]
    batch, n = case["batch"], case["draft"]
    lens = lengths_of(case)
    room = pages_of(case["length"] + (n if kind == "append" else 0), ps)
    held = sum(pages_of(x + (n if kind == "append" else 0), ps) for x in lens)
    total = held + 3
    order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((batch, max(1, room)), -1, dtype=torch.int32, device="cuda")
    first = 0
    for s, x in enumerate(lens):
        c = pages_of(x + (n if kind == "append" else 0), ps)
        table[s, :c] = order[first:first + c]
        first += c
    lengths = torch.tensor(lens, dtype=torch.int32, device="cuda")
    state = dict(kind=kind, table=table, lengths=lengths)
    if kind == "append":
        layers = case["layers"]
        state["k_pages"] = random(gen, layers, total, hkv, ps, d, dtype=ct)
        state["v_pages"] = random(gen, layers, total, hkv, ps, d, dtype=ct)
        state["k_means"] = state["k_pages"].float().mean(3)
        state["k"] = random(gen, layers, batch, n, hkv, d, dtype=at)
        state["v"] = random(gen, layers, batch, n, hkv, d, dtype=at)
        # the accepted path of each tree: ascending drafted tokens, some trees with fewer, behind them -1
        picked = random(gen, batch, n).argsort(1)[:, :case["accept"]].sort(1).values.to(torch.int32)
        some = torch.arange(batch, device="cuda") % (case["accept"] + 1)
        keep = torch.arange(case["accept"], device="cuda") < (case["accept"] - some)[:, None]
        state["rows"] = torch.where(keep, picked, -1)
        return state

    h = case["heads"]
    # q, k, v as a projection leaves them: side by side in one row a token
    qkv = random(gen, batch, n, (h + 2 * hkv) * d, dtype=at)
    state["q"] = qkv[..., :h * d].view(batch, n, h, d)
    state["k"] = qkv[..., h * d:(h + hkv) * d].view(batch, n, hkv, d)
    state["v"] = qkv[..., (h + hkv) * d:].view(batch, n, hkv, d)
    state["parents"] = tree_of(gen, batch, n) if n > 1 else None
    k = random(gen, total, hkv, ps, d, dtype=ct)
    if kind == "sparse":   # pages about different things: a common part in the keys of a page
        k += random(gen, total, hkv, 1, d, dtype=ct)
        state["k_means"] = k.float().mean(2)
        state["top"] = case["top"]
    state["k_pages"], state["v_pages"] = k, random(gen, total, hkv, ps, d, dtype=ct)
    return state


# -- one pass -------------------------------------------------------------------------------------


def ancestors(parents, batch, n, device):
    """[batch, n, n]: token j is token i or one that i follows. Products of the parent matrix with
    itself double the distance covered."""
    eye = torch.eye(n, device=device).expand(batch, n, n)
    if parents is None:
        return eye > 0
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


def plain_tree(q, k, v, k_pages, v_pages, table, lengths, parents):
    batch, n, h, d = q.shape
    hkv, ps = k_pages.shape[1], k_pages.shape[2]
    at = table.long().clamp(min=0)
    here = torch.arange(at.shape[1] * ps, device=q.device) < lengths[:, None]                        # [S, T]

    def keys(pages, new):
        cached = pages[at].float().permute(0, 2, 1, 3, 4).reshape(batch, hkv, -1, d)
        cached = torch.where(here[:, None, :, None], cached, 0.0)
        return torch.cat([cached, new.to(pages.dtype).float().transpose(1, 2)], 2)                    # [S, Hkv, T + N, D]

    rows = q.float().view(batch, n, hkv, h // hkv, d).permute(0, 2, 1, 3, 4).reshape(batch, hkv, -1, d)
    scores = (rows @ keys(k_pages, k).transpose(2, 3).contiguous()) * (1.0 / math.sqrt(d))
    tree = ancestors(parents, batch, n, q.device)
    ok = torch.cat([here[:, None, :].expand(batch, n, -1), tree], 2)                                  # [S, N, T + N]
    ok = ok.repeat_interleave(h // hkv, 1)[:, None]
    out = softmax_product(scores, ok, keys(v_pages, v))
    return out.view(batch, hkv, n, h // hkv, d).permute(0, 2, 1, 3, 4).reshape(batch, n, h, d).to(q.dtype)


def plain_select(q, k_means, table, lengths, ps, top):
    batch, n, h, d = q.shape
    hkv = k_means.shape[1]
    width = table.shape[1]
    rows = q.double().view(batch, n, hkv, h // hkv, d).sum(3).permute(0, 2, 1, 3)                     # [S, Hkv, N, D]
    means = k_means[table.long().clamp(min=0)].double().permute(0, 2, 3, 1).contiguous()              # [S, Hkv, D, W]
    scores = rows @ means
    held = (lengths.long() + ps - 1) // ps
    index = torch.arange(width, device=q.device)
    scores = torch.where((index == held[:, None] - 1)[:, None, None], float("inf"), scores)
    scores = torch.where((index < held[:, None])[:, None, None], scores, float("-inf"))
    best = scores.sort(dim=-1, descending=True, stable=True)
    picked = torch.where(best.values > float("-inf"), best.indices, width)[..., :top].sort(-1).values
    picked = torch.where(picked < width, picked, -1)
    if picked.shape[-1] < top:
        picked = torch.cat([picked, picked.new_full((batch, hkv, n, top - picked.shape[-1]), -1)], -1)
    return picked.permute(0, 2, 1, 3).to(torch.int32)                                                 # [S, N, Hkv, top]


def plain_selected(q, k, v, k_pages, v_pages, table, lengths, selected, parents):
    batch, n, h, d = q.shape
    hkv, ps = k_pages.shape[1], k_pages.shape[2]
    top = selected.shape[-1]
    sel = selected.long()
    at = table.long().clamp(min=0).gather(1, sel.clamp(min=0).reshape(batch, -1)).view(batch, n, hkv, top)
    head = torch.arange(hkv, device=q.device)[:, None]
    token = sel[..., None] * ps + torch.arange(ps, device=q.device)                                    # [S, N, Hkv, top, ps]
    here = ((sel[..., None] >= 0) & (token < lengths[:, None, None, None, None])).reshape(batch, n, hkv, -1)

    def keys(pages, new):
        cached = pages[at, head].float().view(batch, n, hkv, -1, d)
        cached = torch.where(here[..., None], cached, 0.0)
        fresh = new.to(pages.dtype).float().transpose(1, 2)[:, None].expand(batch, n, hkv, n, d)
        return torch.cat([cached, fresh], 3)

    rows = q.float().view(batch, n, hkv, h // hkv, d)
    scores = (rows @ keys(k_pages, k).transpose(3, 4).contiguous()) * (1.0 / math.sqrt(d))
    tree = ancestors(parents, batch, n, q.device)[:, :, None].expand(batch, n, hkv, n)
    ok = torch.cat([here, tree], 3)[..., None, :]
    out = softmax_product(scores, ok, keys(v_pages, v))
    return out.reshape(batch, n, h, d).to(q.dtype)


def plain_append(k, v, k_pages, v_pages, table, lengths, rows, k_means):
    count, ps = rows.shape[1], k_pages.shape[3]
    start = lengths.long()[:, None]
    kept = rows >= 0                                                                                   # [S, A]
    place = start + torch.arange(count, device=k.device)
    page, slot = table.long().gather(1, place // ps), place % ps
    seq = torch.arange(len(rows), device=k.device)[:, None]
    for pages, new in ((k_pages, k), (v_pages, v)):
        there = pages[:, page, :, slot]                      # what is not kept gets back what is there
        new = new[:, seq, rows.long().clamp(min=0)].to(pages.dtype).permute(1, 2, 0, 3, 4)
        pages[:, page, :, slot] = torch.where(kept[:, :, None, None, None], new, there)
    # the means of the touched pages, over the tokens each then holds
    end = start + kept.sum(1, keepdim=True)
    index = start // ps + torch.arange((count - 1) // ps + 2, device=k.device)                         # [S, J]
    index = torch.where(index * ps < end, index, start // ps)
    page = table.long().gather(1, index.clamp(max=table.shape[1] - 1))
    held = (end - index * ps).clamp(1, ps)
    inside = torch.arange(ps, device=k.device) < held[..., None]
    total = torch.where(inside[..., None, :, None], k_pages[:, page].float(), 0.0).sum(4)
    means = torch.where((end > start)[..., None, None], total / held[..., None, None], k_means[:, page])
    k_means[:, page] = means


def run(state):
    kind = state["kind"]
    if kind == "copy":
        if own:
            kiln().copy_pages([state["k_pages"], state["v_pages"]], state["source"], state["target"])
        else:
            for pages in (state["k_pages"], state["v_pages"]):
                pages[:, state["target"]] = pages[:, state["source"]]
        return state["k_pages"], state["v_pages"]
    if kind == "append":
        args = [state[x] for x in ("k", "v", "k_pages", "v_pages", "table", "lengths", "rows", "k_means")]
        if own:
            kiln().cache_append(*args[:6], rows=args[6], k_means=args[7])
        else:
            plain_append(*args)
        return state["k_pages"], state["v_pages"], state["k_means"]
    args = [state[x] for x in ("q", "k", "v", "k_pages", "v_pages", "table", "lengths")]
    if kind == "tree":
        if own:
            return kiln().tree_attention(*args, state["parents"])
        return plain_tree(*args, state["parents"])
    page, top = state["k_pages"].shape[2], state["top"]
    if own:
        package = kiln()
        selected = package.select_pages(state["q"], state["k_means"], state["table"], state["lengths"],
                                        page_size=page, pages=top)
        return package.selected_attention(*args, selected, state["parents"]), selected
    selected = plain_select(state["q"], state["k_means"], state["table"], state["lengths"], page, top)
    return plain_selected(*args, selected, state["parents"]), selected


# -- what a pass cannot do without ------------------------------------------------------------------


def work(case):
    kind, hkv, d, ps = case["kind"], case["kv_heads"], case["dim"], case["page"]
    cb = BYTES[case["cache"]]
    if kind == "copy":
        return {"bytes": 2 * 2 * case["layers"] * case["moved"] * hkv * ps * d * cb, "flops": 0}
    ab = BYTES[case["act"]]
    batch, n = case["batch"], case["draft"]
    lens = lengths_of(case)
    if kind == "append":
        # new rows read and written, the touched pages' other rows read for the means, the means written
        total, touched, rest = 0, 0, 0
        for s, x in enumerate(lens):
            c = case["accept"] - s % (case["accept"] + 1)
            total += c
            if c:
                touched += (x + c - 1) // ps - x // ps + 1
                rest += x % ps
        row = hkv * d
        return {"bytes": case["layers"] * row * (2 * total * (ab + cb) + rest * cb + touched * 4),
                "flops": case["layers"] * row * (total + rest)}
    h = case["heads"]
    own_bytes = batch * n * d * ab * (2 * h + 2 * hkv)
    if kind == "tree":
        cached = sum(lens) * hkv * d
        return {"bytes": 2 * cached * cb + own_bytes, "flops": 4 * cached * n * (h // hkv) + 2 * batch * n * n * h * d}
    pages = sum(pages_of(x, ps) for x in lens)
    picked = sum(min(pages_of(x, ps), case["top"]) for x in lens) * ps
    # the picked pages of one sequence are at most its cache: drafted tokens may share them
    cached = sum(min(n * min(pages_of(x, ps), case["top"]), pages_of(x, ps)) for x in lens) * ps * hkv * d
    return {"bytes": 2 * cached * cb + pages * hkv * d * 4 + own_bytes + batch * n * hkv * case["top"] * 4,
            "flops": 4 * picked * n * h * d + 2 * pages * n * hkv * d}


# -- the definitions, in 64 bits ---------------------------------------------------------------------


def exact(case, seed):
    state = prepare(case, seed)
    kind, ps = case["kind"], case["page"]
    if kind == "copy":
        k, v = state["k_pages"].double(), state["v_pages"].double()
        for i, o in zip(state["source"], state["target"]):   # no page is both a source and a target
            k[:, o], v[:, o] = k[:, i], v[:, i]
        return k, v
    table, lens = state["table"].tolist(), lengths_of(case)
    if kind == "append":
        k, v, m = state["k_pages"].double(), state["v_pages"].double(), state["k_means"].double()
        ct = DTYPES[case["cache"]]
        rows = state["rows"].tolist()
        for s, x in enumerate(lens):
            path = [r for r in rows[s] if r >= 0]
            for i, r in enumerate(path):
                page, slot = table[s][(x + i) // ps], (x + i) % ps
                k[:, page, :, slot] = state["k"][:, s, r].to(ct).double()
                v[:, page, :, slot] = state["v"][:, s, r].to(ct).double()
            for b in range(x // ps, pages_of(x + len(path), ps)) if path else ():
                m[:, table[s][b]] = k[:, table[s][b], :, :min(ps, x + len(path) - b * ps)].mean(2)
        return k, v, m
    q, parents = state["q"].double(), state["parents"]
    batch, n, h, d = q.shape
    hkv = case["kv_heads"]
    g = h // hkv
    ct = DTYPES[case["cache"]]
    out = torch.zeros(batch, n, h, d, dtype=torch.float64, device="cuda")
    picked = torch.full((batch, n, hkv, case.get("top", 1)), -1, dtype=torch.int32)
    for s, x in enumerate(lens):
        follows = [-1] * n if parents is None else parents[s].tolist()
        see = torch.zeros(n, n, dtype=torch.bool)
        for i in range(n):
            j = i
            while j >= 0:
                see[i, j] = True
                j = follows[j]
        see = see.cuda()
        held = table[s][:pages_of(x, ps)]
        kc = state["k_pages"][held].double()                     # [pages, Hkv, ps, D]
        vc = state["v_pages"][held].double()
        new_k, new_v = state["k"][s].to(ct).double(), state["v"][s].to(ct).double()
        if kind == "tree":
            kc, vc = (t.transpose(0, 1).reshape(hkv, -1, d)[:, :x] for t in (kc, vc))
            for head in range(h):
                kk = torch.cat([kc[head // g], new_k[:, head // g]])
                vv = torch.cat([vc[head // g], new_v[:, head // g]])
                a = (q[s, :, head] @ kk.T) / math.sqrt(d)
                a[:, x:] = a[:, x:].masked_fill(~see, -math.inf)
                out[s, :, head] = torch.softmax(a, 1) @ vv
            continue
        kept = len(held)
        for c in range(hkv):
            group = slice(c * g, (c + 1) * g)
            score = (q[s, :, group].sum(1) @ state["k_means"][held, c].double().T).cpu().tolist()   # [N, pages]
            for i in range(n):
                order = sorted(range(kept), key=lambda b: (b != kept - 1, -score[i][b], b))
                choice = sorted(order[:case["top"]])
                picked[s, i, c, :len(choice)] = torch.tensor(choice, dtype=torch.int32)
                tokens = sum(min(ps, x - b * ps) for b in choice)      # the last page's are the last ones
                kk = torch.cat([kc[choice, c].reshape(-1, d)[:tokens], new_k[see[i], c]])
                vv = torch.cat([vc[choice, c].reshape(-1, d)[:tokens], new_v[see[i], c]])
                a = (q[s, i, group] @ kk.T) / math.sqrt(d)
                out[s, i, group] = torch.softmax(a, 1) @ vv
    return out if kind == "tree" else (out, picked.cuda())
