"""The decoding step's further operators in 64 bits, from their definitions, with
loops: blocks of 4 bits, windows, and the verification of drafted tokens."""

import math

import torch

LEVELS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def block(x):
    """(codes, scale byte) of 32 numbers."""
    x = [float(a) for a in x]
    if not all(math.isfinite(a) for a in x):
        return [0] * 32, 255
    largest, e = max(map(abs, x)), 2
    while largest >= 7 * 2.0 ** (e - 127) and e < 252:
        e += 1
    codes = []
    for a in x:
        y = abs(a) / 2.0 ** (e - 127)
        codes.append(min(range(8), key=lambda c: (abs(y - LEVELS[c]), c % 2)) + 8 * (math.copysign(1, a) < 0))
    return codes, e


def values(codes, e):
    if e > 252:
        return [math.nan] * 32
    return [(-1 if c > 7 else 1) * LEVELS[c % 8] * 2.0 ** (e - 127) for c in codes]


def rounded(x):
    """x [..., dim] as 4-bit pages hold it, float64."""
    flat = x.double().reshape(-1, 32)
    return torch.tensor([values(*block(row)) for row in flat.tolist()], dtype=torch.float64).view(x.shape)


def places(t, d, dim, page, keys):
    """(code byte, scale byte) of element (t, d) inside a page of a head."""
    if keys:
        return t * dim // 2 + d // 2, page * dim // 2 + t * (dim // 32) + d // 32
    return (t // 16 * 8 * dim + (t % 16 // 4 * (dim // 8) + d // 8) * 16 + t % 4 * 4 + d % 8 // 2,
            page * dim // 2 + t // 16 * (dim // 2) + (t % 16 // 4 * (dim // 32) + d // 32) * 4 + t % 4)


def pack(x, keys):
    """x [..., page, dim] as uint8 pages [..., page, 17 dim / 32]."""
    page, dim = x.shape[-2:]
    out = torch.zeros(*x.shape[:-2], page * 17 * dim // 32, dtype=torch.uint8)
    for one, to in zip(x.double().reshape(-1, page, dim), out.view(-1, page * 17 * dim // 32)):
        store(to.view(page, -1), one, range(page), keys)
    return out.view(*x.shape[:-2], page, 17 * dim // 32)


def store(page, rows, slots, keys):
    """rows [n, dim] into the slots of one page of a head."""
    to, size = page.reshape(-1), page.shape[0]
    dim = rows.shape[1]
    for t, row in zip(slots, rows.tolist()):
        for b in range(0, dim, 32):
            codes, e = block(row[b:b + 32])
            to[places(t, b, dim, size, keys)[1]] = e
            for d, c in enumerate(codes, b):
                at = places(t, d, dim, size, keys)[0]
                to[at] = (int(to[at]) & 15 | c << 4) if d % 2 else (int(to[at]) & 240 | c)


def unpack(pages, keys):
    """float64 values of uint8 pages [..., page, 17 dim / 32]."""
    page, dim = pages.shape[-2], pages.shape[-1] // 17 * 32
    flat = pages.cpu().reshape(-1, page * 17 * dim // 32)
    t, d = torch.arange(page)[:, None], torch.arange(dim)[None]
    code, scale = places(t, d, dim, page, keys)
    c, e = flat[:, code].long() >> 4 * (d % 2) & 15, flat[:, scale].double()
    x = torch.tensor(LEVELS, dtype=torch.float64)[c % 8] * torch.where(c > 7, -1.0, 1.0) * 2.0 ** (e - 127)
    return torch.where(e > 252, math.nan, x).view(*pages.shape[:-1], dim)


def stored(x, dtype):
    return rounded(x) if dtype == torch.uint8 else x.to(dtype).double()


def paths(parents, n):
    """Each token's path as a list, None where it is unused."""
    out = []
    for i in range(n):
        up = i - 1 if parents is None else int(parents[i])
        before = [] if up == -1 else out[up] if 0 <= up < i else None
        out.append(None if before is None else before + [i])
    return out


def attention(q, k, v, k_pages, v_pages, table, lengths, parents=None, scale=None, window=None, sinks=0, selected=None):
    """float64 [sequences, tokens, heads, dim], over pages of any type."""
    q, k, v, table, lengths = (t.cpu() for t in (q, k, v, table, lengths))
    new_k, new_v = stored(k, k_pages.dtype), stored(v, v_pages.dtype)
    if k_pages.dtype == torch.uint8:
        k_pages, v_pages = unpack(k_pages, True), unpack(v_pages, False)
    k_pages, v_pages = k_pages.cpu().double(), v_pages.cpu().double()
    batch, n, heads, dim = q.shape
    pages, kv, ps, _ = k_pages.shape
    scale = 1.0 / math.sqrt(dim) if scale is None else scale
    out = torch.zeros(batch, n, heads, dim, dtype=torch.float64)
    for s in range(batch):
        length = max(0, min(int(lengths[s]), table.shape[1] * ps))
        for i, path in enumerate(paths(None if parents is None else parents[s].tolist(), n)):
            if path is None:
                continue
            mine = length + len(path) - 1
            def seen(p):
                return window is None or p < sinks or p > mine - window

            for c in range(kv):
                columns = range(-(-length // ps))
                if selected is not None:
                    row = [-1, *map(int, selected[s, i, c])]
                    columns = [b for a, b in zip(row, row[1:]) if b > a and 0 <= b < table.shape[1]]
                spots = [(int(table[s, b]), t) for b in columns if 0 <= int(table[s, b]) < pages
                         for t in range(ps) if b * ps + t < length and seen(b * ps + t)]
                at = [p for p, _ in spots], [t for _, t in spots]
                own = [j for a, j in enumerate(path) if seen(length + a)]
                kk = torch.cat([k_pages[at[0], c, at[1]], new_k[s, own, c]])
                vv = torch.cat([v_pages[at[0], c, at[1]], new_v[s, own, c]])
                for h in range(c * (heads // kv), (c + 1) * (heads // kv)):
                    w = torch.softmax((kk @ q[s, i, h].double()) * scale, 0)
                    out[s, i, h] = w @ vv
    return out


def problem(gen, cache=torch.uint8, act=torch.float32, device="cpu", **sizes):
    """As paged_reference.problem; with 4-bit pages where `cache` is uint8."""
    import paged_reference

    p = paged_reference.problem(gen, cache=torch.float32 if cache == torch.uint8 else cache, act=torch.float32, **sizes)
    for name in ("q", "k", "v"):
        p[name] = p[name].to(act)
    if cache == torch.uint8:
        p["k_pages"], p["v_pages"] = fast_pack(p["k_pages"], True), fast_pack(p["v_pages"], False)
    return {name: t.to(device) for name, t in p.items()}


def fast_pack(x, keys):
    """Pages of random codes and scales near those of normal values (x gives the shape alone where large)."""
    if x.numel() <= 20000:
        return pack(x, keys)
    page, dim = x.shape[-2:]
    g = torch.Generator().manual_seed(x.numel())
    codes = torch.randint(0, 256, (*x.shape[:-2], page * dim // 2), generator=g, dtype=torch.uint8)
    scales = torch.randint(124, 128, (*x.shape[:-2], page * dim // 32), generator=g, dtype=torch.uint8)
    return torch.cat([codes, scales], -1).view(*x.shape[:-2], page, 17 * dim // 32)


def append(k, v, k_pages, v_pages, table, lengths, rows=None, k_means=None):
    """(k_pages, v_pages, k_means) after the call, 4-bit pages of 5 dimensions."""
    k_pages, v_pages = k_pages.cpu().clone(), v_pages.cpu().clone()
    k_means = None if k_means is None else k_means.cpu().double().clone()
    k, v, table, lengths = k.cpu(), v.cpu(), table.cpu(), lengths.cpu()
    layers, batch, n, kv, dim = k.shape
    pages, ps = k_pages.shape[1], k_pages.shape[3]
    for s in range(batch):
        path = list(range(n)) if rows is None else rows[s].tolist()
        touched = {}
        for a, r in enumerate(path):
            if not 0 <= r < n or int(lengths[s]) < 0:
                break
            column, slot = divmod(int(lengths[s]) + a, ps)
            if column >= table.shape[1] or not 0 <= int(table[s, column]) < pages:
                continue
            p = int(table[s, column])
            for layer in range(layers):
                for c in range(kv):
                    store(k_pages[layer, p, c], k[layer, s, r, c][None].double(), [slot], True)
                    store(v_pages[layer, p, c], v[layer, s, r, c][None].double(), [slot], False)
            touched[p] = slot + 1
        for p, m in touched.items():
            if k_means is not None:
                k_means[:, p] = unpack(k_pages[:, p], True)[:, :, :m].mean(2)
    return k_pages, v_pages, k_means


def read(k_pages, v_pages, table, starts, ends, tokens):
    """float64 (k, v) [layers, sequences, tokens, kv_heads, dim] of pages of 5 dimensions."""
    if k_pages.dtype == torch.uint8:
        k_pages, v_pages = unpack(k_pages, True), unpack(v_pages, False)
    k_pages, v_pages, table = k_pages.cpu().double(), v_pages.cpu().double(), table.cpu()
    layers, pages, kv, ps, dim = k_pages.shape
    k, v = (torch.zeros(layers, len(table), tokens, kv, dim, dtype=torch.float64) for _ in "kv")
    for s in range(len(table)):
        for a in range(tokens):
            p = int(starts[s]) + a
            if 0 <= p < int(ends[s]) and p // ps < table.shape[1] and 0 <= int(table[s, p // ps]) < pages:
                k[:, s, a] = k_pages[:, int(table[s, p // ps]), :, p % ps]
                v[:, s, a] = v_pages[:, int(table[s, p // ps]), :, p % ps]
    return k, v


def weights(row):
    x = row.double().cpu()
    return torch.where(x > 0, x, 0.0)


def drawn(w, u):
    """The first index whose running sum passes u of the whole."""
    whole = float(w.sum())
    if not whole < math.inf or whole <= 0:
        return -1
    past = (torch.cumsum(w, 0) > max(u, 0.0) * whole).nonzero()
    return int(past[0]) if len(past) else int(w.nonzero()[-1])


def verify(tokens, target, uniforms, parents=None, draft=None):
    """(rows, counts, after), lists."""
    batch, n, vocab = target.shape
    out = [], [], []
    for s in range(batch):
        follows = list(range(-1, n - 1)) if parents is None else parents[s].tolist()
        token, u = tokens[s].tolist(), uniforms[s].double().tolist()
        path, after = [], -1
        if follows[0] == -1:
            path, w, whole = [0], weights(target[s, 0]), 1.0
            choice = drawn(w, u[0])
            for i in range(1, n):
                if follows[i] != path[-1] or not 0 <= token[i] < vocab:
                    continue
                if draft is None:
                    if token[i] != choice:
                        continue
                else:
                    q = draft[s, path[-1]].double().cpu()
                    if not u[i] * whole * float(q[token[i]]) < float(w[token[i]]):
                        w = weights(w - whole * q)
                        whole = float(w.sum())
                        continue
                path.append(i)
                w, whole = weights(target[s, i]), 1.0
                choice = drawn(w, u[i])
            after = choice if draft is None else drawn(w if float(w.sum()) > 0 else weights(target[s, path[-1]]), u[0])
        out[0].append(path + [-1] * (n - len(path)))
        out[1].append(len(path))
        out[2].append(after)
    return out


def drafted(gen, batch, n, vocab, dtype=torch.float32, tree=True, probs=True, noise=0.7, device="cpu", root=True):
    """Operands of verify_tokens: a noisy draft's tokens, so that some are kept and some are not."""
    target = 2 * torch.randn(batch, n, vocab, generator=gen)
    draft = (target + noise * torch.randn(batch, n, vocab, generator=gen)).softmax(-1).to(dtype)
    target = target.softmax(-1).to(dtype)
    parents = None
    up = (torch.arange(n) - 1).clamp(min=0).expand(batch, n)
    if tree:
        back = 1 + (torch.randn(batch, n, generator=gen).abs() * 2).long()
        up = (torch.arange(n) - back).clamp(min=0)
        parents = up.to(torch.int32).clone()
        parents[:, 0] = -1
    rows = draft[torch.arange(batch)[:, None], up].float()
    tokens = torch.multinomial(rows.flatten(0, 1), 1, generator=gen).view(batch, n)
    p = dict(tokens=tokens, target=target, uniforms=torch.rand(batch, n, generator=gen), parents=parents,
             draft=draft if probs else None)
    return {name: None if t is None else t.to(device) for name, t in p.items()}
