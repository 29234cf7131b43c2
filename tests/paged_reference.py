"""The paged cache's operators in 64 bits, from their definitions, with loops."""

import math

import torch


def see(parents, n):
    """[n][n] bools (token i sees token j) and which tokens are used."""
    path, used = torch.zeros(n, n, dtype=torch.bool), [True] * n
    for i in range(n):
        j = i
        while j >= 0:
            path[i, j] = True
            up = j - 1 if parents is None else int(parents[j])
            if not -1 <= up < j:
                used[i] = False
                break
            j = up
    return path, used


def held(table, length, page_size, pages, selected=None):
    """[(page, slots)] of the cached tokens, in order."""
    length = max(0, min(int(length), len(table) * page_size))
    columns = range(-(-length // page_size))
    if selected is not None:
        chosen = [int(x) for x in selected]
        columns = [c for i, c in enumerate(chosen) if c > (chosen[i - 1] if i else -1) and 0 <= c < len(table)]
    out = []
    for c in columns:
        n = min(page_size, length - c * page_size)
        if n > 0 and 0 <= int(table[c]) < pages:
            out.append((int(table[c]), n))
    return out


def attention(q, k, v, k_pages, v_pages, table, lengths, parents=None, selected=None, scale=None):
    """float64 [sequences, tokens, heads, dim]"""
    q, k, v, k_pages, v_pages, table, lengths = (t.cpu() for t in (q, k, v, k_pages, v_pages, table, lengths))
    batch, n, heads, dim = q.shape
    pages, kv, ps, _ = k_pages.shape
    scale = 1.0 / math.sqrt(dim) if scale is None else scale
    out = torch.zeros(batch, n, heads, dim, dtype=torch.float64)
    new_k, new_v = k.to(k_pages.dtype).double(), v.to(k_pages.dtype).double()
    k_pages, v_pages, q = k_pages.double(), v_pages.double(), q.double()
    for s in range(batch):
        path, used = see(None if parents is None else parents[s].tolist(), n)
        for h in range(heads):
            c = h // (heads // kv)
            whole = held(table[s], lengths[s], ps, pages) if selected is None else None
            for i in range(n):
                if not used[i]:
                    continue
                spots = whole if selected is None else held(table[s], lengths[s], ps, pages, selected[s, i, c])
                kk = torch.cat([k_pages[p, c, :m] for p, m in spots] + [new_k[s, path[i], c]])
                vv = torch.cat([v_pages[p, c, :m] for p, m in spots] + [new_v[s, path[i], c]])
                w = torch.softmax((kk @ q[s, i, h]) * scale, 0)
                out[s, i, h] = w @ vv
    return out


def select(q, k_means, table, lengths, page_size, top):
    q, k_means, table, lengths = (t.cpu() for t in (q, k_means, table, lengths))
    batch, n, heads, dim = q.shape
    pages, kv, _ = k_means.shape
    out = torch.full((batch, n, kv, top), -1, dtype=torch.int32)
    for s in range(batch):
        length = max(0, min(int(lengths[s]), table.shape[1] * page_size))
        count = -(-length // page_size)
        for i in range(n):
            for c in range(kv):
                group = q[s, i, c * (heads // kv):(c + 1) * (heads // kv)].double().sum(0)
                score = []
                for b in range(count):
                    p = int(table[s, b])
                    x = float(group @ k_means[p, c].double()) if 0 <= p < pages else 0.0
                    score.append((b != count - 1, math.isnan(x), -x if not math.isnan(x) else 0.0, b))
                best = sorted(b for *_, b in sorted(score)[:top])
                out[s, i, c, :len(best)] = torch.tensor(best, dtype=torch.int32)
    return out


def append(k, v, k_pages, v_pages, table, lengths, rows=None, k_means=None):
    """(k_pages, v_pages, k_means) after the call, new tensors; 5 dimensions."""
    k_pages, v_pages = k_pages.cpu().clone(), v_pages.cpu().clone()
    k_means = None if k_means is None else k_means.cpu().double().clone()
    k, v, table, lengths = k.cpu(), v.cpu(), table.cpu(), lengths.cpu()
    layers, batch, n, kv, dim = k.shape
    pages, ps = k_pages.shape[1], k_pages.shape[3]
    for s in range(batch):
        path = list(range(n)) if rows is None else rows[s].tolist()
        length = int(lengths[s])
        touched = {}
        for a, r in enumerate(path):
            if not 0 <= r < n or length < 0:
                break
            column, slot = divmod(length + a, ps)
            if column >= table.shape[1] or not 0 <= int(table[s, column]) < pages:
                continue
            p = int(table[s, column])
            k_pages[:, p, :, slot] = k[:, s, r].to(k_pages.dtype)
            v_pages[:, p, :, slot] = v[:, s, r].to(v_pages.dtype)
            touched[p] = slot + 1
        for p, m in touched.items():
            if k_means is not None:
                k_means[:, p] = k_pages[:, p, :, :m].double().mean(2)
    return k_pages, v_pages, k_means


def problem(gen, batch=2, draft=3, heads=4, kv=2, dim=64, page=16, lengths=(40, 17), cache=torch.float32,
            act=torch.float32, spare=2, columns=None, tree=True, device="cpu"):
    """A cache with its tokens and drafted ones: a dict of operands."""
    lengths = list(lengths)
    need = [-(-max(n, 0) // page) for n in lengths]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=gen).to(torch.int32)
    columns = max([1] + need) if columns is None else columns
    table = torch.full((batch, columns), -1, dtype=torch.int32)
    at = 0
    for s, c in enumerate(need):
        table[s, :c] = order[at:at + c]
        at += c

    def normal(*shape, dtype):
        return torch.randn(*shape, generator=gen).to(dtype)

    p = dict(q=normal(batch, draft, heads, dim, dtype=act), k=normal(batch, draft, kv, dim, dtype=act),
             v=normal(batch, draft, kv, dim, dtype=act), k_pages=normal(pages, kv, page, dim, dtype=cache),
             v_pages=normal(pages, kv, page, dim, dtype=cache), table=table,
             lengths=torch.tensor(lengths, dtype=torch.int32))
    if tree:
        back = 1 + (torch.randn(batch, draft, generator=gen).abs() * 2).long()
        p["parents"] = (torch.arange(draft) - back).clamp(min=-1).to(torch.int32)
    return {name: t.to(device) for name, t in p.items()}
