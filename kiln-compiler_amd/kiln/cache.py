"""``kiln.PagedCache``: the keys and values of many sequences in pages.

    cache = kiln.PagedCache(layers=12, pages=4096, page_size=16, kv_heads=12, dim=64)
    seq = cache.open()
    table, lengths = cache.batch([seq])
    y = kiln.tree_attention(q, k, v, cache.k[layer], cache.v[layer], table, lengths, parents)
    cache.append([seq], k_all, v_all, rows=[[0, 2, 5]])       # the accepted path, every layer

A page holds ``page_size`` tokens of one sequence in every layer. Which pages
a sequence has, and how many of their tokens, is kept on the host; a page may
belong to several sequences (``fork`` shares pages and copies none), and is
copied when one of them writes to it. The device work - appending, copying
pages - is ``kiln.cache_append`` and ``kiln.copy_pages`` on the current
stream; a caller that works on several streams orders them itself, as for any
tensor. Calls that need more pages than are free raise MemoryError and change
nothing. A graph being captured would replay device work without its
book-keeping: ``batch``, ``append`` and ``compact`` refuse that (the operators
on tables made before can be captured). Not thread-safe.
"""

from __future__ import annotations

import heapq
import operator

import torch

from kiln.hip import paged
from kiln.hip.interpret import interpreting


class PagedCache:
    """The pages ``k`` and ``v`` ``[layers, pages, kv_heads, page_size, dim]``,
    with ``means=True`` the pages' mean keys ``means`` ``[layers, pages,
    kv_heads, dim]`` (what ``select_pages`` reads), and their book-keeping.
    ``dtype``: fp32, bf16, fp16, or ``torch.float4_e2m1fn_x2`` for pages of 4
    bits (uint8 ``[layers, pages, kv_heads, page_size, 17 * dim // 32]``: codes
    and the scales of every 32 dimensions, kiln/hip/paged.py)."""

    def __init__(self, layers, pages, page_size, kv_heads, dim, dtype=torch.bfloat16, means=False, device=None):
        for name, n in (("layers", layers), ("pages", pages), ("kv_heads", kv_heads)):
            if n < 1:
                raise ValueError(f"{name} must be at least 1, got {n}")
        packed = dtype == torch.float4_e2m1fn_x2
        if dtype not in paged.TYPES and not packed:
            raise TypeError(f"dtype must be one of {', '.join(map(str, paged.TYPES))}, {torch.float4_e2m1fn_x2}, got {dtype}")
        if page_size < 16 or page_size > 1024 or page_size & (page_size - 1):
            raise NotImplementedError(f"page_size {page_size}: powers of two from 16 to 1024 have kernels")
        if dim < 8 or dim % 8 or dim > 256:
            raise NotImplementedError(f"dim {dim}: multiples of 8 up to 256 have kernels")
        if packed and dim % paged.BLOCK:
            raise NotImplementedError(f"dim {dim}: multiples of {paged.BLOCK} up to 256 have kernels over 4-bit pages")
        row = dim // paged.BLOCK * paged.BLOCK_BYTES if packed else dim   # elements of a token's row
        if device is None:
            from kiln.hip.runtime import device as gpu

            device = torch.device("cpu") if interpreting() else gpu()
        self.device = torch.device(device)
        if self.device.type == "cuda":
            from kiln.hip.runtime import check_memory

            size = 1 if packed else torch.empty(0, dtype=dtype).element_size()
            need = layers * pages * kv_heads * (2 * page_size * size * row + (4 * dim if means else 0))
            check_memory(self.device, need, f"the cache's {pages} pages")
        self.page_size = page_size
        self.pages = pages
        self.dim = dim
        self.k = torch.zeros((layers, pages, kv_heads, page_size, row), dtype=torch.uint8 if packed else dtype,
                             device=self.device)
        self.device = self.k.device              # ("cuda" alone follows the current device)
        self.v = torch.zeros_like(self.k)
        self.means = torch.zeros((layers, pages, kv_heads, dim), dtype=torch.float32, device=self.device) if means else None
        self._free = list(range(pages))          # a heap: the lowest free page is taken first
        self._refs = [0] * pages                 # sequences that have the page
        self._pages = {}                         # sequence -> its pages, in order
        self._length = {}                        # sequence -> its tokens
        self._gone = {}                          # sequence -> the tokens before this one may be released
        self._next = 0

    # -- sequences ----------------------------------------------------------------------

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def length(self, seq) -> int:
        return self._length[self._known(seq)]

    def pages_of(self, seq) -> tuple:
        """The sequence's pages, in order; -1 for those that were released."""
        return tuple(self._pages[self._known(seq)])

    def _known(self, seq):
        if seq not in self._pages:
            raise ValueError(f"no sequence {seq!r} in this cache")
        return seq

    def open(self) -> int:
        """A new, empty sequence."""
        seq, self._next = self._next, self._next + 1
        self._pages[seq], self._length[seq], self._gone[seq] = [], 0, 0
        return seq

    def fork(self, seq, n=1) -> list:
        """``n`` new sequences with the tokens of ``seq``, on the same pages."""
        self._known(seq)
        if n < 0:
            raise ValueError(f"cannot fork {n} times")
        made = []
        for _ in range(n):
            new = self.open()
            self._pages[new] = list(self._pages[seq])
            self._length[new], self._gone[new] = self._length[seq], self._gone[seq]
            for page in self._pages[new]:
                if page >= 0:
                    self._refs[page] += 1
            made.append(new)
        return made

    def _drop(self, page):
        if page < 0:
            return
        self._refs[page] -= 1
        if not self._refs[page]:
            heapq.heappush(self._free, page)

    def free(self, seq):
        """Forget ``seq``; its pages that no other sequence has become free."""
        for page in self._pages[self._known(seq)]:
            self._drop(page)
        del self._pages[seq], self._length[seq], self._gone[seq]

    def truncate(self, seq, length):
        """Keep the first ``length`` tokens of ``seq``. Where pages were
        released, only so far back that the window of the next token still
        holds what it held."""
        if not 0 <= length <= self._length[self._known(seq)]:
            raise ValueError(f"cannot keep {length} of {self._length[seq]} tokens")
        if 0 < length < self._gone[seq]:
            raise ValueError(f"cannot keep {length} tokens: pages of the window before them were released")
        keep = -(-length // self.page_size)
        for page in self._pages[seq][keep:]:
            self._drop(page)
        del self._pages[seq][keep:]
        self._length[seq] = length
        if not length:
            self._gone[seq] = 0

    def release(self, seq, *, window, sinks=0):
        """Give back the pages of ``seq`` that no token appended from now on
        can see through ``tree_attention(..., window=window, sinks=sinks)``:
        those behind the window of the next token, but for the first
        ``sinks`` tokens'. Its length stays; ``batch`` names -1 in their place,
        and ``read`` gives zeros."""
        have = self._pages[self._known(seq)]
        window, sinks = operator.index(window), operator.index(sinks)
        if window < 1 or sinks < 0:
            raise ValueError(f"a window of {window} tokens and {sinks} sinks")
        first = self._length[seq] - window + 1           # the next token's first key
        for column in range(-(-sinks // self.page_size), max(0, first) // self.page_size):
            if have[column] >= 0:
                self._drop(have[column])
                have[column] = -1
                self._gone[seq] = self._length[seq]

    def _not_captured(self, what):
        if self.device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            raise RuntimeError(f"PagedCache.{what} while a graph is captured: its replay would not repeat the "
                               f"book-keeping; call it before, or between replays")

    # -- the device's view ------------------------------------------------------------------

    def batch(self, seqs, columns=None):
        """(table, lengths) of the sequences, as the operators take them: int32
        ``[sequences, columns]`` (as many as the longest needs, or ``columns``)
        and ``[sequences]``, uploaded without waiting for the device."""
        self._not_captured("batch")
        rows = [self._pages[self._known(s)] for s in seqs]
        need = max([1] + [len(r) for r in rows])
        columns = need if columns is None else columns
        if columns < need:
            raise ValueError(f"{need} columns are needed, got {columns}")
        table = torch.full((len(rows), columns), -1, dtype=torch.int32)
        for i, r in enumerate(rows):
            if r:
                table[i, :len(r)] = torch.tensor(r, dtype=torch.int32)
        lengths = torch.tensor([self._length[s] for s in seqs], dtype=torch.int32)
        return self._upload(table), self._upload(lengths)

    def _upload(self, t):
        # (torch's pinned allocator keeps the block until the copy has run)
        return t.pin_memory().to(self.device, non_blocking=True) if self.device.type == "cuda" else t

    # -- tokens ----------------------------------------------------------------------------------

    def _pools(self):
        return [self.k, self.v] + ([self.means.unsqueeze(-2)] if self.means is not None else [])

    def append(self, seqs, k, v, rows=None):
        """Tokens written behind those of ``seqs``, in every layer: all of ``k``
        and ``v`` ``[layers, sequences, tokens, kv_heads, dim]``, or of sequence
        i the tokens ``rows[i]`` (a list of ints: a drafted tree's accepted
        path). Pages are taken as needed; a page that other sequences have too
        is copied before it is written to."""
        self._not_captured("append")
        seqs = list(seqs)
        if len(set(seqs)) != len(seqs):
            raise ValueError("a sequence is named twice")
        for s in seqs:
            self._known(s)
        layers, _, kv_heads, _, _ = self.k.shape
        dim = self.dim
        if k.dim() != 5 or tuple(k.shape) != (layers, len(seqs), k.shape[2], kv_heads, dim):
            raise ValueError(f"k must have shape ({layers}, {len(seqs)}, tokens, {kv_heads}, {dim}), got {tuple(k.shape)}")
        if v.shape != k.shape or v.dtype != k.dtype:
            raise ValueError("v must be shaped and typed as k")
        tokens = k.shape[2]
        if rows is None:
            counts = [tokens] * len(seqs)
        else:
            rows = [list(r) for r in rows]
            if len(rows) != len(seqs):
                raise ValueError(f"{len(rows)} lists of rows for {len(seqs)} sequences")
            if any(not 0 <= r < tokens for path in rows for r in path):
                raise ValueError(f"a row is outside the {tokens} tokens")
            counts = [len(r) for r in rows]
        if not any(counts):
            return
        # the pages to come: new ones, and copies of shared ones that are written to
        taken, source, target, plans = [], [], [], []
        refs = {}

        def take():
            if not self._free:
                raise MemoryError(f"the cache has no free page left ({self.pages} pages)")
            taken.append(heapq.heappop(self._free))
            return taken[-1]

        try:
            for s, n in zip(seqs, counts):
                have = list(self._pages[s])
                at = self._length[s] // self.page_size
                if n and at < len(have):           # the last page has room (only it can: truncate drops those behind)
                    old = have[at]
                    if refs.setdefault(old, self._refs[old]) > 1:
                        refs[old] -= 1
                        have[at] = take()
                        source.append(old)
                        target.append(have[at])
                while len(have) * self.page_size < self._length[s] + n:
                    have.append(take())
                plans.append(have)
            table = torch.full((len(seqs), max(len(p) for p in plans)), -1, dtype=torch.int32)
            for i, p in enumerate(plans):
                table[i, :len(p)] = torch.tensor(p, dtype=torch.int32)
            lengths = torch.tensor([self._length[s] for s in seqs], dtype=torch.int32)
            path = None
            if rows is not None:
                path = torch.full((len(seqs), max(counts)), -1, dtype=torch.int32)
                for i, r in enumerate(rows):
                    if r:
                        path[i, :len(r)] = torch.tensor(r, dtype=torch.int32)
                path = self._upload(path)
            if source:
                paged.copy_pages(self._pools(), source, target)
            paged.cache_append(k, v, self.k, self.v, self._upload(table), self._upload(lengths), rows=path,
                               k_means=self.means)
        except BaseException:
            for page in taken:                 # nothing names them yet
                heapq.heappush(self._free, page)
            raise
        for page in source:
            self._refs[page] -= 1
        for page in taken:
            self._refs[page] = 1
        for s, n, have in zip(seqs, counts, plans):
            self._pages[s] = have
            self._length[s] += n

    def read(self, seqs, dtype=None):
        """The tokens of ``seqs`` as dense tensors ``(k, v)``, ``[layers,
        sequences, longest, kv_heads, dim]``, zeros behind each one's last:
        what ``append`` takes, of another cache too. ``dtype`` as for
        ``kiln.cache_read``."""
        seqs = list(seqs)
        table, lengths = self.batch(seqs)
        return paged.cache_read(self.k, self.v, table, torch.zeros_like(lengths), lengths,
                                tokens=max([0] + [self._length[s] for s in seqs]), dtype=dtype)

    # -- pages --------------------------------------------------------------------------------------

    def compact(self) -> int:
        """Move the pages in use to the front of the pool; returns how many
        there are. Tables made before by ``batch`` name the old places."""
        self._not_captured("compact")
        used = self.pages - len(self._free)
        holes = sorted(p for p in self._free if p < used)
        moved = [p for p in range(used, self.pages) if self._refs[p]]
        if moved:
            paged.copy_pages(self._pools(), moved, holes)
            place = dict(zip(moved, holes))
            for seq, have in self._pages.items():
                self._pages[seq] = [place.get(p, p) for p in have]   # (-1 stays)
            for old, new in place.items():
                self._refs[new], self._refs[old] = self._refs[old], 0
        self._free = list(range(used, self.pages))
        return used
