"""Kiln: an inference compiler for PyTorch models, with an MI355X (gfx950) backend.

    import kiln
    compiled = kiln.compile(model, (example_input,), device="cuda")
    y = compiled(x)

    compiled = torch.compile(model, backend=kiln.backend, dynamic=False)

    cache = kiln.PagedCache(layers, pages, page_size, kv_heads, dim)   # decoding: kiln/cache.py, kiln/hip/paged.py
    y = kiln.tree_attention(q, k, v, cache.k[0], cache.v[0], *cache.batch(seqs))

The compiler front half (IR, freeze/fusion/buffer/memory-plan passes) keeps the
reference Kiln's contracts; below it, every fused kernel runs on a hand-written
HIP kernel family from libkiln_hip.so, replayed as one hipGraph.
"""

from kiln.api import CompiledModule, Options, Report, compile, compile_graph
from kiln.backend import backend, stats
from kiln.cache import PagedCache
from kiln.hip.paged import cache_append, copy_pages, select_pages, selected_attention, tree_attention

__all__ = ["compile", "compile_graph", "Options", "Report", "CompiledModule", "backend", "stats",
           "PagedCache", "tree_attention", "select_pages", "selected_attention", "cache_append", "copy_pages"]
