"""The operators over a paged key/value cache, as functions on torch tensors.

    tree_attention      N drafted tokens a sequence over its cached tokens and
                        each other, along a tree (one token: plain decoding)
    select_pages        the pages a cheap score picks for each drafted token
    selected_attention  tree_attention over those pages alone
    cache_append        new tokens' keys and values written into the pages
    copy_pages          whole pages copied within the pools

A cache's pages are ``k_pages`` and ``v_pages``, ``[pages, kv_heads,
page_size, dim]`` in fp32, bf16 or fp16; token t of sequence s lies in page
``table[s, t // page_size]`` at slot ``t % page_size``, for ``t < lengths[s]``
(int32 both). ``kiln.PagedCache`` keeps such a cache and its book-keeping.

The first three are also what a model given to ``kiln.compile`` or
``torch.compile(backend=kiln.backend)`` may call: they are the operators
``torch.ops.kiln.paged_attention`` and ``select_pages``, which the frontend
translates. The last two change their arguments, which a compiled graph does
not; they are called between the calls of a compiled step. Where a tracer or a
dispatch mode watches (``torch.jit.trace``, ``make_fx``, a flop counter), a call
goes through its operator in ``torch.ops.kiln``, which those see;
``torch.jit.trace`` does not keep the last two, which refuse it.

Each call runs on the current stream of its tensors' device, allocates its
result and workspace from torch's allocator (so it can be captured into a
graph) and reads or changes nothing else; what it changes counts as changed in
place for autograd. There is no CPU path; with
``KILN_HIP_INTERPRET=1`` (tests) the library's CPU meaning runs instead.
"""

from __future__ import annotations

import array
import ctypes
import math

import torch
from torch.autograd import forward_ad

from kiln.hip import lib as kl
from kiln.hip.interpret import interpreting

# asked at every call
_is_tracing, _dispatch_modes = torch._C._is_tracing, torch._C._len_torch_dispatch_stack
_increment_version = torch._C._increment_version

TYPES = {torch.float32: kl.TYPE_F32, torch.bfloat16: kl.TYPE_BF16, torch.float16: kl.TYPE_F16}


# -- checks --------------------------------------------------------------------------------


def _tensor(t, name, rank, dtypes):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    if t.dim() != rank:
        raise ValueError(f"{name} must have {rank} dimensions, got shape {tuple(t.shape)}")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} must be {' or '.join(str(d) for d in dtypes)}, got {t.dtype}")


def _shape(t, name, shape):
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")


def _int32(t, name, rank, shape):
    _tensor(t, name, rank, (torch.int32,))
    _shape(t, name, shape)


def _no_grad(*tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise NotImplementedError("the paged cache's operators have no backward pass: call them under torch.no_grad()")


def _no_tangent(*tensors):
    """Where a level of forward mode is open (no_grad does not close it)."""
    if any(isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError("the paged cache's operators have no forward-mode derivative: pass the primal tensors "
                                  "(torch.autograd.forward_ad.unpack_dual)")


def _one_device(first, *others):
    if first.device.type != "cuda" and not interpreting():
        raise NotImplementedError(f"the paged cache's operators run on the GPU only, got tensors on {first.device}")
    for t in others:
        if t is not None and t.device != first.device:
            raise ValueError(f"all tensors must be on one device, got {first.device} and {t.device}")


def check_pages(k_pages, v_pages, rank=4):
    """The pages of one layer (rank 4) or of a stack of layers (rank 5)."""
    _tensor(k_pages, "k_pages", rank, tuple(TYPES))
    _tensor(v_pages, "v_pages", rank, (k_pages.dtype,))
    _shape(v_pages, "v_pages", k_pages.shape)


def _rows_in_place(t, name):
    """Pages are read where they are: rows along the last dimension, each at a multiple of 16 bytes."""
    size = t.element_size()
    if t.stride(-1) != 1 or t.data_ptr() % 16 or any(s * size % 16 for s, n in zip(t.stride()[:-1], t.shape) if n > 1):
        raise ValueError(f"{name}: rows must be contiguous and start at multiples of 16 bytes")


def _rows(t):
    """A small operand whose rows start at multiples of 16 bytes: itself, or a copy."""
    size = t.element_size()
    if t.stride(-1) != 1 or t.data_ptr() % 16 or any(s * size % 16 for s in t.stride()[:-1]):
        return t.clone(memory_format=torch.contiguous_format)   # (a new tensor is aligned, a contiguous view may not be)
    return t


def _rows_strided(t):
    """As _rows, by the strides alone."""
    size = t.element_size()
    return _rows(t) if t.stride(-1) != 1 or any(s * size % 16 for s in t.stride()[:-1]) else t


def _head_dim(dim):
    if dim % 8 or not 0 < dim <= 256:
        raise NotImplementedError(f"head dimension {dim}: multiples of 8 up to 256 have kernels")


def check_attention(q, k, v, k_pages, v_pages, table, lengths, parents, selected):
    """(sizes of the call) after checking types, shapes and their agreement."""
    check_pages(k_pages, v_pages)
    pages, kv_heads, page_size, dim = k_pages.shape
    _tensor(q, "q", 4, (torch.float32,) if k_pages.dtype == torch.float32 else (torch.float32, k_pages.dtype))
    batch, draft, heads, _ = q.shape
    _shape(q, "q", (batch, draft, heads, dim))
    _head_dim(dim)
    for t, name in ((k, "k"), (v, "v")):
        _tensor(t, name, 4, (q.dtype,))
        _shape(t, name, (batch, draft, kv_heads, dim))
    if kv_heads == 0 or heads % kv_heads or heads == 0:
        raise ValueError(f"{heads} query heads do not divide over {kv_heads} heads of the cache")
    if not isinstance(table, torch.Tensor) or table.dim() != 2:
        raise ValueError("table must be a tensor [sequences, columns]")
    _int32(table, "table", 2, (batch, table.shape[1]))
    _int32(lengths, "lengths", 1, (batch,))
    if parents is not None:
        _int32(parents, "parents", 2, (batch, draft))
    if selected is not None:
        if not isinstance(selected, torch.Tensor) or selected.dim() != 4:
            raise ValueError("selected must be a tensor [sequences, tokens, kv heads, pages]")
        _int32(selected, "selected", 4, (batch, draft, kv_heads, selected.shape[3]))
        if selected.shape[3] == 0:
            raise ValueError("selected names no pages")
    return batch, draft, heads, kv_heads, dim, page_size, pages


def check_select(q, k_means, table, lengths, page_size, pages):
    _tensor(q, "q", 4, tuple(TYPES))
    _tensor(k_means, "k_means", 3, (torch.float32,))
    batch, draft, heads, dim = q.shape
    total, kv_heads, _ = k_means.shape
    _shape(k_means, "k_means", (total, kv_heads, dim))
    _head_dim(dim)
    if kv_heads == 0 or heads % kv_heads or heads == 0:
        raise ValueError(f"{heads} query heads do not divide over {kv_heads} heads of the cache")
    if not isinstance(table, torch.Tensor) or table.dim() != 2:
        raise ValueError("table must be a tensor [sequences, columns]")
    _int32(table, "table", 2, (batch, table.shape[1]))
    _int32(lengths, "lengths", 1, (batch,))
    if pages < 1:
        raise ValueError(f"pages must be at least 1, got {pages}")
    return batch, draft, heads, kv_heads, dim, total


def default_scale(scale, dim):
    return 1.0 / math.sqrt(dim) if scale is None else float(scale)


# -- running -------------------------------------------------------------------------------------


def _columns(t):
    """int32 operands are read with their last dimension contiguous."""
    return t if t.stride(-1) == 1 or t.numel() == 0 else t.contiguous()


def _stream(device):
    return torch._C._cuda_getCurrentRawStream(device.index)


def _on_device(device, entry, *args):
    """entry(*args, stream) with `device` current (a launch goes to the current device)."""
    if device.index == torch._C._cuda_getDevice():
        return entry(*args, _stream(device))
    with torch.cuda.device(device):
        return entry(*args, _stream(device))


def _ready(device):
    from kiln.hip.runtime import init_device, _ready_devices

    if device.type == "cuda" and device.index not in _ready_devices:
        # kh_init makes the device current and asks for its facts
        with torch.cuda.device(device):
            init_device(device)


def _form(*tensors):
    """What the checks and an operator's sizes and strides depend on, of each tensor."""
    return tuple([None if t is None else (t.shape, t.stride(), t.dtype, t.get_device()) for t in tensors])


# (operator, form of a call) -> its descriptor without addresses, and what
# belongs to it: the checks and the descriptor are worked out once per form.
# Forms are shapes, strides and types alone; a program has few, and the oldest
# go first.
_forms = {}
MOST_FORMS = 4096


def _keep(key, found):
    while len(_forms) >= MOST_FORMS:
        _forms.pop(next(iter(_forms)), None)
    _forms[key] = found
    return found


def _remember(key, op):
    size = ctypes.c_size_t()
    kl.check(kl.load().kh_paged_workspace_bytes(ctypes.byref(op), ctypes.byref(size)), "paged")
    return _keep(key, (bytes(op), size.value))


def _launch(op: kl.Paged, size: int, device, what: str):
    lib = kl.load()
    if device.type != "cuda":
        rc = lib.kh_paged_host(ctypes.byref(op))
    elif device.index == torch._C._cuda_getDevice():
        if size:
            workspace = torch.empty(size, dtype=torch.uint8, device=device)
            rc = lib.kh_paged_run(ctypes.byref(op), workspace.data_ptr(), size, _stream(device))
        else:
            rc = lib.kh_paged_run(ctypes.byref(op), None, 0, _stream(device))
    else:   # (a launch goes to the current device)
        with torch.cuda.device(device):
            return _launch(op, size, device, what)
    if rc:
        kl.check(rc, what)


def _attention_form(q, k, v, k_pages, v_pages, table, lengths, parents, selected, scale):
    """(descriptor without addresses) of a call, checked; operands' rows are in place."""
    batch, draft, heads, kv_heads, dim, page_size, pages = check_attention(
        q, k, v, k_pages, v_pages, table, lengths, parents, selected)
    _one_device(q, k, v, k_pages, v_pages, table, lengths, parents, selected)
    _rows_in_place(k_pages, "k_pages")
    _rows_in_place(v_pages, "v_pages")
    if pages == 0:
        raise ValueError("the cache has no pages")
    _ready(q.device)
    h, d = heads * dim, dim
    return kl.Paged(kl.PAGED_ATTENTION, batch, draft, heads, kv_heads, dim, page_size, pages, table.shape[1],
                    0 if selected is None else selected.shape[3], TYPES[k_pages.dtype], TYPES[q.dtype], 0, scale,
                    None, None, None, None, None, None, None, None, None, None, None,
                    *q.stride()[:3], *k.stride()[:3], *v.stride()[:3], draft * h, h, d,
                    *k_pages.stride()[:3], *v_pages.stride()[:3], 0, 0, table.stride(0),
                    0 if parents is None else parents.stride(0),
                    *((0, 0, 0) if selected is None else selected.stride()[:3]))


def run_attention(q, k, v, k_pages, v_pages, table, lengths, parents, selected, scale, what):
    try:
        key = ("attention", q.shape, q.dtype, q.stride(), q.get_device(), k.shape, k.dtype, k.stride(), k.get_device(),
               v.shape, v.dtype, v.stride(), v.get_device(), k_pages.shape, k_pages.dtype, k_pages.stride(),
               k_pages.get_device(), v_pages.shape, v_pages.dtype, v_pages.stride(), v_pages.get_device(),
               table.shape, table.dtype, table.stride(), table.get_device(), lengths.shape, lengths.dtype,
               lengths.stride(), lengths.get_device(),
               None if parents is None else (parents.shape, parents.dtype, parents.stride(), parents.get_device()),
               None if selected is None else (selected.shape, selected.dtype, selected.stride(), selected.get_device()),
               scale)
    except AttributeError:
        check_attention(q, k, v, k_pages, v_pages, table, lengths, parents, selected)   # names what is no tensor
        raise
    found = _forms.get(key)
    if found is None:
        check_attention(q, k, v, k_pages, v_pages, table, lengths, parents, selected)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or k_pages.requires_grad
                                    or v_pages.requires_grad):
        _no_grad(q, k, v, k_pages, v_pages)
    if found is None:
        straight = [_rows_strided(t) for t in (q, k, v)] + [_columns(t) for t in (table, lengths)]
        if any(a is not b for a, b in zip(straight, (q, k, v, table, lengths))):
            q, k, v, table, lengths = straight
            return run_attention(q, k, v, k_pages, v_pages, table, lengths, parents, selected, scale, what)
        if (parents is not None and _columns(parents) is not parents) or (selected is not None and _columns(selected) is not selected):
            parents, selected = (None if t is None else _columns(t) for t in (parents, selected))
            return run_attention(q, k, v, k_pages, v_pages, table, lengths, parents, selected, scale, what)
        op = _attention_form(q, k, v, k_pages, v_pages, table, lengths, parents, selected, scale)
        if q.numel() == 0:
            return torch.empty(q.shape, dtype=q.dtype, device=q.device)
        found = _remember(key, op)
    elif q.device.type != "cuda" and not interpreting():
        _one_device(q)
    op = kl.Paged.from_buffer_copy(found[0])
    out = q.new_empty(q.shape)
    at = (q.data_ptr(), k.data_ptr(), v.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr())
    if (at[0] | at[1] | at[2] | at[3] | at[4]) & 15:
        _rows_in_place(k_pages, "k_pages")
        _rows_in_place(v_pages, "v_pages")
        return run_attention(_rows(q), _rows(k), _rows(v), k_pages, v_pages, table, lengths, parents, selected, scale, what)
    op.q, op.k, op.v, op.k_pages, op.v_pages = at
    op.table, op.lengths, op.out = table.data_ptr(), lengths.data_ptr(), out.data_ptr()
    if parents is not None:
        op.parents = parents.data_ptr()
    if selected is not None:
        op.selected = selected.data_ptr()
    _launch(op, found[1], q.device, what)
    return out


def run_select(q, k_means, table, lengths, page_size, pages):
    try:
        key = ("select", _form(q, k_means, table, lengths), page_size, pages)
    except AttributeError:
        check_select(q, k_means, table, lengths, page_size, pages)
        raise
    found = _forms.get(key)
    if found is None:
        batch, draft, heads, kv_heads, dim, total = check_select(q, k_means, table, lengths, page_size, pages)
    if torch.is_grad_enabled() and (q.requires_grad or k_means.requires_grad):
        _no_grad(q, k_means)
    if found is None:
        straight = _rows_strided(q), _columns(table), _columns(lengths)
        if any(a is not b for a, b in zip(straight, (q, table, lengths))):
            return run_select(straight[0], k_means, straight[1], straight[2], page_size, pages)
        _one_device(q, k_means, table, lengths)
        _rows_in_place(k_means, "k_means")
        if batch * draft == 0:
            return torch.empty((batch, draft, kv_heads, pages), dtype=torch.int32, device=q.device)
        if total == 0:
            raise ValueError("the cache has no pages")
        _ready(q.device)
        op = kl.Paged(kl.PAGED_SELECT, batch, draft, heads, kv_heads, dim, page_size, total, table.shape[1], pages,
                      kl.TYPE_F32, TYPES[q.dtype], 0, 1.0)
        op.q_s, op.q_n, op.q_h = q.stride()[:3]
        op.m_p, op.m_h = k_means.stride()[:2]
        op.table_s = table.stride(0)
        op.sel_s, op.sel_n, op.sel_h = draft * kv_heads * pages, kv_heads * pages, pages
        found = _remember(key, op)
    elif q.device.type != "cuda" and not interpreting():
        _one_device(q)
    op = kl.Paged.from_buffer_copy(found[0])
    out = table.new_empty((op.batch, op.draft, op.kv_heads, pages))
    op.q, op.k_means = q.data_ptr(), k_means.data_ptr()
    if (op.q | op.k_means) & 15:
        _rows_in_place(k_means, "k_means")
        return run_select(_rows(q), k_means, table, lengths, page_size, pages)
    op.table, op.lengths, op.selected = table.data_ptr(), lengths.data_ptr(), out.data_ptr()
    _launch(op, found[1], q.device, "select_pages")
    return out


# -- as operators of torch, for graphs -----------------------------------------------------------


@torch.library.custom_op("kiln::paged_attention", mutates_args=())
def _paged_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                     table: torch.Tensor, lengths: torch.Tensor, parents: torch.Tensor | None,
                     selected: torch.Tensor | None, scale: float) -> torch.Tensor:
    with torch.no_grad():
        return run_attention(q, k, v, k_pages, v_pages, table, lengths, parents, selected, scale, "paged_attention")


@_paged_attention.register_fake
def _(q, k, v, k_pages, v_pages, table, lengths, parents, selected, scale):
    check_attention(q, k, v, k_pages, v_pages, table, lengths, parents, selected)
    return q.new_empty(tuple(q.shape))


@torch.library.custom_op("kiln::select_pages", mutates_args=())
def _select_pages(q: torch.Tensor, k_means: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, page_size: int,
                  pages: int) -> torch.Tensor:
    with torch.no_grad():
        return run_select(q, k_means, table, lengths, page_size, pages)


@_select_pages.register_fake
def _(q, k_means, table, lengths, page_size, pages):
    check_select(q, k_means, table, lengths, page_size, pages)
    return q.new_empty((q.shape[0], q.shape[1], k_means.shape[1], pages), dtype=torch.int32)


@torch.library.custom_op("kiln::cache_append", mutates_args=("k_pages", "v_pages", "k_means"))
def _cache_append(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor,
                  lengths: torch.Tensor, rows: torch.Tensor | None, k_means: torch.Tensor | None) -> None:
    with torch.no_grad():
        run_append(k, v, k_pages, v_pages, table, lengths, rows, k_means)


@_cache_append.register_fake
def _(k, v, k_pages, v_pages, table, lengths, rows, k_means):
    pass


@torch.library.custom_op("kiln::copy_pages", mutates_args=("pools",))
def _copy_pages(pools: list[torch.Tensor], source: list[int], target: list[int]) -> None:
    with torch.no_grad():
        run_copy(pools, source, target)


@_copy_pages.register_fake
def _(pools, source, target):
    pass


def _watched(*tensors) -> bool:
    """Whether a compiler, a tracer or a dispatch mode is to see the call: not
    what it allocates, but the operator. ``tensors``: those that a derivative
    could be asked of."""
    if torch.compiler.is_compiling():
        return True
    if forward_ad._current_level >= 0:
        _no_tangent(*tensors)
    if not (_dispatch_modes() or _is_tracing()):
        return False
    _no_grad(*tensors)
    return True


# -- the public functions ------------------------------------------------------------------------------


def tree_attention(q, k, v, k_pages, v_pages, table, lengths, parents=None, *, scale=None):
    """Attention of drafted tokens over a paged cache and over each other.

    ``q`` ``[sequences, tokens, heads, dim]``, ``k`` and ``v`` ``[sequences,
    tokens, kv_heads, dim]``: the drafted tokens', in fp32 or the cache's
    type; they are not in the cache yet. ``parents`` ``[sequences, tokens]``
    (int32): the earlier drafted token that token i follows, -1 where it
    follows the cached ones; any other value marks the token, and those that
    follow it, as unused (rows of zeros). Without ``parents`` each token
    follows the one before it. Query heads ``h`` share head ``h // (heads /
    kv_heads)`` of the cache. Returns ``softmax(scale q . keys) values``,
    shaped and typed as ``q``; ``scale`` is 1 / sqrt(dim) by default.

    Drafted keys and values are rounded to the cache's type first, so a token
    is attended to as it will be once it is appended. fp32 activations keep
    fp32's accuracy over bf16 and fp16 caches too; 16-bit ones are exact in
    the scores, their softmax weights keep 16 bits (bf16) or 22 (fp16), sums
    are fp32, and the result is rounded once. Up to 256 tokens and 4096
    sequences, dim a multiple of 8 up to 256, page_size a power of two from
    16 to 1024. A table entry outside the pool holds no tokens.
    """
    scale = default_scale(scale, k_pages.shape[-1])
    if _watched(q, k, v, k_pages, v_pages):
        return torch.ops.kiln.paged_attention(q, k, v, k_pages, v_pages, table, lengths, parents, None, scale)
    return run_attention(q, k, v, k_pages, v_pages, table, lengths, parents, None, scale, "tree_attention")


def selected_attention(q, k, v, k_pages, v_pages, table, lengths, selected, parents=None, *, scale=None):
    """``tree_attention`` in which token i of sequence s attends, of the
    cached tokens, to those of the pages ``selected[s, i, kv_head]`` alone
    (int32 ``[sequences, tokens, kv_heads, pages]``: columns of ``table``, as
    ``select_pages`` gives them). An entry counts only where it is larger
    than the one before it, so lists ascend and end with -1."""
    if selected is None:
        raise TypeError("selected must be a tensor (tree_attention reads every page)")
    scale = default_scale(scale, k_pages.shape[-1])
    if _watched(q, k, v, k_pages, v_pages):
        return torch.ops.kiln.paged_attention(q, k, v, k_pages, v_pages, table, lengths, parents, selected, scale)
    return run_attention(q, k, v, k_pages, v_pages, table, lengths, parents, selected, scale, "selected_attention")


def select_pages(q, k_means, table, lengths, *, page_size, pages):
    """The ``pages`` pages of each sequence that a cheap score picks for each
    drafted token and head of the cache: the largest (sum of the group's
    queries) . ``k_means[page]`` (fp32 ``[pages of the pool, kv_heads, dim]``,
    the mean key of each page), summed in 64 bits; the page of the last
    cached token is always among them. Ties go to the lower column. Returns
    int32 ``[sequences, tokens, kv_heads, pages]``: columns of ``table``,
    ascending, then -1."""
    if _watched(q, k_means):
        return torch.ops.kiln.select_pages(q, k_means, table, lengths, int(page_size), int(pages))
    return run_select(q, k_means, table, lengths, int(page_size), int(pages))


def _recorded(what):
    """Refuse what does not keep a call that changes its arguments."""
    if torch.compiler.is_compiling():
        raise NotImplementedError(f"{what} changes its arguments, which a compiled graph does not: call it between "
                                  f"the calls of the compiled step")
    if _is_tracing():   # (torch.jit.trace drops an operator without results)
        raise NotImplementedError(f"{what} changes its arguments, which torch.jit.trace does not record")


def cache_append(k, v, k_pages, v_pages, table, lengths, *, rows=None, k_means=None):
    """Write new tokens behind the cached ones, in place: token
    ``rows[s, a]`` of ``k`` and ``v`` ``[sequences, tokens, kv_heads, dim]``
    becomes token ``lengths[s] + a`` of sequence s, rounded to the cache's
    type. ``rows`` (int32 ``[sequences, accepted]``): the accepted path of a
    drafted tree; a row ends at its first entry outside [0, tokens). Without
    ``rows`` all tokens, in order. With ``k_means`` the mean key of every page
    written to is brought up to date. ``lengths`` is not changed.

    With a leading dimension of layers on ``k``, ``v`` (5 dimensions), the
    pages (5) and ``k_means`` (4), all layers are written at once; ``table``,
    ``lengths`` and ``rows`` hold for each. Tokens whose page the table does
    not name are dropped. No page may belong to two of the sequences."""
    if _watched(k, v, k_pages, v_pages, k_means):
        _recorded("cache_append")
        return torch.ops.kiln.cache_append(k, v, k_pages, v_pages, table, lengths, rows, k_means)
    run_append(k, v, k_pages, v_pages, table, lengths, rows, k_means)


def run_append(k, v, k_pages, v_pages, table, lengths, rows, k_means):
    try:
        key = ("append", _form(k, v, k_pages, v_pages, table, lengths, rows, k_means))
    except AttributeError:
        _append_form(k, v, k_pages, v_pages, table, lengths, rows, k_means)
        raise
    template = _forms.get(key)
    if template is None:
        op = _append_form(k, v, k_pages, v_pages, table, lengths, rows, k_means)
        if isinstance(op, tuple):     # operands moved to where rows are in place
            return run_append(*op, k_means)
        if op is None:
            return
        template = _keep(key, bytes(op))
    elif k.device.type != "cuda" and not interpreting():
        _one_device(k)
    if torch.is_grad_enabled() and (k.requires_grad or v.requires_grad or k_pages.requires_grad or v_pages.requires_grad
                                    or (k_means is not None and k_means.requires_grad)):
        _no_grad(k, v, k_pages, v_pages, k_means)
    op = kl.CacheAppend.from_buffer_copy(template)
    op.k, op.v, op.k_pages, op.v_pages = at = (k.data_ptr(), v.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr())
    if (at[0] | at[1] | at[2] | at[3]) & 15:
        _rows_in_place(k_pages, "k_pages")
        _rows_in_place(v_pages, "v_pages")
        return run_append(_rows(k), _rows(v), k_pages, v_pages, table, lengths, rows, k_means)
    op.table, op.lengths = table.data_ptr(), lengths.data_ptr()
    if rows is not None:
        op.rows = rows.data_ptr()
    if k_means is not None:
        op.k_means = k_means.data_ptr()
    lib, device = kl.load(), k.device
    if device.type != "cuda":
        rc = lib.kh_cache_append_host(ctypes.byref(op))
    else:
        rc = _on_device(device, lib.kh_cache_append, ctypes.byref(op))
    if rc:
        kl.check(rc, "cache_append")
    _increment_version((k_pages, v_pages) if k_means is None else (k_pages, v_pages, k_means))


def _append_form(k, v, k_pages, v_pages, table, lengths, rows, k_means):
    """The descriptor of a call without addresses, checked; None for a call
    that writes nothing; a tuple of operands to call with where some had to be
    laid out anew."""
    rank = k_pages.dim() if isinstance(k_pages, torch.Tensor) and k_pages.dim() == 5 else 4
    check_pages(k_pages, v_pages, rank)
    given = (k, v, k_pages, v_pages, table, lengths, rows)
    if rank == 4:
        k, v = (t.unsqueeze(0) if isinstance(t, torch.Tensor) else t for t in (k, v))
        k_pages, v_pages = k_pages.unsqueeze(0), v_pages.unsqueeze(0)
        k_means = k_means.unsqueeze(0) if isinstance(k_means, torch.Tensor) else k_means
    layers, pages, kv_heads, page_size, dim = k_pages.shape
    _head_dim(dim)
    _tensor(k, "k", 5, tuple(TYPES))
    batch, draft = k.shape[1], k.shape[2]
    _shape(k, "k", (layers, batch, draft, kv_heads, dim))
    _tensor(v, "v", 5, (k.dtype,))
    _shape(v, "v", k.shape)
    if not isinstance(table, torch.Tensor) or table.dim() != 2:
        raise ValueError("table must be a tensor [sequences, columns]")
    _int32(table, "table", 2, (batch, table.shape[1]))
    _int32(lengths, "lengths", 1, (batch,))
    if rows is not None:
        if not isinstance(rows, torch.Tensor) or rows.dim() != 2:
            raise ValueError("rows must be a tensor [sequences, accepted]")
        _int32(rows, "rows", 2, (batch, rows.shape[1]))
    if k_means is not None:
        _tensor(k_means, "k_means", 4, (torch.float32,))
        _shape(k_means, "k_means", (layers, pages, kv_heads, dim))
        if k_means.stride(-1) != 1:
            raise ValueError("k_means: rows must be contiguous")
    _no_grad(k, v, k_pages, v_pages, k_means)
    _one_device(k, v, k_pages, v_pages, table, lengths, rows, k_means)
    _rows_in_place(k_pages, "k_pages")
    _rows_in_place(v_pages, "v_pages")
    straight = (_rows_strided(given[0]), _rows_strided(given[1]), given[2], given[3], _columns(table), _columns(lengths),
                None if rows is None else _columns(rows))
    if any(a is not b for a, b in zip(straight, given)):
        return straight
    accept = draft if rows is None else rows.shape[1]
    if layers * batch * accept * draft == 0:
        return None
    _ready(k.device)
    return kl.CacheAppend(layers, batch, draft, accept, kv_heads, dim, page_size, pages, table.shape[1],
                          TYPES[k_pages.dtype], TYPES[k.dtype], None, None, None, None, None, None, None, None,
                          *k.stride()[:4], *v.stride()[:4], *k_pages.stride()[:4], *v_pages.stride()[:4],
                          *(k_means.stride()[:3] if k_means is not None else (0, 0, 0)), table.stride(0),
                          rows.stride(0) if rows is not None else 0)


def _page_list(x, name):
    try:
        numbers = array.array("i", x)
    except TypeError:
        raise TypeError(f"{name} must be a sequence of page numbers (ints)") from None
    except OverflowError:
        raise ValueError(f"{name} holds a number that no page has") from None
    return (ctypes.c_int32 * len(numbers)).from_buffer(numbers)


def _pool_forms(pools):
    """(the pools' descriptors without addresses, their number of pages), checked."""
    descs = (kl.Pool * max(1, len(pools)))()
    pages = None
    for i, t in enumerate(pools):
        if not isinstance(t, torch.Tensor) or t.dim() < 2:
            raise TypeError("a pool is a tensor of pages")
        shape, strides, size = t.shape, t.stride(), t.element_size()
        first = 1 if len(shape) == 5 else 0     # the dimension of pages
        inner = 1
        for n, step in zip(reversed(shape[first:]), reversed(strides[first:])):
            if n > 1 and step != inner:
                raise ValueError("a pool's pages must be contiguous within a layer")
            inner *= n
        if pages is not None and pages != shape[first]:
            raise ValueError(f"pools of {pages} and of {shape[first]} pages")
        pages = shape[first]
        descs[i] = kl.Pool(None, shape[0] if first else 1, strides[0] * size if first else 0,
                           inner // pages * size if pages else 0)
    return bytes(descs), pages


def copy_pages(pools, source, target):
    """Copy pages within each of ``pools``, in place: page ``source[i]`` to
    page ``target[i]``. A pool is a tensor ``[pages, ...]`` or, with 5
    dimensions (4 for fp32 means of 5-dimensional pools: pass
    ``means.unsqueeze(-2)``), ``[layers, pages, ...]``, contiguous within a
    layer. ``source`` and ``target`` are sequences of ints; targets are
    distinct and none is a source, so no order of the copies matters."""
    pools = list(pools)
    if _watched(*pools):
        _recorded("copy_pages")
        return torch.ops.kiln.copy_pages(pools, [int(x) for x in source], [int(x) for x in target])
    run_copy(pools, source, target)


def run_copy(pools, source, target):
    if len(source) != len(target):
        raise ValueError(f"{len(source)} source pages, but {len(target)} target pages")
    try:
        key = ("copy", _form(*pools))
    except AttributeError:
        raise TypeError("a pool is a tensor of pages") from None
    found = _forms.get(key)
    if found is None:
        found = _pool_forms(pools)
        if not pools or len(source) == 0:
            return
        _one_device(*pools)
        _ready(pools[0].device)
        _keep(key, found)
    elif pools[0].device.type != "cuda" and not interpreting():
        _one_device(*pools)
    if len(source) == 0:
        return
    if torch.is_grad_enabled():
        _no_grad(*pools)
    template, pages = found
    descs = (kl.Pool * len(pools)).from_buffer_copy(template)
    for desc, t in zip(descs, pools):
        desc.base = t.data_ptr()
    src, dst = _page_list(source, "source"), _page_list(target, "target")
    lib, device = kl.load(), pools[0].device
    if device.type != "cuda":
        rc = lib.kh_cache_copy_host(descs, len(pools), pages, src, dst, len(src))
    else:
        rc = _on_device(device, lib.kh_cache_copy, descs, len(pools), pages, src, dst, len(src))
    if rc:
        kl.check(rc, "copy_pages")
    _increment_version(pools)
