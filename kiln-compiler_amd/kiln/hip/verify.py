"""Verification of drafted tokens, as a function on torch tensors.

    verify_tokens       which of the drafted tokens the target model keeps, and
                        the token that comes after them

It stands between ``tree_attention`` of a drafted tree (kiln/hip/paged.py) and
``cache_append`` of the tokens that are kept, whose ``rows`` it returns:

    rows, counts, after = kiln.verify_tokens(tokens, target, uniforms, parents, draft=draft)
    kiln.cache_append(k, v, k_pages, v_pages, table, lengths, rows=rows)

``after`` is the next step's token 0. Streams, workspaces, tracers and
``KILN_HIP_INTERPRET`` as for the operators over the cache.
"""

from __future__ import annotations

import ctypes

import torch

from kiln.hip import lib as kl
from kiln.hip import paged

TOKEN_TYPES = (torch.int32, torch.int64)
UNIFORM_TYPES = (torch.float32, torch.float64)


def check_verify(tokens, target, uniforms, parents, draft):
    paged._tensor(tokens, "tokens", 2, TOKEN_TYPES)
    batch, n = tokens.shape
    paged._tensor(target, "target", 3, tuple(paged.TYPES))
    vocab = target.shape[2]
    paged._shape(target, "target", (batch, n, vocab))
    paged._tensor(uniforms, "uniforms", 2, UNIFORM_TYPES)
    paged._shape(uniforms, "uniforms", (batch, n))
    if parents is not None:
        paged._int32(parents, "parents", 2, (batch, n))
    if draft is not None:
        paged._tensor(draft, "draft", 3, (target.dtype,))
        paged._shape(draft, "draft", (batch, n, vocab))
    if n == 0 or vocab == 0:
        raise ValueError(f"{n} drafted tokens of a vocabulary of {vocab}: token 0 is the root")
    for count, most, what in ((batch, 65535, "sequences"), (n, 256, "drafted tokens"), (vocab, 2 ** 24, "tokens of a vocabulary")):
        if count > most:   # (here, before any operand is copied)
            raise NotImplementedError(f"{count} {what}: at most {most} have kernels")
    return batch, n, vocab


def _rows_together(t):
    """Rows of probabilities are read where they are, if their elements lie together."""
    return t if t is None or t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def run_verify(tokens, target, uniforms, parents, draft):
    try:
        key = ("verify", paged._form(tokens, target, uniforms, parents, draft))
    except AttributeError:
        check_verify(tokens, target, uniforms, parents, draft)
        raise
    found = paged._forms.get(key)
    if found is None:
        batch, n, vocab = check_verify(tokens, target, uniforms, parents, draft)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (target, uniforms, draft)):
        raise NotImplementedError("verify_tokens has no backward pass: call it under torch.no_grad()")
    if found is None:
        straight = [paged._columns(t) if t is not None else None for t in (tokens, uniforms, parents)]
        straight += [_rows_together(target), _rows_together(draft)]
        if any(a is not b for a, b in zip(straight, (tokens, uniforms, parents, target, draft))):
            tokens, uniforms, parents, target, draft = straight
            return run_verify(tokens, target, uniforms, parents, draft)
        paged._one_device(tokens, target, uniforms, parents, draft)
        if batch:
            paged._ready(tokens.device)
        op = kl.Verify(batch, n, vocab, paged.TYPES[target.dtype], tokens.dtype == torch.int64, uniforms.dtype == torch.float64)
        op.tokens_s, op.target_s, op.target_n = tokens.stride(0), target.stride(0), target.stride(1)
        op.uniforms_s = uniforms.stride(0)
        if draft is not None:
            op.drafted_s, op.drafted_n = draft.stride()[:2]
        if parents is not None:
            op.parents_s = parents.stride(0)
        size = ctypes.c_size_t()
        kl.check(kl.load().kh_verify_workspace_bytes(ctypes.byref(op), ctypes.byref(size)), "verify_tokens")
        found = paged._keep(key, (bytes(op), size.value))
    elif tokens.device.type != "cuda" and not paged.interpreting():
        paged._one_device(tokens)
    op = kl.Verify.from_buffer_copy(found[0])
    device = tokens.device
    batch, n = op.batch, op.draft
    # (memory of their own: one that is kept or saved keeps no other, nor the workspace)
    rows = tokens.new_empty((batch, n), dtype=torch.int32)
    counts, after = rows.new_empty(batch), rows.new_empty(batch)
    if batch == 0:
        return rows, counts, after
    op.tokens, op.target, op.uniforms = tokens.data_ptr(), target.data_ptr(), uniforms.data_ptr()
    if draft is not None:
        op.drafted = draft.data_ptr()
    if parents is not None:
        op.parents = parents.data_ptr()
    op.rows, op.counts, op.next = rows.data_ptr(), counts.data_ptr(), after.data_ptr()
    lib = kl.load()
    if device.type != "cuda":
        rc = lib.kh_verify_host(ctypes.byref(op))
    else:
        workspace = torch.empty(found[1], dtype=torch.uint8, device=device) if found[1] else None
        rc = paged._on_device(device, lib.kh_verify_run, ctypes.byref(op), workspace.data_ptr() if found[1] else None, found[1])
    if rc:
        kl.check(rc, "verify_tokens")
    return rows, counts, after


@torch.library.custom_op("kiln::verify_tokens", mutates_args=())
def _verify_tokens(tokens: torch.Tensor, target: torch.Tensor, uniforms: torch.Tensor, parents: torch.Tensor | None,
                   draft: torch.Tensor | None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    with torch.no_grad():
        return run_verify(tokens, target, uniforms, parents, draft)


@_verify_tokens.register_fake
def _(tokens, target, uniforms, parents, draft):
    batch, n, _ = check_verify(tokens, target, uniforms, parents, draft)
    return tuple(tokens.new_empty(shape, dtype=torch.int32) for shape in ((batch, n), (batch,), (batch,)))


def verify_tokens(tokens, target, uniforms, parents=None, *, draft=None):
    """Which drafted tokens are kept, and the token after them: so that what
    comes out is distributed as if the target model had made each token.

    ``tokens`` ``[sequences, tokens]`` (int32 or int64): a drafted tree as
    ``tree_attention`` takes it, ``parents`` (int32) likewise. Token 0 is the
    root, the sequence's last token, which the cache does not have yet: its
    parent is -1, every other token follows an earlier one (a second token
    without a parent is never kept). Any other parent of token 0 marks a
    sequence without a draft: nothing is kept. ``target`` ``[sequences, tokens,
    vocabulary]`` (fp32, bf16 or fp16): the target model's probabilities after
    each token. ``uniforms`` ``[sequences, tokens]`` (fp32 or fp64): random
    numbers in [0, 1).

    With ``draft``, shaped and typed as ``target``, the probabilities that the
    children of each token were drawn from, independently: child c of the
    current token is kept if ``uniforms[c]`` times the draft's probability of c
    is below the target's, and is the current token from then on; if not, the
    draft's probabilities are taken off the target's, and the next child is
    asked over what is left. When no child is left the token after is drawn
    from that, with ``uniforms[0]``: the first whose running sum passes that
    part of the whole. Without ``draft`` (tokens chosen in any way) a token is
    drawn from the target's row of the current one with its own uniform; a
    child that is this token is kept, else it is the token after.

    Returns int32 ``rows`` ``[sequences, tokens]`` (the kept tokens, root first,
    then -1: what ``cache_append`` takes), ``counts`` and the token after,
    ``[sequences]``. Sums are 64-bit. With ``draft`` the rows of both are taken
    to sum to 1, as the first comparison under a token weighs the two as they
    are: tokens come out as the target's as nearly as the rows do (16-bit rows of
    a large vocabulary only nearly). Without it, rows need not sum to 1.
    Probabilities that are not above 0 count as 0; a target row without any, or
    with an infinite one, gives -1 as the token after. (A NaN of the draft's does
    not count as 0: its token is refused, and a refusal leaves nothing of it.) A
    token outside the vocabulary is not kept. Up to 256 tokens, 65535 sequences
    and a vocabulary of 2^24."""
    if paged._watched(target, uniforms, draft):
        return torch.ops.kiln.verify_tokens(tokens, target, uniforms, parents, draft)
    return run_verify(tokens, target, uniforms, parents, draft)
