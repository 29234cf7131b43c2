"""The GPT-2 block (models/transformer.py) as a decoder: rows are drafted tokens
of several sequences whose earlier tokens are in a paged cache. It returns the
rows' result and their keys and values, which the caller appends to the cache
once it knows which tokens are accepted."""

import torch
import torch.nn as nn
import torch.nn.functional as F

import kiln


class CachedBlock(nn.Module):
    """`top`: attend to that many picked pages instead of the whole cache."""

    def __init__(self, block, tokens, top=None):
        super().__init__()
        self.block = block
        self.tokens = tokens
        self.top = top

    def attend(self, x, k_pages, v_pages, table, lengths, parents, k_means):
        b = self.block
        c = x.shape[-1]
        split = (len(x) // self.tokens, self.tokens, b.nh, c // b.nh)
        q, k, v = (y.view(split) for y in b.c_attn(b.ln1(x)).split(c, dim=1))
        if self.top is None:
            y = kiln.tree_attention(q, k, v, k_pages, v_pages, table, lengths, parents)
        else:
            picked = kiln.select_pages(q, k_means, table, lengths, page_size=k_pages.shape[2], pages=self.top)
            y = kiln.selected_attention(q, k, v, k_pages, v_pages, table, lengths, picked, parents)
        return x + b.c_proj(y.reshape(x.shape)), k, v

    def forward(self, x, k_pages, v_pages, table, lengths, parents=None, k_means=None):
        x, k, v = self.attend(x, k_pages, v_pages, table, lengths, parents, k_means)
        b = self.block
        return x + b.proj(F.gelu(b.fc(b.ln2(x)), approximate="tanh")), k, v


class CachedStack(nn.Module):
    """Every block of a Stack over the cache's layers; keys and values of all
    layers come back as [layers, sequences, tokens, heads, dim]."""

    def __init__(self, stack, tokens, top=None):
        super().__init__()
        self.blocks = nn.ModuleList(CachedBlock(b, tokens, top) for b in stack.blocks)
        self.ln_f = stack.ln_f

    def forward(self, x, k_pages, v_pages, table, lengths, parents=None, k_means=None):
        ks, vs = [], []
        for i, block in enumerate(self.blocks):
            x, k, v = block(x, k_pages[i], v_pages[i], table, lengths, parents, None if k_means is None else k_means[i])
            ks.append(k)
            vs.append(v)
        return self.ln_f(x), ks, vs
