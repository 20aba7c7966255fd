"""Steps over a paged cache for the tests of its operators, and their definition in 64 bits."""

import math

import numpy as np
import torch


def i32(values, device="cpu"):
    return torch.tensor(np.asarray(values, dtype=np.int32), device=device)


class Step:
    """Requests of `lengths` keys, of which the last `tokens` are the step's; `shared` = (requests, keys) per group: consecutive
    requests whose first keys lie in the same pages (a page that the border cuts is copied). Pages in any order, -1 behind a request's last one;
    what no request owns holds NaN."""

    def __init__(self, lengths, tokens, heads, kv_heads, dim, page, dtype, seed, shared=(), query_std=1.5, key_std=1.0, width=None):
        gen = torch.Generator().manual_seed(seed)
        self.lengths, self.tokens, self.heads, self.kv_heads, self.dim, self.page, self.dtype = list(lengths), list(tokens), heads, kv_heads, dim, page, dtype
        seqs = len(self.lengths)
        self.prefix = [n for count, n in shared for _ in range(count)] or [0] * seqs
        self.group_start = [0, *np.cumsum([count for count, _ in shared]).tolist()] if shared else list(range(seqs + 1))
        first_of = {b: start for start, end in zip(self.group_start, self.group_start[1:]) for b in range(start, end)}
        counts = [-(-n // page) for n in self.lengths]
        whole = [min(p // page, c) for p, c in zip(self.prefix, counts)]
        total = sum(counts) + 3
        order = np.random.RandomState(seed).permutation(total).astype(np.int32)
        table = np.full((seqs, width or max(1, *counts)), -1, dtype=np.int32)
        at = 0
        for b in range(seqs):
            first = first_of[b]
            keep = 0 if b == first else min(whole[b], whole[first])
            table[b, :keep] = table[first, :keep]
            table[b, keep : counts[b]] = order[at : at + counts[b] - keep]
            at += counts[b] - keep
        self.table = torch.from_numpy(table)

        def normal(std, *shape):
            return (torch.randn(shape, generator=gen) * std).to(dtype)

        self.qkv = normal(query_std, sum(self.tokens), (heads + 2 * kv_heads) * dim)
        self.keys, self.values = normal(key_std, total, kv_heads, page, dim), normal(key_std, total, kv_heads, page, dim)
        owned = torch.zeros(total, page, dtype=torch.bool)
        for b, n in enumerate(self.lengths):
            j = torch.arange(n)
            owned[self.table[b].long()[j // page], j % page] = True
            first = first_of[b]
            cut = torch.arange(whole[b] * page, min(self.prefix[b], n))
            if b != first and len(cut):
                for pool in (self.keys, self.values):
                    pool[self.table[b].long()[cut // page], :, cut % page] = pool[self.table[first].long()[cut // page], :, cut % page]
        self.owned = owned
        for pool in (self.keys, self.values):
            pool.masked_fill_(~owned[:, None, :, None], math.nan)
        self.mass = torch.rand(total, kv_heads, page, generator=gen) * 0.05
        self.scale = dim ** -0.5
        self.q_start = i32([0, *np.cumsum(self.tokens)])
        self.kv_len, self.q_pos0 = i32(self.lengths), i32([n - t for n, t in zip(self.lengths, self.tokens)])
        self.prefix_len, self.groups = i32(self.prefix), i32(self.group_start)

    def rows(self, pool, b):
        """[kv_heads, keys, ...] of request b."""
        j = torch.arange(self.lengths[b])
        return pool[self.table[b].long()[j // self.page], :, j % self.page].transpose(0, 1)

    def weights(self, b):
        """Softmax weights in 64 bits: [heads, the step's tokens, keys]."""
        n, t, start = self.lengths[b], self.tokens[b], int(self.q_start[b])
        q = self.qkv[start : start + t, : self.heads * self.dim].double().view(t, self.heads, self.dim).transpose(0, 1)
        k = self.rows(self.keys, b).double().repeat_interleave(self.heads // self.kv_heads, 0)
        hidden = torch.arange(n)[None, :] > torch.arange(n - t, n)[:, None]
        return torch.softmax((q @ k.transpose(1, 2) * self.scale).masked_fill(hidden, -math.inf), -1)

    def attention(self):
        """[tokens, heads * dim] in 64 bits."""
        out = torch.zeros(sum(self.tokens), self.heads, self.dim, dtype=torch.float64)
        for b, t in enumerate(self.tokens):
            if t:
                v = self.rows(self.values, b).double().repeat_interleave(self.heads // self.kv_heads, 0)
                start = int(self.q_start[b])
                out[start : start + t] = (self.weights(b) @ v).transpose(0, 1)
        return out.flatten(1)

    def masses(self, keep_first=0, pads=()):
        """`mass` after the step, in 64 bits."""
        out = self.mass.double()
        for b, (n, t) in enumerate(zip(self.lengths, self.tokens)):
            if not t or b in pads:
                continue
            added = self.weights(b).sum(1).view(self.kv_heads, -1, n).sum(1)
            j = torch.arange(min(keep_first, n), n)
            p, o = self.table[b].long()[j // self.page], j % self.page
            out[p, :, o] = torch.where(j[:, None] >= n - t, 0.0, out[p, :, o]) + added[:, len(added[0]) - len(j) :].T
        return out

    def on(self, device="cuda"):
        """The tensors that an attention takes first, on the device."""
        return [t.to(device) for t in (self.qkv, self.keys, self.values)], [t.to(device) for t in (self.table, self.q_start, self.q_pos0, self.kv_len)]

    @property
    def sizes(self):
        return self.heads, self.kv_heads, self.dim, self.page

    @property
    def longest(self):
        """max_q_len, max_kv_len"""
        return max(self.tokens), max(self.lengths)


def output_tolerance(dtype, want):
    """Of an attention's output against 64 bits, as a share of the largest output.

    float32: scores of |q . k| * scale up to S carry a relative error of about dim * 2^-24 at worst, which the exponential turns into a relative
    error of S * dim * 2^-24 of each weight; the tests' scores stay below 16, so 2 * 16 * 128 * 2^-24 = 2.4e-4 bounds it and errors
    add up like their root: 2e-5 is 80 steps of 2^-22. bfloat16: the output's rounding (2^-9 of its value) and that of every weight (2^-9 each,
    2^-9 of the output at most together): 2^-8, and as much again for weights that are rounded against a running maximum."""
    return (2e-5 if dtype == torch.float32 else 2.0 ** -7) * max(1e-3, float(want.abs().max()))
