"""A shared prefix, decoding that adds up attention weights, eviction by them, and decoding behind the prefix over what stayed: the
operators and the allocator as a server would use them, against the definitions in 64 bits."""

import math

import pytest
import torch

from cache_operators import i32, output_tolerance
from paged_attention_engine_b200.cache.allocator import BlockAllocator

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from paged_attention_engine_b200.kernels import ops as kernel_ops

    return kernel_ops


@pytest.mark.parametrize("dtype,heads,kv_heads,dim,page", [(torch.bfloat16, 12, 2, 128, 16), (torch.bfloat16, 8, 8, 64, 32), (torch.float32, 6, 3, 64, 16)])
def test_a_served_batch(ops, dtype, heads, kv_heads, dim, page):
    gen = torch.Generator().manual_seed(dim + heads)
    shared, steps, budget_behind, keep_last, share = 4 * page, 30, 24, 6, heads // kv_heads
    prompts = [5, 60, 23, 90, 41]
    seqs = len(prompts)
    pool = BlockAllocator(80, page)
    keys, values = (torch.zeros(80, kv_heads, page, dim, dtype=dtype, device="cuda") for _ in range(2))
    mass = torch.full((80, kv_heads, page), 7.0, device="cuda")          # what earlier requests left: a new key starts from nothing
    exact = {}                                                           # request -> [kv_heads, own keys] in 64 bits
    history = {}                                                         # request -> list of (k, v) of its whole context
    scale = dim ** -0.5

    def normal(*shape):
        return torch.randn(shape, generator=gen).to(dtype)

    def put(table, position, k, v):
        for pool_tensor, rows in ((keys, k), (values, v)):
            pool_tensor[table[position // page], :, position % page] = rows.cuda()

    pool.create_sequence("prefix")
    assert pool.append_tokens("prefix", shared).ok
    front = list(pool.block_table("prefix"))
    common = [(normal(kv_heads, dim), normal(kv_heads, dim)) for _ in range(shared)]
    for j, (k, v) in enumerate(common):
        put(front, j, k, v)

    def tables():
        rows = [front + list(pool.block_table(b)) for b in range(seqs)]
        return torch.tensor([r + [-1] * (max(map(len, rows)) - len(r)) for r in rows], dtype=torch.int32)

    def extend(b, count):
        assert pool.append_tokens(b, count).ok
        table = front + list(pool.block_table(b))
        for j in range(len(history[b]), len(history[b]) + count):
            k, v = normal(kv_heads, dim), normal(kv_heads, dim)
            history[b].append((k, v))
            put(table, j, k, v)

    def weights(b, q):
        """[heads, queries, keys] of the last queries of request b, [tokens, heads, dim]."""
        k = torch.stack([r[0] for r in history[b]]).double().transpose(0, 1).repeat_interleave(share, 0)
        n, t = k.shape[1], q.shape[0]
        hidden = torch.arange(n)[None] > torch.arange(n - t, n)[:, None]
        return torch.softmax((q.double().transpose(0, 1) @ k.transpose(1, 2) * scale).masked_fill(hidden, -math.inf), -1)

    def outputs(b, q):
        v = torch.stack([r[1] for r in history[b]]).double().transpose(0, 1).repeat_interleave(share, 0)
        return (weights(b, q) @ v).transpose(0, 1).flatten(1)

    def step(tokens, attend):
        """All requests bring `tokens[b]` new tokens; `attend` is called with the step's tensors and its output is checked."""
        for b, t in enumerate(tokens):
            extend(b, t)
        qkv = normal(sum(tokens), (heads + 2 * kv_heads) * dim)
        starts = [sum(tokens[:b]) for b in range(seqs + 1)]
        lengths = [len(history[b]) for b in range(seqs)]
        q = qkv[:, : heads * dim].view(-1, heads, dim)
        out = attend(qkv.cuda(), keys, values, tables().cuda(), i32(starts, "cuda"), i32([n - t for n, t in zip(lengths, tokens)], "cuda"), i32(lengths, "cuda"),
                     max(tokens), lengths)
        want = torch.cat([outputs(b, q[starts[b] : starts[b + 1]]) for b in range(seqs)])
        assert (out.cpu().double() - want).abs().max() <= output_tolerance(dtype, want)
        return [q[starts[b] : starts[b + 1]] for b in range(seqs)]

    def with_mass(qkv, keys, values, table, q_start, q_pos0, kv_len, longest, lengths):
        return ops.paged_attention_mass(qkv, keys, values, mass, table, q_start, q_pos0, kv_len, heads, kv_heads, dim, page, longest, max(lengths), scale,
                                        keep_first=shared)

    def behind_prefix(qkv, keys, values, table, q_start, q_pos0, kv_len, longest, lengths):
        return ops.paged_attention_prefix(qkv, keys, values, table, q_start, q_pos0, kv_len, i32([shared] * seqs, "cuda"), i32([0, seqs], "cuda"), heads, kv_heads,
                                          dim, page, longest, shared, max(lengths) - shared, longest * seqs, scale)

    def add_exact(queries):
        for b, q in enumerate(queries):
            w = weights(b, q).sum(1).view(kv_heads, share, -1).sum(1)[:, shared:]
            before = torch.zeros_like(w)
            if b in exact:
                before[:, : exact[b].shape[1]] = exact[b]
            exact[b] = before + w

    # Prompts behind the prefix, then tokens one by one.
    for b in range(seqs):
        pool.create_sequence(b)
        history[b] = list(common)
    add_exact(step(prompts, with_mass))
    for _ in range(steps):
        add_exact(step([1] * seqs, with_mass))
    step([1] * seqs, lambda *a: behind_prefix(*a))          # brings keys without weights: these start from nothing at the next step that adds
    for b in range(seqs):
        n = len(history[b])
        table = front + list(pool.block_table(b))
        got = torch.stack([mass[table[j // page], :, j % page] for j in range(shared, n - 1)], 1).cpu().double()
        assert (got - exact[b]).abs().max() <= 1e-4 * max(1.0, float(exact[b].max()))
        mass[table[(n - 1) // page], :, (n - 1) % page] = 0.0
    shared_rows = (keys[front].clone(), values[front].clone(), mass[front].clone())

    # Back to the prefix and `budget_behind` keys behind it.
    budget = shared + budget_behind
    lengths = [len(history[b]) for b in range(seqs)]
    table, kv_len = tables().cuda(), i32(lengths, "cuda")
    kept = ops.choose_kept(mass, table, kv_len, budget, shared, keep_last, max(lengths))
    before = mass.clone()
    ops.compact_kept(keys, values, mass, table, kv_len, kept)
    assert all(torch.equal(a, b) for a, b in zip(shared_rows, (keys[front], values[front], mass[front])))
    for b in range(seqs):
        n = lengths[b]
        t = front + list(pool.block_table(b))
        per_head = []
        for g in range(kv_heads):
            m = [float(before[t[j // page], g, j % page]) for j in range(n)]
            middle = sorted(range(shared, n - keep_last), key=lambda j: (-m[j], j))[: budget_behind - keep_last]
            want = sorted([*range(shared), *middle, *range(n - keep_last, n)]) if n > budget else list(range(n))
            assert kept[b, g].tolist() == want + [-1] * (budget - len(want))
            per_head.append(want)
        count = len(per_head[0])
        history[b] = [(torch.stack([history[b][per_head[g][i]][0][g] for g in range(kv_heads)]), torch.stack([history[b][per_head[g][i]][1][g] for g in range(kv_heads)]))
                      for i in range(count)]
        pool.shorten_sequence(b, count - shared)
    # The pages that came back serve others, whose rows are not the kept ones'.
    pool.create_sequence("other")
    assert pool.append_tokens("other", 6 * page).ok
    for block in pool.block_table("other"):
        keys[block], values[block], mass[block] = 99.0, math.inf, math.nan
    for tokens in ([1] * seqs, [3, 1, 2, 1, 5], [1] * seqs):
        step(tokens, behind_prefix)
    step([1] * seqs, with_mass)
    ops.check_device_errors()
