"""Eviction from the paged cache (csrc/evict.cu): the choice of the keys that stay is that of a stable sort, whatever
the weights are, and the move of their rows to the front leaves everything else as it was."""

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from paged_attention_engine_b200.kernels import ops as kernel_ops

    return kernel_ops


def _tables(lengths, page, seed, spare=2):
    """Block tables over pages in any order, -1 behind a request's last page."""
    counts = [-(-n // page) for n in lengths]
    order = np.random.RandomState(seed).permutation(sum(counts) + spare).astype(np.int32)
    table, at = np.full((len(lengths), max(1, max(counts))), -1, dtype=np.int32), 0
    for b, c in enumerate(counts):
        table[b, :c] = order[at : at + c]
        at += c
    return table, sum(counts) + spare


def _chosen(weights, n, budget, first, last):
    """The definition: all of n <= budget; else the protected keys and the largest weights, equal ones in order."""
    if n <= budget:
        return list(range(n))
    value = lambda i: math.inf if math.isnan(weights[i]) else float(weights[i])  # noqa: E731
    middle = sorted(range(first, n - last), key=lambda i: (-math.isnan(weights[i]), -value(i), i))
    return sorted([*range(first), *middle[: budget - first - last], *range(n - last, n)])


def _weights(kind, gen, *shape):
    if kind == "spread":
        return torch.randn(shape, generator=gen).mul_(3).exp_()
    if kind == "equal":
        return torch.full(shape, 0.25)
    if kind == "few values":
        return torch.randint(0, 3, shape, generator=gen).float() * 1e-30
    if kind == "near":                        # neighbours among the 32-bit numbers
        return (torch.randint(0, 400, shape, generator=gen) + (1 << 23) * 127).int().view(torch.float32)
    w = torch.randn(shape, generator=gen)     # signs, zeros of both signs, infinities, no numbers
    pick = torch.randint(0, 8, shape, generator=gen)
    for code, value in ((0, math.inf), (1, -math.inf), (2, math.nan), (3, 0.0), (4, -0.0)):
        w[pick == code] = value
    return w


@pytest.mark.parametrize("kind", ["spread", "equal", "few values", "near", "special"])
@pytest.mark.parametrize("lengths,budget,first,last,page,kv_heads", [
    ([1, 2, 5, 0], 1, 0, 0, 16, 2), ([5, 1, 700, 64, 65], 64, 3, 10, 16, 3), ([300, 301, 299, 1000], 300, 0, 300, 16, 1),
    ([300, 777], 300, 300, 0, 48, 2), ([4097, 2047, 9000], 2000, 4, 64, 16, 2), ([100, 90], 99, 1, 0, 7, 2), ([33], 32, 0, 31, 1, 1), ([20000] * 3, 19999, 5, 6, 64, 1)])
def test_choice(ops, kind, lengths, budget, first, last, page, kv_heads):
    gen = torch.Generator().manual_seed(len(lengths) + budget)
    table, pages = _tables(lengths, page, budget)
    mass = _weights(kind, gen, pages, kv_heads, page)
    kept = ops.choose_kept(mass.cuda(), torch.from_numpy(table).cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(), budget, first, last, max(lengths))
    assert kept.shape == (len(lengths), kv_heads, budget) and kept.dtype == torch.int32
    for b, n in enumerate(lengths):
        rows = mass[torch.from_numpy(table[b, : -(-n // page)]).long()].transpose(0, 1).reshape(kv_heads, -1)[:, :n].numpy()
        for g in range(kv_heads):
            want = _chosen(rows[g], n, budget, first, last)
            assert kept[b, g].tolist() == want + [-1] * (budget - len(want)), (b, g)


@pytest.mark.parametrize("lengths,budget", [([140000], 5000), ([131072, 17], 131071), ([420000], 30000)])
def test_choice_of_long_rows(ops, lengths, budget):
    """Clusters of blocks, and rows longer than the cluster's shared memory; the reference is a stable sort."""
    page, kv_heads = 64, 2
    gen = torch.Generator().manual_seed(budget)
    table, pages = _tables(lengths, page, 3)
    mass = torch.randn(pages, kv_heads, page, generator=gen).half().float()
    kept = ops.choose_kept(mass.cuda(), torch.from_numpy(table).cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(), budget, 4, 100, max(lengths)).cpu()
    for b, n in enumerate(lengths):
        if n <= budget:
            assert (kept[b, :, :n] == torch.arange(n)).all() and (kept[b, :, n:] == -1).all()
            continue
        rows = mass[torch.from_numpy(table[b, : -(-n // page)]).long()].transpose(0, 1).reshape(kv_heads, -1)[:, :n].clone()
        rows[:, :4] = math.inf
        rows[:, n - 100 :] = math.inf
        want = rows.sort(dim=1, descending=True, stable=True).indices[:, :budget].sort(dim=1).values
        assert torch.equal(kept[b].long(), want)


@pytest.mark.parametrize("dtype,dim,value_dim", [(torch.bfloat16, 128, 128), (torch.float32, 64, 64), (torch.bfloat16, 36, 128), (torch.bfloat16, 7, 7), (torch.bfloat16, 576, 0),
                                                 (torch.float32, 3, 5), (torch.bfloat16, 32, 32)])
@pytest.mark.parametrize("lengths,budget,page", [([3000, 1200, 900, 1], 1000, 16), ([50, 49], 20, 7), ([2500], 2499, 64), ([4000], 1, 16)])
def test_compaction(ops, dtype, dim, value_dim, lengths, budget, page):
    """Rows of the kept keys at the front, everything else bit for bit as before: other requests' pages, pages of nobody, rows behind."""
    kv_heads = 2
    gen = torch.Generator().manual_seed(dim + budget)
    table, pages = _tables(lengths, page, dim)
    keys = torch.randn(pages, kv_heads, page, dim, generator=gen).to(dtype)
    values = torch.randn(pages, kv_heads, page, value_dim, generator=gen).to(dtype) if value_dim else None
    mass = torch.rand(pages, kv_heads, page, generator=gen)
    kept = torch.full((len(lengths), kv_heads, budget), -1, dtype=torch.int32)
    for b, n in enumerate(lengths):
        for g in range(kv_heads):
            stay = min(n, budget)
            kept[b, g, :stay] = torch.randperm(n, generator=gen)[:stay].sort().values.int()
    pools = [keys] + ([values] if value_dim else []) + [mass]
    want = [t.clone() for t in pools]
    for pool, moved in zip(pools, want):
        for b, n in enumerate(lengths):
            at = torch.arange(n)
            p, o = torch.from_numpy(table[b])[at // page].long(), at % page
            for g in range(kv_heads):
                k = kept[b, g, : min(n, budget)].long()
                moved[p[: len(k)], g, o[: len(k)]] = pool[p[k], g, o[k]]
    dev = [t.cuda() for t in pools]
    ops.compact_kept(dev[0], dev[1] if value_dim else None, dev[-1], torch.from_numpy(table).cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(), kept.cuda())
    for got, expected in zip(dev, want):
        assert torch.equal(got.cpu().view(torch.uint8), expected.view(torch.uint8))


def test_values_in_the_keys_move_once_and_mass_may_be_absent(ops):
    lengths, budget, page = [200], 90, 16
    table, pages = _tables(lengths, page, 1)
    keys = torch.randn(pages, 1, page, 64).to(torch.bfloat16)
    kept = torch.arange(20, 200, 2, dtype=torch.int32).view(1, 1, 90)
    dev = keys.cuda()
    ops.compact_kept(dev, dev, None, torch.from_numpy(table).cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(), kept.cuda())
    at = torch.arange(200)
    p, o = torch.from_numpy(table[0])[at // page].long(), at % page
    rows = dev.cpu()[p, 0, o]
    before = keys[p, 0, o]
    assert torch.equal(rows[:90], before[kept[0, 0].long()]) and torch.equal(rows[90:], before[90:])


def test_indices_that_name_no_row_move_nothing(ops):
    """-1, an index that is not below the request's length, and one below its place."""
    lengths, page = [64, 64], 16
    table, pages = _tables(lengths, page, 2)
    keys = torch.randn(pages, 1, page, 8)
    kept = torch.tensor([[[-1, 64, 1, 1000000, -2147483648, 63]], [[0, 1, 2, 3, 3, 2147483647]]], dtype=torch.int32)
    dev = keys.cuda()
    ops.compact_kept(dev, None, None, torch.from_numpy(table).cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(), kept.cuda())
    want = keys.clone()
    at = torch.arange(64)
    p, o = torch.from_numpy(table[0])[at // page].long(), at % page
    want[p[5], 0, o[5]] = keys[p[63], 0, o[63]]
    assert torch.equal(dev.cpu(), want)


def test_captured_and_replayed_with_other_lengths_and_weights(ops):
    page, kv_heads, dim, budget = 16, 2, 64, 200
    lengths = [500, 150, 333]
    table, pages = _tables([600, 600, 600], page, 9)
    table = torch.from_numpy(table).cuda()
    gen = torch.Generator(device="cuda").manual_seed(4)
    keys, values = (torch.randn(pages, kv_heads, page, dim, device="cuda", generator=gen) for _ in range(2))
    mass = torch.rand(pages, kv_heads, page, device="cuda", generator=gen)
    kv_len = torch.tensor(lengths, dtype=torch.int32, device="cuda")

    def once(k, v, m):
        kept = ops.choose_kept(m, table, kv_len, budget, 4, 20, 600)
        ops.compact_kept(k, v, m, table, kv_len, kept)
        return kept

    once(keys.clone(), values.clone(), mass.clone())
    fixed = [t.clone() for t in (keys, values, mass)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded = once(*fixed)
    for new in ([600, 200, 201], [1, 0, 599]):
        kv_len.copy_(torch.tensor(new, dtype=torch.int32))
        for t, start in zip(fixed, (keys, values, mass)):
            t.copy_(start.roll(new[0], 0))
        eager = [t.clone() for t in fixed]
        graph.replay()
        kept = once(*eager)
        assert torch.equal(kept, recorded) and all(torch.equal(a, b) for a, b in zip(fixed, eager))


def test_on_another_stream(ops):
    """The kernels run on the current stream, behind what made their inputs there."""
    page, budget = 16, 1000
    table, pages = _tables([4000] * 8, page, 5)
    table, kv_len = torch.from_numpy(table).cuda(), torch.full((8,), 4000, dtype=torch.int32, device="cuda")
    mass = torch.rand(pages, 4, page, device="cuda")
    want = ops.choose_kept(mass, table, kv_len, budget, 0, 10, 4000)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        late = torch.zeros_like(mass)
        for _ in range(20):
            late.add_(1.0)
        late.copy_(mass)
        got = ops.choose_kept(late, table, kv_len, budget, 0, 10, 4000)
    side.synchronize()
    assert torch.equal(got, want)
