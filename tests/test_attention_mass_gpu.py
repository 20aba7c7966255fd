"""Attention that adds up its weights per key (csrc/attention_mass.cu) against the definition in 64 bits."""

import pytest
import torch

from cache_operators import Step, i32, output_tolerance

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
# Of a key's added weight, relative to its value plus the weight that a row's rounding can move: scores are sums of at most 256 products in
# 32 bits, |score| < 16 in units of log2, so a weight is off by 256 * 2^-24 * 16 at worst and by some 1e-6 of itself as a rule.
MASS_RTOL, MASS_ATOL = 1e-4, 1e-6


@pytest.fixture(scope="module")
def ops():
    from paged_attention_engine_b200.kernels import ops as kernel_ops

    return kernel_ops


def _run(ops, step, keep_first=0, slots=None, **more):
    pools, tables = step.on()
    mass = step.mass.cuda()
    out = ops.paged_attention_mass(*pools, mass, *tables, *step.sizes, *step.longest, step.scale, keep_first=keep_first, slots=slots, **more)
    torch.cuda.synchronize()
    return out, mass


def _check(step, out, mass, keep_first=0, pads=()):
    want = step.attention()
    rows = [r for b, t in enumerate(step.tokens) if b not in pads for r in range(int(step.q_start[b]), int(step.q_start[b]) + t)]
    assert torch.isfinite(out).all()
    assert (out.cpu().double() - want)[rows].abs().max() <= output_tolerance(step.dtype, want)
    expected = step.masses(keep_first, pads)
    got = mass.cpu().double()
    # Exactly as before where nothing is to be added.
    same = expected == step.mass.double()
    assert torch.equal(got[same], expected[same])
    assert ((got - expected).abs() <= MASS_RTOL * expected + MASS_ATOL).all()


SIZES = [(12, 2, 128, 16, BF16), (28, 4, 128, 16, BF16), (8, 8, 64, 32, BF16), (16, 1, 32, 48, BF16), (3, 1, 32, 16, F32), (12, 2, 64, 16, F32), (4, 4, 128, 7, F32),
         (5, 5, 48, 8, BF16), (40, 2, 64, 16, BF16), (4, 2, 256, 4, F32)]


@pytest.mark.parametrize("heads,kv_heads,dim,page,dtype", SIZES)
@pytest.mark.parametrize("lengths,keep_first", [([1], 0), ([1, 2, 16, 17, 33], 0), ([900, 64, 1500, 5], 4), ([2100], 600)])
def test_single_tokens(ops, heads, kv_heads, dim, page, dtype, lengths, keep_first):
    step = Step(lengths, [1] * len(lengths), heads, kv_heads, dim, page, dtype, heads + len(lengths))
    _check(step, *_run(ops, step, keep_first), keep_first)


@pytest.mark.parametrize("heads,kv_heads,dim,page,dtype", SIZES)
@pytest.mark.parametrize("lengths,tokens", [([5], [5]), ([70, 200, 9], [70, 33, 9]), ([130, 400], [1, 129]), ([300], [64]), ([64, 65, 1], [2, 64, 1])])
def test_portions(ops, heads, kv_heads, dim, page, dtype, lengths, tokens):
    step = Step(lengths, tokens, heads, kv_heads, dim, page, dtype, heads + sum(tokens))
    for keep_first in (0, 20):
        _check(step, *_run(ops, step, keep_first), keep_first)


def test_many_requests_and_slices(ops):
    step = Step([3 + 37 * i % 1200 for i in range(70)], [1] * 70, 28, 4, 128, 16, BF16, 2)
    _check(step, *_run(ops, step))
    step = Step([9000, 12], [1, 1], 12, 2, 128, 64, BF16, 3)
    _check(step, *_run(ops, step))


@pytest.mark.parametrize("tokens", [[1, 1, 1], [3, 1, 2]])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rows_that_pad_a_step_add_nothing(ops, tokens, dtype):
    """As a recorded step's padding rows: position 0 of nobody's request, in page 0, slot -1."""
    step = Step([40, 1, 300], tokens if tokens[1] == 1 else tokens, 4, 2, 64, 16, dtype, 5)
    step.table[1, 0] = step.table[0, 0]                       # the page of a request's first keys
    step.q_pos0[1] = 0
    slots = i32([s for b, t in enumerate(tokens) for s in [-1 if b == 1 else 0] * t], "cuda")
    _check(step, *_run(ops, step, slots=slots), pads=(1,))


def test_pages_of_kept_keys_may_be_shared(ops):
    step = Step([100, 130, 77], [1, 1, 1], 12, 2, 128, 16, BF16, 7, shared=((3, 64),))
    _check(step, *_run(ops, step, keep_first=64), keep_first=64)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("tokens", [1, 70])
def test_captured_and_replayed(ops, dtype, tokens):
    steps = [Step(lengths, [tokens] * 3, 12, 2, 64, 16, dtype, 11 + i, width=20) for i, lengths in enumerate(([300, 90, 70], [71, 270, 300]))]
    first, second = ([*s.on()[0], s.mass.cuda(), *s.on()[1]] for s in steps)
    args = (*steps[0].sizes, tokens, 320, steps[0].scale)
    pages = max(t.shape[0] for t in (first[1], second[1]))
    fixed = [torch.zeros((pages, *a.shape[1:]), dtype=a.dtype, device="cuda") if i in (1, 2, 3) else a.clone() for i, a in enumerate(first)]

    def fill(source):
        for to, a in zip(fixed, source):
            to[: a.shape[0]].copy_(a)

    fill(first)
    ops.paged_attention_mass(*fixed, *args)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.paged_attention_mass(*fixed, *args)
    for step, source in zip(steps[::-1], (second, first)):
        fill(source)
        graph.replay()
        torch.cuda.synchronize()
        _check(step, out, fixed[3][: source[3].shape[0]])


def test_equal_bits_in_every_run_and_batch(ops):
    """Nothing is added by atomics, and a request's weights do not depend on what else is in the step (as long as the slices are the same)."""
    step = Step([700] * 6, [1] * 6, 12, 2, 128, 16, BF16, 13)
    runs = [_run(ops, step) for _ in range(3)]
    assert all(torch.equal(o, runs[0][0]) and torch.equal(m, runs[0][1]) for o, m in runs)
    step = Step([260, 90], [100, 90], 12, 2, 64, 16, F32, 13)
    runs = [_run(ops, step) for _ in range(3)]
    assert all(torch.equal(o, runs[0][0]) and torch.equal(m, runs[0][1]) for o, m in runs)


@pytest.mark.parametrize("heads,kv_heads,dim,page", [(28, 4, 128, 16), (12, 2, 64, 64), (40, 8, 128, 128), (5, 1, 128, 32), (128, 1, 64, 16), (8, 8, 128, 16)])
@pytest.mark.parametrize("lengths,tokens", [([1500], [1500]), ([2000, 900, 333], [700, 900, 1]), ([129, 128, 127, 1, 700], [129, 2, 127, 1, 1]), ([1800], [257])])
def test_long_portions(ops, heads, kv_heads, dim, page, lengths, tokens):
    """Keys as the rows of a tensor-core product, rows in chunks, beside requests of one token."""
    step = Step(lengths, tokens, heads, kv_heads, dim, page, BF16, heads + sum(tokens))
    for keep_first in (0, 130):
        _check(step, *_run(ops, step, keep_first), keep_first)
    ops.check_device_errors()


def test_a_mixed_step_as_the_engine_describes_it(ops):
    """`num_single` and the list of the requests that bring more than one token."""
    step = Step([300, 500, 77, 200], [1, 130, 1, 200], 12, 2, 128, 16, BF16, 9)
    _check(step, *_run(ops, step, num_single=2, multi_index=i32([1, 3], "cuda")))
    step = Step([300, 500], [64, 130], 12, 2, 128, 16, BF16, 9)
    _check(step, *_run(ops, step, num_single=0))


@pytest.mark.parametrize("heads,kv_heads,dim,page", [(28, 4, 128, 16), (12, 2, 64, 128), (40, 2, 128, 32), (8, 8, 64, 64)])
@pytest.mark.parametrize("lengths,tokens", [([900, 33, 2000, 5, 64], [5, 5, 5, 5, 5]), ([700, 300, 17], [16, 1, 9]), ([3, 2], [3, 2]), ([128, 4000], [2, 2])])
def test_few_tokens(ops, heads, kv_heads, dim, page, lengths, tokens):
    """Drafted tokens: slices of the keys that keep their scores."""
    step = Step(lengths, tokens, heads, kv_heads, dim, page, BF16, heads + sum(tokens))
    for keep_first in (0, 50):
        _check(step, *_run(ops, step, keep_first), keep_first)
    ops.check_device_errors()


@pytest.mark.parametrize("dim,requests", [(64, 4), (64, 8), (128, 4)])
def test_few_tokens_behind_more_than_32_slices(ops, dim, requests):
    """A long context beside short ones; a warp merges a row, 32 slices a round."""
    step = Step([26000, 40, 300, 17, 16, 90, 5000, 64][:requests], [16] * requests, 20, 1, dim, 16, BF16, requests)
    _check(step, *_run(ops, step))
    ops.check_device_errors()


@pytest.mark.parametrize("dtype,dim,page", [(BF16, 128, 16), (BF16, 64, 64), (F32, 64, 16)])
@pytest.mark.parametrize("tokens,max_q_len", [(1, 1), (3, 3), (90, 90)])
def test_requests_without_keys(ops, dtype, dim, page, tokens, max_q_len):
    """Steps that padding alone makes up, and a step without requests: rows without a key are zeros, no weight changes."""
    step = Step([70, 100], [1, 1], 12, 2, dim, page, dtype, 3)
    pools, (table, *_) = step.on()
    qkv = torch.randn(2 * tokens, 16 * dim, device="cuda").to(dtype)
    mass = step.mass.cuda()
    zeros = i32([0, 0], "cuda")
    for longest in (0, 64):
        for slots in (None, torch.full((2 * tokens,), -1, dtype=torch.int32, device="cuda")):
            out = ops.paged_attention_mass(qkv, pools[1], pools[2], mass, table, i32([0, tokens, 2 * tokens], "cuda"), zeros, zeros, *step.sizes, max_q_len, longest, step.scale,
                                           slots=slots)
            assert torch.equal(out, torch.zeros_like(out))
    assert ops.paged_attention_mass(qkv, pools[1], pools[2], mass, table[:0], i32([0], "cuda"), zeros[:0], zeros[:0], *step.sizes, max_q_len, 64, step.scale).shape == (2 * tokens, 12 * dim)
    assert torch.equal(mass.cpu(), step.mass)
    assert torch.equal(ops.choose_kept(mass, table, zeros, 5, 1, 1, 64), torch.full((2, 2, 5), -1, dtype=torch.int32, device="cuda"))
    ops.check_device_errors()
