"""`paged_attention_mass` with more than 16 query heads a kv head, which the slices of single tokens do not take: the tensor-core kernels of few tokens and of portions, the
latter with the requests of one token among them."""

import pytest
import torch

from cache_operators import Step, i32, output_tolerance

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
# As test_attention_mass_gpu.py derives them.
MASS_RTOL, MASS_ATOL = 1e-4, 1e-6


@pytest.fixture(scope="module")
def ops():
    from paged_attention_engine_b200.kernels import ops as kernel_ops

    return kernel_ops


def _check(ops, step, kernel, keep_first=0, pads=(), **more):
    pools, tables = step.on()
    mass, info = step.mass.cuda(), {}
    out = ops.paged_attention_mass(*pools, mass, *tables, *step.sizes, *step.longest, step.scale, keep_first=keep_first, info=info, **more)
    torch.cuda.synchronize()
    ops.check_device_errors()
    want = step.attention()
    rows = [r for b, t in enumerate(step.tokens) if b not in pads for r in range(int(step.q_start[b]), int(step.q_start[b]) + t)]
    assert (out.cpu().double() - want)[rows].abs().max() <= output_tolerance(BF16, want)
    expected, got = step.masses(keep_first, pads), mass.cpu().double()
    same = expected == step.mass.double()
    assert torch.equal(got[same], expected[same])
    assert ((got - expected).abs() <= MASS_RTOL * expected + MASS_ATOL).all()
    assert info["kernel"] == kernel


HEADS = [(40, 2, 128, 16), (17, 1, 64, 64), (128, 1, 64, 16), (66, 2, 128, 128)]


@pytest.mark.parametrize("heads,kv_heads,dim,page", HEADS)
@pytest.mark.parametrize("lengths,tokens,kernel", [
    ([1], [1], "few"), ([900, 64, 1500, 5], [1] * 4, "few"), ([70, 33], [5, 1], "few"), ([17], [17], "portions"), ([700, 300, 1], [200, 1, 1], "portions"),
    ([1500, 129], [33, 129], "portions")])
def test_steps(ops, heads, kv_heads, dim, page, lengths, tokens, kernel):
    step = Step(lengths, tokens, heads, kv_heads, dim, page, BF16, heads + sum(tokens))
    for keep_first in (0, 40):
        _check(ops, step, kernel, keep_first)


@pytest.mark.parametrize("heads,kv_heads,dim,page", HEADS[:2])
def test_mixed_and_padded_steps(ops, heads, kv_heads, dim, page):
    step = Step([300, 500, 77, 200], [1, 130, 1, 200], heads, kv_heads, dim, page, BF16, 9)
    _check(ops, step, "portions", num_single=2, multi_index=i32([1, 3], "cuda"))
    slots = torch.cat([torch.full((t,), -1 if b in (0, 3) else 5, dtype=torch.int32) for b, t in enumerate(step.tokens)]).cuda()
    _check(ops, step, "portions", pads=(0, 3), slots=slots)


def test_what_ran_by_the_sizes(ops):
    """The kernel that a step takes where 16 query heads and fewer share a kv head, and on CUDA cores."""
    for heads, dim, page, dtype, tokens, kernel in ((12, 128, 16, BF16, [1, 1], "single"), (12, 32, 48, BF16, [1, 1], "single"), (12, 128, 16, BF16, [3, 1], "few"),
                                                    (12, 64, 16, BF16, [17, 1], "portions"), (12, 64, 48, BF16, [17, 1], "rows"), (12, 64, 16, torch.float32, [1, 1], "single simt"),
                                                    (12, 64, 16, torch.float32, [2, 1], "rows"), (40, 64, 16, torch.float32, [1, 1], "rows"), (40, 48, 16, BF16, [1, 1], "rows")):
        step = Step([60, 50], tokens, heads, 2, dim, page, dtype, 3)
        pools, tables = step.on()
        info = {}
        ops.paged_attention_mass(*pools, step.mass.cuda(), *tables, *step.sizes, *step.longest, step.scale, info=info)
        assert info["kernel"] == kernel
    ops.check_device_errors()
