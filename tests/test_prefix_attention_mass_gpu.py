"""Steps of `paged_attention_prefix` between steps of `paged_attention_mass`: the keys that such a step brings start from nothing in the weights."""

import math

import pytest
import torch

from cache_operators import Step, output_tolerance

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
# As test_attention_mass_gpu.py derives them.
MASS_RTOL, MASS_ATOL = 1e-4, 1e-6


@pytest.fixture(scope="module")
def ops():
    from paged_attention_engine_b200.kernels import ops as kernel_ops

    return kernel_ops


def _prefix(ops, step, mass, slots=None):
    pools, tables = step.on()
    groups = zip(step.group_start, step.group_start[1:])
    limits = max(step.tokens), max(step.prefix), max(n - p for n, p in zip(step.lengths, step.prefix)), max(sum(step.tokens[a:b]) for a, b in groups)
    info = {}
    out = ops.paged_attention_prefix(*pools, *tables, step.prefix_len.cuda(), step.groups.cuda(), *step.sizes, *limits, step.scale, mass=mass, slots=slots, info=info)
    torch.cuda.synchronize()
    ops.check_device_errors()
    want = step.attention()
    assert (out.cpu().double() - want).abs().max() <= output_tolerance(step.dtype, want)
    return info["kernel"]


CASES = [(12, 2, 128, 16, BF16, [1, 3, 1, 2], "shared"), (14, 2, 64, 128, BF16, [1, 1, 1, 1], "shared"), (12, 2, 128, 16, BF16, [70, 1, 3, 90], "tcgen05"),
         (3, 1, 32, 16, BF16, [1, 2, 1, 1], "mma"), (6, 3, 48, 7, F32, [1, 40, 1, 3], "simt")]


@pytest.mark.parametrize("heads,kv_heads,dim,page,dtype,tokens,kernel", CASES)
@pytest.mark.parametrize("padding", [None, 1])
def test_the_steps_keys_start_from_nothing(ops, heads, kv_heads, dim, page, dtype, tokens, kernel, padding):
    prefix = 200
    step = Step([prefix + t + 17 * b for b, t in enumerate(tokens)], tokens, heads, kv_heads, dim, page, dtype, dim, shared=((4, prefix),))
    left = torch.full_like(step.mass, math.nan)
    mass = left.clone().cuda()
    slots = None if padding is None else torch.cat([torch.full((t,), -1 if b == padding else 3, dtype=torch.int32) for b, t in enumerate(tokens)]).cuda()
    assert _prefix(ops, step, mass, slots) == kernel
    expected = left
    for b, (n, t) in enumerate(zip(step.lengths, tokens)):
        if b != padding:
            j = torch.arange(n - t, n)
            expected[step.table[b].long()[j // page], :, j % page] = 0.0
    assert torch.equal(mass.cpu().nan_to_num(-1.0), expected.nan_to_num(-1.0))


@pytest.mark.parametrize("heads,kv_heads,dim,page,dtype,tokens,kernel", CASES)
def test_weights_of_a_later_step_are_added_to_nothing(ops, heads, kv_heads, dim, page, dtype, tokens, kernel):
    """A step with weights over keys of which the last but one came with a step without: the weights of those are the later step's alone."""
    prefix, lengths = 200, [200 + t + 17 * b for b, t in enumerate(tokens)]
    before = Step(lengths, tokens, heads, kv_heads, dim, page, dtype, dim, shared=((4, prefix),))
    mass = before.mass.cuda()
    _prefix(ops, before, mass)
    after = Step([n + 1 for n in lengths], [1] * 4, heads, kv_heads, dim, page, dtype, dim + 1, shared=((4, prefix),))
    # The later step's cache stands in pages of its own: the weights go where they belong.
    moved = torch.zeros_like(after.mass)
    for b, n in enumerate(lengths):
        j = torch.arange(n)
        moved[after.table[b].long()[j // page], :, j % page] = mass.cpu()[before.table[b].long()[j // page], :, j % page]
    after.mass = moved
    pools, tables = after.on()
    mass = moved.cuda()
    ops.paged_attention_mass(*pools, mass, *tables, *after.sizes, *after.longest, after.scale, keep_first=prefix)
    torch.cuda.synchronize()
    ops.check_device_errors()
    for b, (n, t) in enumerate(zip(lengths, tokens)):
        j = torch.arange(n - t, n)
        got = mass.cpu()[after.table[b].long()[j // page], :, j % page].double()
        want = after.weights(b).sum(1).view(kv_heads, -1, n + 1).sum(1)[:, j].T
        assert ((got - want).abs() <= MASS_RTOL * want + MASS_ATOL).all()
