"""Which head sizes the attentions of the shared and pruned cache take does not depend on a step's lengths: multiples of 4 up to 256, whatever the step."""

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


SIZES = [(5, 1, 20, 16, BF16), (3, 3, 4, 5, F32), (20, 1, 100, 48, BF16), (8, 2, 12, 16, F32), (4, 2, 252, 16, BF16), (6, 3, 48, 7, F32)]


@pytest.mark.parametrize("heads,kv_heads,dim,page,dtype", SIZES)
@pytest.mark.parametrize("shared,own,tokens", [
    (((3, 200),), [70, 1, 40], [1, 1, 1]),                       # short prefixes
    (((2, 0), (1, 90)), [70, 130, 40], [1, 5, 40]),              # nothing shared, a group of one
    (((2, 1100), (1, 30)), [90, 130, 40], [70, 130, 1]),         # portions
])
def test_shared_prefixes(ops, heads, kv_heads, dim, page, dtype, shared, own, tokens):
    prefix = [n for count, n in shared for _ in range(count)]
    step = Step([p + o for p, o in zip(prefix, own)], tokens, heads, kv_heads, dim, page, dtype, dim + sum(tokens), shared=shared)
    pools, tables = step.on()
    limits = max(tokens), max(prefix), max(own), max(sum(tokens[a:b]) for a, b in zip(step.group_start, step.group_start[1:]))
    out = ops.paged_attention_prefix(*pools, *tables, step.prefix_len.cuda(), step.groups.cuda(), *step.sizes, *limits, step.scale)
    want = step.attention()
    assert (out.cpu().double() - want).abs().max() <= output_tolerance(dtype, want)
    ops.check_device_errors()


@pytest.mark.parametrize("heads,kv_heads,dim,page,dtype", SIZES)
@pytest.mark.parametrize("lengths,tokens", [([300, 1, 40], [1, 1, 1]), ([70, 200, 9], [5, 16, 1]), ([400, 90], [130, 1])])
def test_weights(ops, heads, kv_heads, dim, page, dtype, lengths, tokens):
    step = Step(lengths, tokens, heads, kv_heads, dim, page, dtype, dim + sum(tokens))
    pools, tables = step.on()
    mass = step.mass.cuda()
    out = ops.paged_attention_mass(*pools, mass, *tables, *step.sizes, *step.longest, step.scale, keep_first=20)
    want = step.attention()
    assert (out.cpu().double() - want).abs().max() <= output_tolerance(dtype, want)
    expected = step.masses(20)
    assert ((mass.cpu().double() - expected).abs() <= MASS_RTOL * expected + MASS_ATOL).all()
    ops.check_device_errors()
