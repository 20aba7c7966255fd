"""`paged_attention_mass` (csrc/attention_mass.cu) in steps whose buffers and requests are not all alike: rows of the projection behind the last request, requests that
only pad the step, keys that are no number. Against the definition in 64 bits."""

import math

import pytest
import torch

from cache_operators import Step, i32, output_tolerance

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
# As test_attention_mass_gpu.py derives them: scores are sums of at most 256 products in 32 bits, |score| < 16 in units of log2.
MASS_RTOL, MASS_ATOL = 1e-4, 1e-6


@pytest.fixture(scope="module")
def ops():
    from paged_attention_engine_b200.kernels import ops as kernel_ops

    return kernel_ops


def _run(ops, step, qkv=None, keep_first=0, **more):
    pools, tables = step.on()
    mass = step.mass.cuda()
    out = ops.paged_attention_mass(pools[0] if qkv is None else qkv, *pools[1:], mass, *tables, *step.sizes, *step.longest, step.scale, keep_first=keep_first, **more)
    torch.cuda.synchronize()
    ops.check_device_errors()
    return out, mass


def _check(step, out, mass, keep_first=0, pads=()):
    want = step.attention()
    rows = [r for b, t in enumerate(step.tokens) if b not in pads for r in range(int(step.q_start[b]), int(step.q_start[b]) + t)]
    assert (out[: len(want)].cpu().double() - want)[rows].abs().max() <= output_tolerance(step.dtype, want)
    expected = step.masses(keep_first, pads)
    got = mass.cpu().double()
    same = expected == step.mass.double()
    assert torch.equal(got[same], expected[same])
    assert ((got - expected).abs() <= MASS_RTOL * expected + MASS_ATOL).all()


@pytest.mark.parametrize("lengths,tokens", [([300, 500], [1, 130]), ([300, 500, 70], [130, 1, 40]), ([40, 50], [3, 1]), ([40, 50, 9], [1, 1, 1])])
@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (BF16, 64), (F32, 64)])
@pytest.mark.parametrize("behind", [1, 200])
def test_rows_behind_the_last_request(ops, lengths, tokens, dtype, dim, behind):
    """A buffer with more rows than the requests bring, as a padded step has it: every request is served all the same, whatever the further rows hold."""
    step = Step(lengths, tokens, 12, 2, dim, 16, dtype, behind)
    qkv = torch.cat((step.qkv, torch.full((behind, step.qkv.shape[1]), math.nan, dtype=dtype))).cuda()
    _check(step, *_run(ops, step, qkv))


@pytest.mark.parametrize("dtype,dim,tokens", [(BF16, 128, [1, 1]), (BF16, 32, [1, 1]), (F32, 64, [1, 1]), (BF16, 128, [3, 5]), (BF16, 64, [90, 30]), (F32, 64, [4, 30])])
def test_a_key_that_is_no_number(ops, dtype, dim, tokens):
    """A row whose denominator is no number has no weights: that is what all of its keys get, by whichever kernel, and no other row's."""
    step = Step([400, 290], tokens, 12, 2, dim, 16, dtype, dim)
    step.keys[int(step.table[0, 7]), 1, 3] = math.nan           # key 115 of request 0 for kv head 1, which all of its tokens see
    out, mass = (t.cpu().double() for t in _run(ops, step))
    broken = torch.zeros_like(mass, dtype=torch.bool)
    j = torch.arange(400)
    broken[step.table[0].long()[j // 16], 1, j % 16] = True
    expected = step.masses()
    assert torch.equal(expected.isnan(), broken)
    assert torch.equal(mass.isnan(), broken)
    assert ((mass - expected)[~broken].abs() <= MASS_RTOL * expected[~broken] + MASS_ATOL).all()
    assert torch.equal(out.isnan(), step.attention().isnan())
