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


@pytest.mark.parametrize("tokens,heads,kv_heads,longest", [
    ([1] * 64, 40, 8, 9000),                                    # slices of single tokens
    ([5] * 64, 40, 8, 9000),                                    # few tokens
    ([16] + [1 + 5 * b % 16 for b in range(63)], 40, 8, 9000),
    ([16] * 6, 128, 1, 9000),                                   # one request's scores alone are beyond the limit
    ([20] + [17] * 300, 8, 8, 9000),                            # portions
    ([1] * 64, 17, 1, 40000),                                    # more query heads than the slices of single tokens take
])
def test_scratch_has_a_bound(ops, monkeypatch, tokens, heads, kv_heads, longest):
    """One long context among many short ones: what a call takes beside its operands and results stays below the limit, in requests by parts."""
    monkeypatch.setattr(ops, "MASS_SCRATCH_BYTES", 64 << 20, raising=False)
    lengths = [longest] + [max(t, 20 + 37 * b % 300) for b, t in enumerate(tokens[1:])]
    step = Step(lengths, tokens, heads, kv_heads, 128, 64, BF16, 3)
    pools, tables = step.on()
    mass = step.mass.cuda()
    run = lambda: ops.paged_attention_mass(*pools, mass, *tables, *step.sizes, *step.longest, step.scale)
    out = run()
    got = mass.clone()
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    again = run()
    torch.cuda.synchronize()
    beside = torch.cuda.max_memory_allocated() - before - 2 * again.numel()
    ops.check_device_errors()
    assert beside <= ops.MASS_SCRATCH_BYTES + (4 << 20)
    del again
    # The requests of the first and the last part against the definition.
    start = step.q_start.tolist()
    for b in (0, 1, len(tokens) - 1):
        w = step.weights(b)
        v = step.rows(step.values, b).double().repeat_interleave(heads // kv_heads, 0)
        want = (w @ v).transpose(0, 1).flatten(1)
        assert (out[start[b] : start[b + 1]].cpu().double() - want).abs().max() <= output_tolerance(BF16, want)
        n, t = lengths[b], tokens[b]
        j = torch.arange(n)
        p, o = step.table[b].long()[j // 64], j % 64
        expected = torch.where(j[:, None] >= n - t, 0.0, step.mass[p, :, o].double()) + w.sum(1).view(kv_heads, -1, n).sum(1).T
        assert ((got.cpu()[p, :, o].double() - expected).abs() <= MASS_RTOL * expected + MASS_ATOL).all()


@pytest.mark.parametrize("dtype,dim,tokens,padding", [
    (BF16, 128, [70, 20, 130], 1), (BF16, 64, [300, 17, 1, 40], 1), (BF16, 128, [1, 90, 1], 0), (BF16, 64, [3, 2, 5], 1), (BF16, 128, [16, 16], 1), (F32, 64, [3, 2, 5], 1),
    (F32, 64, [70, 90, 1], 1), (BF16, 32, [20, 33, 5], 1), (F32, 64, [1, 1, 1], 2), (BF16, 32, [1, 1, 1], 0)])
def test_requests_that_pad_a_step(ops, dtype, dim, tokens, padding):
    """Slots of -1, whether such a request brings one token or many, in every kernel: the pages it names keep their weights bit for bit."""
    step = Step([340, 150, 420, 95][: len(tokens)], tokens, 12, 2, dim, 16, dtype, dim + sum(tokens))
    named = step.table[padding].clone()
    slots = torch.cat([torch.full((t,), -1 if b == padding else 5, dtype=torch.int32) for b, t in enumerate(tokens)]).cuda()
    out, mass = _run(ops, step, slots=slots)
    _check(step, out, mass, pads=(padding,))
    named = named[named >= 0].long()
    assert torch.equal(mass.cpu()[named], step.mass[named])
