"""The scratch of `paged_attention_prefix` has a bound: beyond it each request reads its keys by itself."""

import pytest
import torch

from cache_operators import Step, output_tolerance

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,dim,tokens,kernels", [(torch.bfloat16, 128, 60, ("shared", "mma")), (torch.float32, 64, 3, ("shared simt", "simt"))])
def test_scratch_has_a_bound(monkeypatch, dtype, dim, tokens, kernels):
    from paged_attention_engine_b200.kernels import ops

    monkeypatch.setattr(ops, "PREFIX_SIMT_MIN_KEYS", 1)
    step = Step([300 + tokens + 500 * b for b in range(6)], [tokens] * 6, 12, 2, dim, 16, dtype, dim, shared=((6, 300),))
    pools, tables = step.on()
    want = step.attention()
    given = (*pools, *tables, step.prefix_len.cuda(), step.groups.cuda(), *step.sizes, tokens, 300, tokens + 2500, 6 * tokens, step.scale)
    for limit, kernel in ((1 << 30, kernels[0]), (100_000, kernels[1])):
        monkeypatch.setattr(ops, "PREFIX_SCRATCH_BYTES", limit, raising=False)
        info = {}
        ops.paged_attention_prefix(*given)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        out = ops.paged_attention_prefix(*given, num_single=0, info=info)
        torch.cuda.synchronize()
        beside = torch.cuda.max_memory_allocated() - before - out.numel() * out.element_size()
        ops.check_device_errors()
        assert (out.cpu().double() - want).abs().max() <= output_tolerance(dtype, want)
        assert info["kernel"] == kernel
        assert kernel == kernels[0] or beside <= 1 << 20
