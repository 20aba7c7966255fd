"""What the pages hold behind a request's last key (an earlier request's rows, no numbers at all) does not reach the output of any of the
attention kernels."""

import pytest
import torch

from cache_operators import Step, output_tolerance

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from paged_attention_engine_b200.kernels import ops as kernel_ops

    yield kernel_ops
    kernel_ops.PLANNED_MIN_TILES = 4000


@pytest.mark.parametrize("lengths,tokens", [([5, 33, 700], [1, 1, 1]), ([40, 200], [40, 3]), ([70, 1000, 9], [70, 65, 9]), ([300, 77, 130], [129, 1, 130]), ([900], [64])])
@pytest.mark.parametrize("heads,kv_heads,dim,page,dtype", [(12, 2, 128, 16, torch.bfloat16), (8, 8, 64, 32, torch.bfloat16), (4, 2, 128, 128, torch.bfloat16),
                                                            (4, 1, 32, 16, torch.bfloat16), (5, 5, 48, 8, torch.bfloat16), (4, 2, 64, 16, torch.float32)])
@pytest.mark.parametrize("form", [0, 1, 2, 4])
def test_rows_behind_the_last_key(ops, lengths, tokens, heads, kv_heads, dim, page, dtype, form):
    step = Step(lengths, tokens, heads, kv_heads, dim, page, dtype, 3)
    pools, tables = step.on()
    out = ops.paged_attention(*pools, *tables, *step.sizes, *step.longest, step.scale, 0, form=form)
    want = step.attention()
    assert (out.cpu().double() - want).abs().max() <= output_tolerance(dtype, want)
    ops.check_device_errors()


def test_planned_slices(ops):
    step = Step([5, 33, 700, 1000, 17], [1] * 5, 12, 2, 128, 16, torch.bfloat16, 4)
    pools, tables = step.on()
    ops.PLANNED_MIN_TILES = 1
    ops.plan_decode(tables[1], tables[3], 1000, 12, 2, 128, 16, 0, torch.bfloat16)
    ops.PLANNED_MIN_TILES = 4000
    out = ops.paged_attention(*pools, *tables, *step.sizes, *step.longest, step.scale, 0)
    want = step.attention()
    assert (out.cpu().double() - want).abs().max() <= output_tolerance(step.dtype, want)
