"""Head sizes and operands that the attentions of the shared and pruned cache refuse, whatever the lengths of a step: without a GPU."""

import pytest
import torch

from paged_attention_engine_b200.kernels import ops


def _i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


@pytest.mark.parametrize("operator", ["prefix", "mass"])
@pytest.mark.parametrize("longest", [1, 2000])
@pytest.mark.parametrize("dim", [2, 6, 30, 258, 260, 264, 512])
def test_head_sizes(operator, longest, dim):
    keys = torch.zeros(9, 2, 16, dim)
    step = torch.zeros(5, 8 * dim), keys, keys.clone()
    tables = _i32(3, 200), _i32(4), _i32(3), _i32(3)
    with pytest.raises(ops.KernelError, match=f"paged_attention_{operator}: head_dim {dim} is not a multiple of 4 in \\[4, 256\\]"):
        if operator == "prefix":
            ops.paged_attention_prefix(*step, *tables, _i32(3), _i32(2), 4, 2, dim, 16, 1, longest, 30, 3, 1.0)
        else:
            ops.paged_attention_mass(*step, torch.zeros(9, 2, 16), *tables, 4, 2, dim, 16, 1, longest, 1.0)


def test_operands_that_start_between_four_elements():
    for dtype, dim, boundary in ((torch.bfloat16, 20, "an 8"), (torch.bfloat16, 24, "a 16"), (torch.float32, 4, "a 16")):
        whole = torch.zeros(1025, dtype=dtype)
        assert whole.data_ptr() % 16 == 0
        operands = whole[:1024], whole[:1024], whole[1:]
        with pytest.raises(ops.KernelError, match=f"paged_attention_mass: an operand does not start on {boundary}-byte boundary"):
            ops._aligned_operands("paged_attention_mass", *operands, dim)
        assert ops._aligned_operands("paged_attention_mass", *operands[:2], whole[8:], dim)
