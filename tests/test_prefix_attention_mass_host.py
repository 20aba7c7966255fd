"""What `paged_attention_prefix` refuses of the weights it is given: said before any kernel is looked for, so without a GPU."""

import pytest
import torch

from paged_attention_engine_b200.kernels import ops


def _i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


@pytest.mark.parametrize("arguments,message", [
    (dict(mass=torch.zeros(9, 2, 16, dtype=torch.bfloat16)), "paged_attention_prefix: mass torch.bfloat16"), (dict(mass=torch.zeros(8, 2, 16)), "mass torch.float32 \\(8, 2, 16\\)"),
    (dict(mass=torch.zeros(9, 2, 16), slots=_i32(4)), "slots \\(4,\\) for 5 tokens"), (dict(mass=torch.zeros(9, 2, 16), slots=torch.zeros(5)), "slots is torch.float32"),
    (dict(mass=torch.zeros(9, 2, 16)), "is not on a CUDA device")])
def test_weights_that_do_not_belong_to_the_cache(arguments, message):
    keys = torch.zeros(9, 2, 16, 8)
    with pytest.raises(ops.KernelError, match=message):
        ops.paged_attention_prefix(torch.zeros(5, 64), keys, keys.clone(), _i32(3, 4), _i32(4), _i32(3), _i32(3), _i32(3), _i32(2), 4, 2, 8, 16, 2, 20, 30, 5, 1.0, **arguments)
