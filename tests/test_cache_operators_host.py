"""Refusals of the operators on a shared and pruned paged cache: said before any kernel is looked for, so without a GPU."""

import pytest
import torch

from paged_attention_engine_b200.kernels import ops


def _i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def _choose(mass=None, block_table=None, kv_len=None, budget=8, keep_first=1, keep_last=2, max_kv_len=64):
    return ops.choose_kept(torch.zeros(9, 2, 16) if mass is None else mass, _i32(3, 4) if block_table is None else block_table, _i32(3) if kv_len is None else kv_len,
                           budget, keep_first, keep_last, max_kv_len)


@pytest.mark.parametrize("arguments,message", [
    (dict(mass=torch.zeros(9, 2, 16, dtype=torch.bfloat16)), "mass is torch.bfloat16"), (dict(mass=torch.zeros(9, 16)), "float32 \\[pages, kv_heads, page_size\\] is needed"),
    (dict(block_table=_i32(3, 4).long()), "block_table is torch.int64"), (dict(kv_len=torch.zeros(3)), "kv_len is torch.float32"),
    (dict(kv_len=_i32(4)), "block tables \\(3, 4\\) for lengths \\(4,\\)"), (dict(block_table=_i32(12)), "block tables"), (dict(block_table=_i32(3, 0)), "block tables"),
    (dict(budget=0, keep_first=0, keep_last=0), "of a budget of 0"), (dict(keep_first=-1), "-1 first"), (dict(keep_last=-1), "-1 last"), (dict(keep_first=7), "7 first and 2 last keys of a budget of 8"),
    (dict(max_kv_len=65), "65 keys for tables of 4 pages of 16"), (dict(max_kv_len=-1), "-1 keys"), (dict(), "mass is not on a CUDA device")])
def test_choice_refuses(arguments, message):
    with pytest.raises(ops.KernelError, match=message):
        _choose(**arguments)


def _compact(keys=None, values=None, mass=None, block_table=None, kv_len=None, kept=None):
    return ops.compact_kept(torch.zeros(9, 2, 16, 8) if keys is None else keys, values, mass, _i32(3, 4) if block_table is None else block_table,
                            _i32(3) if kv_len is None else kv_len, _i32(3, 2, 5) if kept is None else kept)


@pytest.mark.parametrize("arguments,message", [
    (dict(keys=torch.zeros(9, 2, 16)), "head size\\] is needed"), (dict(kept=_i32(3, 2, 5).long()), "kept is torch.int64"), (dict(kept=_i32(3, 1, 5)), "kept \\(3, 1, 5\\) for 3 requests of 2 kv heads"),
    (dict(kept=_i32(2, 2, 5)), "kept \\(2, 2, 5\\)"), (dict(values=torch.zeros(9, 2, 8, 8)), "beside keys"), (dict(values=torch.zeros(9, 2, 16, 8, dtype=torch.bfloat16)), "beside keys"),
    (dict(mass=torch.zeros(9, 2, 16, 8)), "mass torch.float32"), (dict(mass=torch.zeros(9, 2, 16, dtype=torch.float64)), "mass torch.float64"),
    (dict(kv_len=_i32(2)), "block tables"), (dict(), "keys is not on a CUDA device")])
def test_compaction_refuses(arguments, message):
    with pytest.raises(ops.KernelError, match=message):
        _compact(**arguments)
