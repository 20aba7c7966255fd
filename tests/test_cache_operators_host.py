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
    (dict(kv_len=_i32(2)), "block tables"), (dict(keys=torch.zeros(1).expand(1 << 20, 2, 1024, 8)), "a pool of 2147483648 rows"),
    (dict(keys=torch.zeros(9, 2, 16, 5, dtype=torch.uint8)), "rows of 5 and 0 bytes"),
    (dict(keys=torch.zeros(9, 2, 16, 4, dtype=torch.uint8), values=torch.zeros(9, 2, 16, 3, dtype=torch.uint8)), "rows of 4 and 3 bytes"), (dict(), "keys is not on a CUDA device")])
def test_compaction_refuses(arguments, message):
    with pytest.raises(ops.KernelError, match=message):
        _compact(**arguments)


HEADS, KV_HEADS, DIM, PAGE = 4, 2, 8, 16


def _attention(**other):
    """The tensors of a step of 3 requests of 5 tokens in all, on the CPU, with some of them replaced."""
    given = dict(qkv=torch.zeros(5, (HEADS + 2 * KV_HEADS) * DIM), keys=torch.zeros(9, KV_HEADS, PAGE, DIM), values=torch.zeros(9, KV_HEADS, PAGE, DIM), block_table=_i32(3, 4),
                 q_start=_i32(4), q_pos0=_i32(3), kv_len=_i32(3))
    given.update({k: v for k, v in other.items() if k in given})
    return given


STEP_REFUSALS = [
    (dict(qkv=torch.zeros(5, 60)), "qkv \\(5, 60\\) for 4\\+2x2 heads of 8"), (dict(qkv=torch.zeros(5, 64, dtype=torch.float16)), "torch.float16 is not supported"),
    (dict(keys=torch.zeros(9, KV_HEADS, PAGE, DIM, dtype=torch.bfloat16)), "keys torch.bfloat16"), (dict(values=torch.zeros(9, KV_HEADS, 8, DIM)), "values torch.float32 \\(9, 2, 8, 8\\)"),
    (dict(values=torch.zeros(8, KV_HEADS, PAGE, DIM)), "values"), (dict(q_start=_i32(3)), "q_start \\(3,\\)"), (dict(q_pos0=_i32(4)), "q_pos0 \\(4,\\)"),
    (dict(kv_len=_i32(3).long()), "kv_len is torch.int64"), (dict(q_start=torch.zeros(4)), "q_start is torch.float32"), (dict(block_table=_i32(2, 4)), "block tables"),
    (dict(qkv=torch.zeros(5, 8, 8)), "qkv \\(5, 8, 8\\)"), (dict(keys=torch.zeros(9, KV_HEADS, PAGE * DIM)), "keys torch.float32 \\(9, 2, 128\\)"),
    (dict(num_heads=3), "3 heads over 2 kv heads"), (dict(num_kv_heads=0), "4 heads over 0 kv heads"), (dict(), "is not on a CUDA device")]


@pytest.mark.parametrize("arguments,message", STEP_REFUSALS + [
    (dict(mass=torch.zeros(9, KV_HEADS, PAGE, dtype=torch.bfloat16)), "mass torch.bfloat16"), (dict(mass=torch.zeros(9, KV_HEADS, 8)), "mass torch.float32 \\(9, 2, 8\\)"),
    (dict(scale=-0.5), "scaled by -0.5"), (dict(scale=float("nan")), "scaled by nan"), (dict(keep_first=-1), "-1 first keys"), (dict(max_kv_len=65), "65 keys"), (dict(slots=_i32(4)), "slots \\(4,\\) for 5 tokens"), (dict(slots=_i32(5).long()), "slots is torch.int64")])
def test_mass_refuses(arguments, message):
    a = dict(mass=torch.zeros(9, KV_HEADS, PAGE), num_heads=HEADS, num_kv_heads=KV_HEADS, head_dim=DIM, page_size=PAGE, max_q_len=3, max_kv_len=64, scale=1.0)
    a.update(_attention(**arguments))
    a.update({k: v for k, v in arguments.items()})
    with pytest.raises(ops.KernelError, match=message):
        ops.paged_attention_mass(**a)


@pytest.mark.parametrize("arguments,message", STEP_REFUSALS + [
    (dict(prefix_len=_i32(2)), "prefix_len \\(2,\\)"), (dict(prefix_len=_i32(3).long()), "prefix_len is torch.int64"), (dict(group_start=_i32(1)), "group_start \\(1,\\)"),
    (dict(group_start=_i32(5)), "group_start \\(5,\\)"), (dict(group_start=torch.zeros(3)), "group_start is torch.float32"), (dict(max_prefix_len=-1), "-1 shared"),
    (dict(scale=-0.5), "scaled by -0.5"), (dict(scale=float("nan")), "scaled by nan"), (dict(max_own_len=-1), "-1 own keys"), (dict(max_prefix_len=65), "65 shared"), (dict(max_q_len=4), "up to 4 tokens in groups of up to 3")])
def test_prefix_refuses(arguments, message):
    a = dict(prefix_len=_i32(3), group_start=_i32(3), num_heads=HEADS, num_kv_heads=KV_HEADS, head_dim=DIM, page_size=PAGE, max_q_len=2, max_prefix_len=20, max_own_len=30,
             max_group_tokens=3, scale=1.0)
    a.update(_attention(**arguments))
    a.update({k: v for k, v in arguments.items()})
    with pytest.raises(ops.KernelError, match=message):
        ops.paged_attention_prefix(**a)


def test_a_shortened_sequence_gives_back_the_blocks_behind_its_tokens():
    from paged_attention_engine_b200.cache.allocator import HOLE, BlockAllocator

    pool = BlockAllocator(10, 4)
    for name, count in (("a", 18), ("b", 9)):
        pool.create_sequence(name)
        assert pool.append_tokens(name, count).ok
    table = pool.block_table("a")
    assert pool.shorten_sequence("a", 9) == table[3:] and pool.block_table("a") == table[:3] and pool.num_tokens("a") == 9
    assert pool.free_block_ids()[-2:] == table[3:] and pool.num_allocated == 6
    assert pool.shorten_sequence("a", 9) == () and pool.append_tokens("a", 3).new_block_ids == ()
    assert pool.append_tokens("a", 1).new_block_ids == (8,)
    with pytest.raises(ValueError, match="13 tokens, it cannot be shortened to 14"):
        pool.shorten_sequence("a", 14)
    with pytest.raises(ValueError, match="-1"):
        pool.shorten_sequence("a", -1)
    with pytest.raises(KeyError):
        pool.shorten_sequence("c", 0)
    assert pool.shorten_sequence("a", 0) == (*table[:3], 8) and pool.block_table("a") == ()
    # Behind a window's holes.
    assert pool.append_tokens("a", 16).ok
    freed = pool.release_before("a", 9)
    held = pool.block_table("a")
    assert len(freed) == 2 and held[:2] == (HOLE, HOLE) and pool.num_held("a") == 2
    assert pool.shorten_sequence("a", 5) == held[2:] and pool.num_held("a") == 0
    everything = pool.num_free
    assert pool.free_sequence("a") == () and pool.num_free == everything and len(set(pool.free_block_ids())) == everything == 7
