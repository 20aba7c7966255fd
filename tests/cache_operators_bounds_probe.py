"""Run with PAE_BOUNDS=1 (tests/test_cache_operators_bounds_gpu.py does): the operators of the shared and pruned cache on the checked build, as
tests/bounds_probe.py has the engine: steps that are in range leave the error word at 0; a page id beyond the pool and a table that is too narrow are
named by it, and the access is not made. The pool that the kernels are told about is the first half of a larger tensor."""

import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent
for extra in (ROOT, ROOT / "tests"):
    sys.path.insert(0, str(extra))

import torch

from cache_operators import Step, i32, output_tolerance
from paged_attention_engine_b200.kernels import build, ops


def limits(step):
    groups = zip(step.group_start, step.group_start[1:])
    return max(step.tokens), max(step.prefix), max(n - p for n, p in zip(step.lengths, step.prefix)), max(sum(step.tokens[a:b]) for a, b in groups)


def in_range() -> None:
    for dtype, dim, page in ((torch.bfloat16, 128, 16), (torch.bfloat16, 64, 128), (torch.float32, 64, 16), (torch.bfloat16, 48, 8)):
        for tokens in ([1] * 5, [1, 70, 1, 130, 2], [3] * 5):
            step = Step([70, 170, 65, 400, 90], tokens, 12, 2, dim, page, dtype, dim + sum(tokens), shared=((5, 20),) if max(tokens) < 60 else ())
            pools, tables = step.on()
            mass = step.mass.cuda()
            want = step.attention()
            outs = [ops.paged_attention_mass(*pools, mass, *tables, *step.sizes, *step.longest, step.scale, keep_first=20)]
            outs.append(ops.paged_attention_prefix(*pools, *tables, step.prefix_len.cuda(), step.groups.cuda(), *step.sizes, *limits(step), step.scale))
            for out in outs:
                assert (out.cpu().double() - want).abs().max() <= output_tolerance(dtype, want)
            kept = ops.choose_kept(mass, tables[0], tables[3], 80, 20, 7, 400)
            ops.compact_kept(*pools[1:], mass, tables[0], tables[3], kept)
            ops.check_device_errors()
    print("steps in range leave no error", flush=True)


def caught(code: int) -> None:
    try:
        ops.check_device_errors()
    except ops.KernelError as exc:
        assert f"bounds code {code}" in str(exc), str(exc)
        return
    raise AssertionError(f"bounds code {code} was not raised")


def out_of_range() -> None:
    heads, kv_heads, d, page = 4, 2, 64, 16
    for dtype in (torch.bfloat16, torch.float32):
        whole = [torch.randn(8, kv_heads, page, d, device="cuda").to(dtype) for _ in range(2)] + [torch.rand(8, kv_heads, page, device="cuda")]
        keys, values, mass = (t[:4] for t in whole)
        beyond = [t[4:].clone() for t in whole]
        q_start, kv_len = i32([0, 1, 2], "cuda"), i32([20, 30], "cuda")
        qkv = torch.randn(2, (heads + 2 * kv_heads) * d, device="cuda").to(dtype)
        bad = i32([[1, 6], [0, 2]], "cuda")                                                  # page 6 of a pool of 4
        narrow = i32([1, 3, 0, 2, 0, 0, 0, 0], "cuda")[:4].view(2, 2)                        # two pages, and 40 keys need three; a page stands behind
        long_len = i32([20, 40], "cuda")
        for table, lengths, longest, code in ((bad, kv_len, 30, 103), (narrow, long_len, 32, 102)):
            step = (qkv, keys, values), (table, q_start, lengths - 1, lengths)
            ops.paged_attention_mass(*step[0], mass, *step[1], heads, kv_heads, d, page, 1, longest, 0.125)
            torch.cuda.synchronize()
            caught(code)
            ops.paged_attention_prefix(*step[0], *step[1], i32([16, 16], "cuda"), i32([0, 2], "cuda"), heads, kv_heads, d, page, 1, 16, 24, 2, 0.125)
            torch.cuda.synchronize()
            caught(code)
        kept = ops.choose_kept(mass, bad, kv_len, 18, 1, 1, 30)
        torch.cuda.synchronize()
        caught(103)
        kept.copy_(torch.arange(2, 20, dtype=torch.int32, device="cuda"))
        ops.compact_kept(keys, values, mass, bad, kv_len, kept)
        torch.cuda.synchronize()
        caught(103)
        assert all(torch.equal(t[4:], b) for t, b in zip(whole, beyond)), "an access beyond the pool was made"
    print("indices out of range were caught and skipped", flush=True)


if __name__ == "__main__":
    assert build.BOUNDS and ops.bounds_checked, "run with PAE_BOUNDS=1"
    in_range()
    out_of_range()
    print("CACHE OPERATORS BOUNDS PROBE OK")
