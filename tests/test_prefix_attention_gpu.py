"""Attention of requests that share a prefix (csrc/attention_prefix.cu) against the definition in 64 bits, in which every request reads its own
whole context."""

import pytest
import torch

from cache_operators import Step, output_tolerance

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture(scope="module")
def ops():
    from paged_attention_engine_b200.kernels import ops as kernel_ops

    least, kernel_ops.PREFIX_SIMT_MIN_KEYS = kernel_ops.PREFIX_SIMT_MIN_KEYS, 1        # every case by the kernel that shares
    yield kernel_ops
    kernel_ops.PREFIX_SIMT_MIN_KEYS = least


def _limits(step):
    groups = zip(step.group_start, step.group_start[1:])
    return (max(step.tokens), max(step.prefix), max(n - p for n, p in zip(step.lengths, step.prefix)), max(sum(step.tokens[a:b]) for a, b in groups))


def _run(ops, step, **more):
    pools, tables = step.on()
    out = ops.paged_attention_prefix(*pools, *tables, step.prefix_len.cuda(), step.groups.cuda(), *step.sizes, *_limits(step), step.scale, **more)
    torch.cuda.synchronize()
    ops.check_device_errors()
    return out


def _check(step, out):
    want = step.attention()
    assert torch.isfinite(out).all()
    assert (out.cpu().double() - want).abs().max() <= output_tolerance(step.dtype, want)


def _step(shared, own, tokens, heads, kv_heads, dim, page, dtype, seed, **more):
    """`shared` = (requests, keys) per group; own[b] keys of request b behind them, the last tokens[b] of which are the step's."""
    prefix = [n for count, n in shared for _ in range(count)]
    return Step([p + o for p, o in zip(prefix, own)], tokens, heads, kv_heads, dim, page, dtype, seed, shared=shared, **more)


SIZES = [(12, 2, 128, 16, BF16), (28, 4, 128, 32, BF16), (14, 2, 64, 64, BF16), (8, 8, 64, 128, BF16), (40, 2, 128, 16, BF16), (3, 1, 32, 16, BF16), (12, 2, 64, 48, BF16),
         (4, 2, 64, 16, F32), (6, 3, 48, 7, F32), (40, 2, 128, 16, F32)]


@pytest.mark.parametrize("heads,kv_heads,dim,page,dtype", SIZES)
@pytest.mark.parametrize("shared,own,tokens", [
    (((2, 1),), [1, 1], [1, 1]),                                                   # one shared key, one own
    (((3, 64),), [1, 40, 17], [1, 1, 1]),
    (((4, 500),), [3, 90, 16, 1], [1] * 4),
    (((2, 63), (1, 129), (3, 0), (1, 200)), [5, 1, 30, 20, 1, 16, 64], [1] * 7),      # groups of one request, and one that shares nothing
    (((3, 333),), [70, 9, 40], [5, 1, 40]),                                        # several tokens a request
    (((2, 1000), (2, 100)), [63, 30, 2, 200], [63, 2, 2, 1]),
])
def test_groups(ops, heads, kv_heads, dim, page, dtype, shared, own, tokens):
    step = _step(shared, own, tokens, heads, kv_heads, dim, page, dtype, heads + len(own))
    info = {}
    out = _run(ops, step, info=info)
    takes = "shared" if dtype == BF16 and dim in (64, 128) and page != 48 else "shared simt" if dtype == F32 else "mma"
    assert info["kernel"] == takes
    _check(step, out)


def test_requests_without_tokens_and_groups_without_requests(ops):
    step = _step(((3, 70), (2, 200)), [20, 9, 4, 33, 50], [1, 0, 2, 0, 1], 12, 2, 128, 16, BF16, 4)
    _check(step, _run(ops, step))
    step.groups = torch.tensor([0, 3, 3, 5], dtype=torch.int32)
    _check(step, _run(ops, step))


@pytest.mark.parametrize("requests,prefix,tokens", [(70, 900, 1), (300, 130, 1), (24, 4000, 5), (2, 9000, 1)])
@pytest.mark.parametrize("heads,kv_heads,dim", [(28, 4, 128), (40, 8, 128), (14, 2, 64)])
def test_many_rows_and_many_keys(ops, requests, prefix, tokens, heads, kv_heads, dim):
    own = [tokens + 53 * b % 200 for b in range(requests)]
    step = _step(((requests, prefix),), own, [tokens] * requests, heads, kv_heads, dim, 16, BF16, requests)
    _check(step, _run(ops, step))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("requests", [4, 200])
def test_maxima_that_grow_along_the_shared_keys(ops, dim, requests):
    """References that move: keys that point ever further along the queries."""
    step = _step(((requests, 1500),), [10] * requests, [1] * requests, 12, 2, dim, 16, BF16, 3)
    along = torch.nn.functional.normalize(torch.randn(dim), dim=0)
    step.qkv += (2 * along).repeat(16).to(BF16)
    j = torch.arange(1500)
    p, o = step.table[0].long()[j // 16], j % 16
    grown = step.keys[p, :, o].float() + torch.linspace(0, 60, 1500)[:, None, None] * along
    step.keys[p, :, o] = grown.to(BF16)
    for b in range(1, requests):                               # the page that the border cuts
        cut = torch.arange(1488, 1500)
        step.keys[step.table[b].long()[cut // 16], :, cut % 16] = step.keys[step.table[0].long()[cut // 16], :, cut % 16]
    _check(step, _run(ops, step))


def test_a_long_portion_and_a_lone_request_read_their_keys_themselves(ops):
    step = _step(((2, 100),), [70, 5], [65, 1], 12, 2, 128, 16, BF16, 6)
    info = {}
    _check(step, _run(ops, step, info=info))
    assert info["kernel"] != "shared"
    step = _step(((1, 100),), [5], [1], 12, 2, 128, 16, BF16, 6)
    _check(step, _run(ops, step, info=info))
    assert info["kernel"] != "shared"


def test_equal_bits_in_every_run(ops):
    step = _step(((40, 700),), [1 + b for b in range(40)], [1] * 40, 28, 4, 128, 16, BF16, 8)
    first = _run(ops, step)
    assert all(torch.equal(first, _run(ops, step)) for _ in range(5))


def test_captured_and_replayed_with_other_lengths(ops):
    page = 16
    steps = [_step(shared, own, [1] * 6, 12, 2, 128, page, BF16, 20 + i, width=50)
             for i, (shared, own) in enumerate((([(4, 600), (2, 90)], [40, 1, 77, 16, 150, 3]), ([(4, 17), (2, 640)], [1, 150, 2, 99, 20, 66])))]
    fixed, sources = None, []
    for s in steps:
        pools, tables = s.on()
        sources.append([*pools, *tables, s.prefix_len.cuda(), s.groups.cuda()])
    pages = max(s[1].shape[0] for s in sources)
    fixed = [torch.zeros((pages, *a.shape[1:]), dtype=a.dtype, device="cuda") if i in (1, 2) else a.clone() for i, a in enumerate(sources[0])]
    args = (*steps[0].sizes, 1, 650, 160, 4, steps[0].scale)

    def fill(source):
        for to, a in zip(fixed, source):
            to[: a.shape[0]].copy_(a)

    fill(sources[0])
    ops.paged_attention_prefix(*fixed, *args)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.paged_attention_prefix(*fixed, *args)
    for step, source in zip(steps[::-1], sources[::-1]):
        fill(source)
        graph.replay()
        torch.cuda.synchronize()
        _check(step, out)
    ops.check_device_errors()


def test_two_streams_at_once(ops):
    """Calls on two streams have scratch of their own."""
    steps = [_step(((30, 2000),), [20] * 30, [1] * 30, 28, 4, 128, 16, BF16, 30 + i) for i in range(2)]
    wants = [_run(ops, s) for s in steps]
    given = [(s.on(), s.prefix_len.cuda(), s.groups.cuda()) for s in steps]
    streams = [torch.cuda.Stream() for _ in steps]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(10):
        for i, s in enumerate(steps):
            with torch.cuda.stream(streams[i]):
                (pools, tables), prefix, groups = given[i]
                outs[i].append(ops.paged_attention_prefix(*pools, *tables, prefix, groups, *s.sizes, *_limits(s), s.scale))
    torch.cuda.synchronize()
    ops.check_device_errors()
    assert all(torch.equal(o, wants[i]) for i in range(2) for o in outs[i])


def test_a_step_without_tokens_and_operands_that_start_anywhere(ops):
    step = _step(((2, 40),), [3, 9], [1, 1], 12, 2, 128, 16, BF16, 6)
    pools, tables = step.on()
    none = ops.paged_attention_prefix(pools[0][:0], *pools[1:], *tables, step.prefix_len.cuda(), step.groups.cuda(), *step.sizes, *_limits(step), step.scale)
    assert none.shape == (0, 12 * 128)
    shifted = torch.empty(pools[1].numel() + 4, dtype=BF16, device="cuda")[4:].view_as(pools[1]).copy_(pools[1])
    with pytest.raises(ops.KernelError, match="16-byte boundary"):
        ops.paged_attention_prefix(pools[0], shifted, pools[2], *tables, step.prefix_len.cuda(), step.groups.cuda(), *step.sizes, *_limits(step), step.scale)
    mass = step.mass.cuda()
    with pytest.raises(ops.KernelError, match="16-byte boundary"):
        ops.paged_attention_mass(pools[0], pools[1], shifted, mass, *tables, *step.sizes, *step.longest, step.scale)
    assert ops.paged_attention_mass(pools[0][:0], *pools[1:], mass, *tables, *step.sizes, *step.longest, step.scale).shape == (0, 12 * 128)
    assert torch.equal(mass.cpu(), step.mass)
    with pytest.raises(ops.KernelError, match="values is not contiguous"):
        ops.paged_attention_mass(pools[0], pools[1], pools[2].transpose(0, 1).contiguous().transpose(0, 1), mass, *tables, *step.sizes, *step.longest, step.scale)


@pytest.mark.parametrize("dim,requests", [(64, 4), (64, 8), (128, 4)])
def test_own_keys_in_more_than_32_slices(ops, dim, requests):
    step = _step(((requests, 100),), [26000, 40, 300, 17, 16, 90, 5000, 64][:requests], [16] * requests, 20, 1, dim, 16, BF16, requests)
    _check(step, _run(ops, step))


@pytest.mark.parametrize("tokens", [16, 63, 64, 65])
def test_up_to_64_tokens_a_request_share(ops, tokens):
    step = _step(((3, 500), (2, 90)), [tokens + 9, 150, tokens, 130, 77], [tokens, 1, 5, tokens, 64], 12, 2, 128, 16, BF16, tokens)
    info = {}
    out = _run(ops, step, info=info)
    assert info["kernel"] == ("shared" if max(step.tokens) <= 64 else "tcgen05")
    _check(step, out)


@pytest.mark.parametrize("heads,kv_heads,dim,page,dtype", [(12, 2, 64, 16, F32), (8, 2, 256, 16, F32), (5, 1, 20, 16, BF16), (3, 3, 4, 5, F32), (20, 1, 100, 48, BF16)])
def test_many_keys_on_cuda_cores(ops, heads, kv_heads, dim, page, dtype):
    step = _step(((9, 1500), (3, 2100)), [1 + 37 * b % 150 for b in range(12)], [1] * 12, heads, kv_heads, dim, page, dtype, dim)
    info = {}
    out = _run(ops, step, info=info)
    assert info["kernel"] == "shared simt"
    _check(step, out)
    ops.PREFIX_SIMT_MIN_KEYS = 1 << 30
    try:
        if dim % 8:                            # no attention of a request by itself takes it
            with pytest.raises(ops.KernelError, match="not a multiple of 8"):
                _run(ops, step)
        else:
            _run(ops, step, info=info)
            assert info["kernel"] == "simt"
    finally:
        ops.PREFIX_SIMT_MIN_KEYS = 1
