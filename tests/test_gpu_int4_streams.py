"""The operators over a cache in 4 bits with several calls in flight: on
streams of their own, beside a graph's replays, and in graphs whose items are
split; and calls of more tokens, heads or slots than one scan, grid or
workgroup takes.

References: the same calls one at a time (equal bits), and 64 bits with the
tolerances of test_gpu_int4.py."""
import pytest
import torch

from libortho_amd import _C_ops
from test_gpu_int4 import attend_case, attend_check, check_read, i32, random_cache

pytestmark = pytest.mark.gpu


def attend(args, **kw):
    q, cache, table, pos = args
    return lambda: _C_ops.paged_attention_int4(q, *cache, table, pos, **kw)


def prompts(lens, new, *args):
    q, cache, table, pos = attend_case(lens, *args, new=new)
    return attend((q, cache, table, pos), rows=i32([r for r in range(len(lens)) for _ in range(new)]))


def calls():
    """Calls that split their items and join them in the launch and in a second one."""
    return [attend(attend_case([9000, 17, 4000], 8, 2, 128, 64, 16, torch.bfloat16)),
            attend(attend_case([1, 30000, 300], 4, 1, 64, 32, 32, torch.float16)),
            attend(attend_case([700] * 9, 4, 4, 80, 80, 16, torch.float16)),
            prompts([900, 20, 3000], 17, 8, 2, 128, 128, 16, torch.bfloat16),
            attend(attend_case([40] * 70 + [25000] + [3] * 20, 8, 4, 64, 64, 13, torch.bfloat16), window=900),
            attend(attend_case([5000, 1], 16, 1, 256, 128, 16, torch.float16))]


def test_calls_in_flight_on_three_streams(gpu):
    todo = calls()
    want = [f() for f in todo]
    torch.cuda.synchronize()
    streams = [torch.cuda.current_stream(), torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[] for _ in streams]
    for again in range(3):
        for i in range(len(todo)):
            for s, stream in enumerate(streams):  # each stream begins at another call
                with torch.cuda.stream(stream):
                    n = (i + 2 * s) % len(todo)
                    got[s].append((n, todo[n]()))
    torch.cuda.synchronize()
    for s, outs in enumerate(got):
        for n, out in outs:
            assert torch.equal(out, want[n]), (s, n)


def test_eager_calls_beside_a_graphs_replays(gpu):
    todo = calls()
    want = [f() for f in todo]
    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        for f in todo:
            f()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=warm):
        captured = [f() for f in todo]
    other = torch.cuda.Stream()
    for again in range(4):
        for t in captured:
            t.fill_(7)
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(other):
            beside = [f() for f in todo]
        behind = [f() for f in todo]
        torch.cuda.synchronize()
        for outs in (captured, beside, behind):
            for n, out in enumerate(outs):
                assert torch.equal(out, want[n]), (again, n)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_captured_attention_of_split_items(gpu, dtype):
    # one long request among short ones, another one each time; items of up to
    # 17 pieces and of more
    q, cache, table, pos = attend_case([25000] + [3000] * 3 + [40] * 8, 8, 2, 128, 64, 16, dtype)
    table = table[0].repeat(12, 1)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        _C_ops.paged_attention_int4(q, *cache, table, pos)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _C_ops.paged_attention_int4(q, *cache, table, pos)
        second = _C_ops.paged_attention_int4(out, *cache, table, pos)
    for i in range(5):
        pos.copy_(i32([[24999, 2999, 2999, 2999] + [39] * 8, [-1] * 11 + [20000], [5000] * 12, [0] * 12,
                       [100, 24000, 7, 1500, 0, 0, 900, 3, 64, 31, 32, 33]][i]))
        q.copy_(torch.randn(q.shape, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        got, again = out.clone(), second.clone()
        assert torch.equal(got, attend_check(q, cache, table, pos)), i
        assert torch.equal(again, _C_ops.paged_attention_int4(got, *cache, table, pos)), i


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("H,G,D,group,P", [(4, 2, 128, 64, 16), (6, 1, 64, 64, 8), (2, 2, 80, 80, 5)])
def test_split_items_behind_many_tokens(gpu, H, G, D, group, P, dtype):
    # more tokens than one scan takes (128), long requests in each block of them
    lens = [(37 * r) % 60 for r in range(330)]
    lens[5], lens[127], lens[128], lens[200], lens[329] = 3000, 9000, 5000, 700, 2500
    attend_check(*attend_case(lens, H, G, D, group, P, dtype))


def test_prompts_single_tokens_and_places_without_a_token(gpu):
    # a prompt of 300 tokens behind 200 cached ones, a draft of 5, a single
    # token, a whole prompt, and places that no token took, in one call
    q, cache, table, _ = attend_case([500, 90, 1000, 160], 8, 2, 128, 64, 16, torch.bfloat16)
    rows = [0] * 300 + [1] * 5 + [2] + [3] * 160 + [-1] * 9
    pos = list(range(200, 500)) + list(range(85, 90)) + [999] + list(range(160)) + [-1] * 9
    q = torch.randn(len(rows), 8, 128, device="cuda").bfloat16()
    got = attend_check(q, cache, table, i32(pos), rows=i32(rows))
    assert not bool(got[-9:].any())
    attend_check(q, cache, table, i32(pos), rows=i32(rows), window=130)


def test_append_of_more_heads_than_a_grid_has_rows(gpu):
    # vectors of 256: eight heads a workgroup, 65,535 workgroups along the heads
    H, D = 8 * 65535 + 21, 256
    q = torch.randn(1, H, D, device="cuda").half()
    cache = _C_ops.int4_cache(1, 1, 1, D)
    k = torch.randn(1, 1, D, device="cuda").half()
    cs = torch.ones(1, D, device="cuda")
    cs[:, D // 2:] = 0
    slots = torch.zeros(1, dtype=torch.int64, device="cuda")
    out = _C_ops.cache_append_int4(k, k, *cache, slots, q=q, positions=i32([0]), cos_sin=cs)
    assert torch.equal(out, q)
    want = _C_ops.int4_cache(1, 1, 1, D)
    _C_ops.cache_append_int4(k, k, *want, slots)
    assert all(torch.equal(a, b) for a, b in zip(cache, want))


def test_append_of_more_tokens_than_one_grid_holds(gpu):
    T, D, P, pages = (1 << 23) + 77, 8, 16, 8
    k = torch.zeros(T, 1, D, dtype=torch.float16, device="cuda")
    slots = torch.full((T,), -1, dtype=torch.int64, device="cuda")
    at = [0, 5, (1 << 22) - 1, 1 << 22, (1 << 23) - 1, 1 << 23, (1 << 23) + 9, T - 1]
    for i, t in enumerate(at):
        k[t], slots[t] = i + 1, 7 * i + 3
    pos = torch.zeros(T, dtype=torch.int32, device="cuda")
    pos[1 << 23] = 1
    q = torch.ones(T, 1, D, dtype=torch.float16, device="cuda")
    cs = torch.tensor([[1.0] * 4 + [0.0] * 4, [0.0] * 4 + [1.0] * 4], device="cuda")  # none, and a quarter turn
    cache = _C_ops.int4_cache(pages, P, 1, D)
    out = _C_ops.cache_append_int4(k, -k, *cache, slots, q=q, positions=pos, cos_sin=cs)
    K, V = _C_ops.cache_read_int4(*cache, torch.arange(pages * P, device="cuda"), D)
    want = torch.zeros_like(K)
    for i in range(len(at)):
        want[7 * i + 3] = i + 1
    assert torch.equal(V, -want)
    want[7 * at.index(1 << 23) + 3, 0, :4] *= -1
    # (the turned one, -6 and 6: 15 steps, each off by half a last place of 0.8, 2^-12, and rounded by 2^-9)
    assert float((K - want).abs().max()) <= 15 * 2.0 ** -12 + 2.0 ** -9
    others = torch.ones(pages * P, dtype=torch.bool, device="cuda")
    others[7 * at.index(1 << 23) + 3] = False
    assert torch.equal(K[others], want[others])
    q[1 << 23, 0, :4] = -1
    assert torch.equal(out, q)


@pytest.mark.parametrize("G,D,group", [(1, 8, 8), (1, 64, 32), (3, 80, 80), (8, 128, 64), (40, 256, 32), (5, 160, 160)])
def test_read_of_slots_that_share_workgroups(gpu, G, D, group):
    # as many slots as make every workgroup take several, one after another
    g = torch.Generator(device="cuda").manual_seed(D)
    cache = random_cache(g, 12, 7, G, D, group)
    each = check_read(cache, torch.arange(84, device="cuda"), D, torch.float16)
    n = max(30000, 40000000 // (G * 2 * D))
    slots = torch.randint(-3, 84, (n,), generator=g, device="cuda")
    k, v = _C_ops.cache_read_int4(*cache, slots, D)
    for got, few in zip((k, v), each):
        assert torch.equal(got, torch.where((slots >= 0)[:, None, None], few[slots.clamp(min=0)], torch.zeros_like(few[:1])))
