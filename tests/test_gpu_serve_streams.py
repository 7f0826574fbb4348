"""The serving operators with several calls in flight: on streams of their
own, beside a graph's replays, and in graphs whose items are split; and
attention whose share search takes several blocks of tokens.

References: the same calls one at a time (equal bits), and 64 bits with the
tolerances of test_gpu_paged.py."""
import pytest
import torch

from libortho_amd import _C_ops
from test_gpu_adapter import case as adapter_case
from test_gpu_paged import attend_case, attend_check, i32

pytestmark = pytest.mark.gpu


def attend(args, window=0):
    return lambda: _C_ops.paged_attention(*args, window=window)


def adapt(args):
    return lambda: _C_ops.adapter_add(*args)


def calls():
    """Calls that split their items, join them in the launch and in a second
    one, and leave partials for a second launch."""
    return [attend(attend_case([9000, 17, 4000], 8, 2, 128, 16, torch.bfloat16)),
            adapt(adapter_case(600, 1000, 200, 64, 1, torch.float16)),
            attend(attend_case([1, 30000, 300], 4, 1, 64, 32, torch.float16)),
            adapt(adapter_case(48, 4096, 1024, 32, 10, torch.bfloat16)),
            attend(attend_case([700] * 9, 4, 4, 80, 16, torch.float16)),
            adapt(adapter_case(300, 2048, 512, 24, 2, torch.float16)),
            attend(attend_case([40] * 70 + [25000] + [3] * 20, 8, 4, 64, 16, torch.bfloat16), window=900)]


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
    q, kc, vc, table, pos = attend_case([25000] + [3000] * 3 + [40] * 8, 8, 2, 128, 16, dtype)
    table = table[0].repeat(12, 1)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        _C_ops.paged_attention(q, kc, vc, table, pos)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _C_ops.paged_attention(q, kc, vc, table, pos)
        second = _C_ops.paged_attention(out, kc, vc, table, pos)
    for i in range(5):
        pos.copy_(i32([[24999, 2999, 2999, 2999] + [39] * 8, [-1] * 11 + [20000], [5000] * 12, [0] * 12,
                       [100, 24000, 7, 1500, 0, 0, 900, 3, 64, 31, 32, 33]][i]))
        q.copy_(torch.randn(q.shape, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        got, again = out.clone(), second.clone()
        assert torch.equal(got, attend_check(q, kc, vc, table, pos)), i
        assert torch.equal(again, _C_ops.paged_attention(got, kc, vc, table, pos)), i


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("H,G,D,P", [(4, 2, 128, 16), (6, 1, 64, 8), (2, 2, 80, 5)])
def test_split_items_behind_many_tokens(gpu, H, G, D, P, dtype):
    # more tokens than one scan takes (128), long requests in each block of them
    lens = [(37 * r) % 60 for r in range(330)]
    lens[5], lens[127], lens[128], lens[200], lens[329] = 3000, 9000, 5000, 700, 2500
    attend_check(*attend_case(lens, H, G, D, P, dtype))


def test_prompts_through_attention(gpu):
    # a prompt of 300 tokens behind 200 cached ones, a draft of 5, single
    # tokens and a whole prompt in one call
    q, kc, vc, table, _ = attend_case([500, 90, 1000, 160], 8, 2, 128, 16, torch.bfloat16)
    rows = [0] * 300 + [1] * 5 + [2] + [3] * 160
    pos = list(range(200, 500)) + list(range(85, 90)) + [999] + list(range(160))
    q = torch.randn(len(rows), 8, 128, device="cuda").bfloat16()
    attend_check(q, kc, vc, table, i32(pos), rows=i32(rows))
    attend_check(q, kc, vc, table, i32(pos), rows=i32(rows), window=130)
