"""Calls of the paged attentions that a server may make beside the plain ones:
two at once, graphs replayed in turn, lengths outside their ranges, a page that is
held twice."""
import pytest
import torch

from paged_helpers import SENTINEL, ints
from test_gpu_paged_attention import Call

pytestmark = pytest.mark.gpu


def two_calls(torch_cuda):
    a = Call(torch_cuda, 31, "f32", 8, 1, 256, 16, [100, 3, 1], [200, 0, 900])
    b = Call(torch_cuda, 32, "f16", 8, 2, 128, 32, [1, 1, 70], [500, 3, 64])
    a.draw_masks(33, words=2)
    b.draw_masks(34, words=2)
    return a, b


def test_two_streams_at_once(torch_cuda):
    """Each with its workspace: the bits of calls one after another."""
    calls = two_calls(torch_cuda)
    expected = [(c.causal(), c.tree()) for c in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    outs = [[(c.fresh_out(), c.fresh_out()) for _ in range(6)] for c in calls]
    torch.cuda.synchronize()
    for i in range(6):
        for c, stream, out in zip(calls, streams, outs):
            c.causal(out[i][0], stream.cuda_stream)
            c.tree(out[i][1], stream=stream.cuda_stream)
    torch.cuda.synchronize()
    for want, out in zip(expected, outs):
        for causal, tree in out:
            assert torch.equal(causal, want[0]) and torch.equal(tree, want[1])


def test_two_graphs_in_turn(torch_cuda):
    calls = two_calls(torch_cuda)
    graphs, outs = [], []
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    for c in calls:
        out = c.fresh_out(), c.fresh_out()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            c.causal(out[0], torch.cuda.current_stream().cuda_stream)
            c.tree(out[1], stream=torch.cuda.current_stream().cuda_stream)
        graphs.append(graph)
        outs.append(out)
    for turn in range(3):
        for c, out in zip(calls, outs):
            c.q.copy_(torch.randn_like(c.q))
            out[0].fill_(SENTINEL)
            out[1].fill_(SENTINEL)
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for c, out in zip(calls, outs):
            assert torch.equal(out[0], c.causal()) and torch.equal(out[1], c.tree()), turn


@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_lengths_outside_their_ranges(torch_cuda, name):
    """Cached rows are taken as 0 up to what the table holds, rows as those of the
    packed tensors."""
    call = Call(torch_cuda, 35, name, 4, 1, 128, 16, [5, 40, 1], [32, 7, 32], behind=3)
    call.draw_masks(36)

    def both(starts, cached):
        call.batch.starts.copy_(ints(starts))
        call.batch.cached.copy_(ints(cached))
        return call.causal(), call.tree()

    within = both([0, 5, 45, 49], [32, 0, 32])
    outside = both([-4, 5, 45, 1 << 30], [1 << 30, -9, 33])
    for a, b in zip(within, outside):
        assert torch.equal(a, b)
        assert (a != SENTINEL).any(1).all()


@pytest.mark.parametrize("name", ["f32", "f16"])
def test_a_page_held_twice(torch_cuda, name):
    """By two sequences, and twice by one."""
    call = Call(torch_cuda, 37, name, 8, 1, 256, 16, [3, 20], [48, 40])
    call.draw_masks(38)
    table = call.table.cpu()
    table[0, 2] = table[0, 0]
    table[1, 0] = table[0, 1]
    call.table.copy_(table)
    for side in range(2):
        call.held[0][side][32:48] = call.held[0][side][0:16]
        call.held[1][side][0:16] = call.held[0][side][16:32]
    call.check(call.causal(), "causal", "causal")
    call.check(call.tree(), "tree", "tree")
