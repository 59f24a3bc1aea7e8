"""Bounds of a page's keys and the pages chosen by them, against plain indexing and
64-bit scores: the choice is the same page for page."""
import math

import numpy as np
import pytest
import torch

from huggingfaceeacp_amd import gemma_q8 as G
from paged_helpers import KIND, SENTINEL, TYPES, Batch, Cache, ints, kv_type, normal

pytestmark = pytest.mark.gpu


def page_bounds(cache, layer, batch, bounds, taken=None, stream=0):
    G.page_bounds(cache.c, layer, batch.c, bounds.c, taken.data_ptr() if taken is not None else None, stream)


def random_table(g, count, width, pages):
    return torch.randperm(pages, generator=g)[:count * width].reshape(count, width).to(torch.int32)


@pytest.mark.parametrize("name", ["f16", "bf16"])
@pytest.mark.parametrize("kv_heads,head_dim,page_rows", [(1, 256, 16), (3, 8, 1), (4, 80, 64), (2, 64, 4),
                                                         (8, 128, 256)])
def test_bounds(torch_cuda, name, kv_heads, head_dim, page_rows):
    g = torch.Generator().manual_seed(1)
    rows, cached = [5, 0, 70, 1, 9, 300], [0, 3, 30, 64, 15, 7]
    width = max(-(-(n + c) // page_rows) for n, c in zip(rows, cached))
    pages = width * len(rows) + 3
    host_table = random_table(g, len(rows), width, pages)
    host_table[3] = -1
    host_table[4, 0] = pages
    table = host_table.cuda()
    cache = Cache(TYPES[name], 2, pages, page_rows, kv_heads, head_dim)
    cache.keys[1].copy_(torch.randn(cache.keys[1].shape, generator=g))
    batch = Batch(rows, cached, table, before=2, behind=3)
    counts = torch.tensor([3, 7, 70, 0, -2, 280], dtype=torch.int32)
    for taken in (None, counts):
        bounds = Cache(TYPES[name], 2, pages, 1, kv_heads, head_dim)
        bounds.keys.fill_(SENTINEL)
        bounds.values.fill_(SENTINEL)
        keys = cache.keys.cpu()
        expected = [torch.full(bounds.keys.shape, SENTINEL, dtype=TYPES[name]) for _ in range(2)]
        for s, n in enumerate(rows):
            n = n if taken is None else min(n, int(taken[s]))
            if n <= 0:
                continue
            for slot in range(cached[s] // page_rows, (cached[s] + n - 1) // page_rows + 1):
                page = int(host_table[s, slot])
                if 0 <= page < pages:
                    held = min(page_rows, cached[s] + n - slot * page_rows)
                    expected[0][1, page, 0] = keys[1, page, :held].amin(0)
                    expected[1][1, page, 0] = keys[1, page, :held].amax(0)
        page_bounds(cache, 1, batch, bounds, taken.cuda() if taken is not None else None)
        torch.cuda.synchronize()
        assert torch.equal(bounds.keys.cpu(), expected[0]) and torch.equal(bounds.values.cpu(), expected[1])


def test_bounds_of_many_rows_and_sequences(torch_cuda):
    """More rows than blocks, and more sequences than lanes with a row each."""
    g = torch.Generator().manual_seed(2)
    for rows, cached, page_rows in (([9000], [5], 8), ([1] * 150, [s % 40 for s in range(150)], 16)):
        width = max(-(-(n + c) // page_rows) for n, c in zip(rows, cached))
        pages = width * len(rows)
        host_table = random_table(g, len(rows), width, pages)
        table = host_table.cuda()
        cache = Cache(torch.float16, 1, pages, page_rows, 1, 32)
        cache.keys.copy_(torch.randn(cache.keys.shape, generator=g))
        bounds = Cache(torch.float16, 1, pages, 1, 1, 32)
        page_bounds(cache, 0, Batch(rows, cached, table), bounds)
        keys, least = cache.keys.cpu(), bounds.keys.cpu()
        for s, (n, c) in enumerate(zip(rows, cached)):
            for slot in range(width):
                page = int(host_table[s, slot])
                held = min(page_rows, c + n - slot * page_rows)
                if slot * page_rows + page_rows <= c or held <= 0:
                    assert torch.isnan(least[0, page]).all()
                else:
                    assert torch.equal(least[0, page, 0], keys[0, page, :held].amin(0))


@pytest.mark.parametrize("name", ["f16", "bf16"])
def test_bounds_of_keys_that_are_not_finite(torch_cuda, name):
    cache = Cache(TYPES[name], 1, 2, 64, 1, 256)
    cache.keys.copy_(torch.randn(cache.keys.shape, generator=torch.Generator().manual_seed(3)))
    for row, channel, value in ((40, 3, math.nan), (0, 5, math.nan), (63, 7, math.nan), (9, 100, math.inf),
                                (10, 101, -math.inf)):
        cache.keys[0, 1, row, 0, channel] = value
    bounds = Cache(TYPES[name], 1, 2, 1, 1, 256)
    page_bounds(cache, 0, Batch([64], [0], ints([[1]])), bounds)
    keys = cache.keys[0, 1, :, 0].float().cpu()
    least, largest = bounds.keys[0, 1, 0, 0].float().cpu(), bounds.values[0, 1, 0, 0].float().cpu()
    odd = torch.isnan(keys).any(0)
    assert odd.sum() == 3 and torch.equal(torch.isnan(least), odd) and torch.equal(torch.isnan(largest), odd)
    assert torch.equal(least[~odd], keys.amin(0)[~odd]) and torch.equal(largest[~odd], keys.amax(0)[~odd])
    assert largest[100] == math.inf and least[101] == -math.inf


class Select:
    """A batch whose bounds are drawn, and a call."""

    def __init__(self, seed, name, q_name, heads, kv_heads, head_dim, page_rows, rows, cached, before=0,
                 behind=0, extra=0, spread=1.5):
        g = torch.Generator().manual_seed(seed)
        self.heads, self.kv_heads, self.d, self.page_rows = heads, kv_heads, head_dim, page_rows
        width = max(-(-(n + c) // page_rows) for n, c in zip(rows, cached))
        pages = width * len(rows) + 2
        self.host_table = random_table(g, len(rows), width, pages)
        self.table = self.host_table.cuda()
        self.batch = Batch(rows, cached, self.table, before, behind)
        a, b = (normal(g, (2, pages, 1, kv_heads, head_dim), kv_type(name)) for _ in range(2))
        self.least, self.largest = torch.minimum(a, b), torch.maximum(a, b)
        self.cache = Cache(kv_type(name), 2, pages, page_rows, kv_heads, head_dim)
        self.bounds = Cache(kv_type(name), 2, pages, 1, kv_heads, head_dim)
        self.upload()
        self.q_stride = heads * head_dim + extra
        self.q_host = normal(g, (self.batch.total, self.q_stride), TYPES[q_name], spread)
        self.q = self.q_host.cuda()

    def upload(self):
        self.bounds.keys.copy_(self.least)
        self.bounds.values.copy_(self.largest)

    def call(self, first, last, top, out=None, stream=0):
        out = torch.full((self.batch.total, self.kv_heads, top), 77, dtype=torch.int32,
                         device="cuda") if out is None else out
        size = G.page_select_workspace_bytes(self.batch.total, self.kv_heads, self.table.shape[1])
        self.workspace = torch.full((size,), 0xFF, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        G.page_select(self.cache.c, 1, self.batch.c, self.bounds.c, self.q.data_ptr(), KIND[self.q.dtype],
                      self.q_stride, self.heads, first, last, top, out.data_ptr(), self.workspace.data_ptr(),
                      size, stream)
        return out

    def expected(self, first, last, top):
        group, d = self.heads // self.kv_heads, self.d
        out = torch.full((self.batch.total, self.kv_heads, top), 77, dtype=torch.int32)
        pages = self.cache.keys.shape[1]
        for s, (a, b) in enumerate(self.batch.spans):
            for i in range(b - a):
                q = self.q_host[a + i, :self.heads * d].double().reshape(self.kv_heads, group, d)
                own = (self.batch.cached_host[s] + i) // self.page_rows
                slots = list(range(min(own + 1, self.table.shape[1])))
                at = [int(self.host_table[s, j]) for j in slots]
                there = torch.tensor([0 <= p < pages for p in at])
                used = torch.tensor([p if 0 <= p < pages else 0 for p in at])
                for g in range(self.kv_heads):
                    low, high = (x[1, used, 0, g].double()[:, None] for x in (self.least, self.largest))
                    term = torch.where(q[g] > 0, q[g] * high, q[g] * low)
                    score = term.sum(-1).amax(-1).float()
                    odd = ~torch.isfinite(low).all(-1)[:, 0] | ~torch.isfinite(high).all(-1)[:, 0]
                    score = torch.where(odd | torch.isnan(score), math.inf, score)
                    # (class, score) by falling order, the lower page first
                    ranked = sorted(slots, key=lambda j: (
                        0 if j < first or j > own - last else 1 if there[j] else 2,
                        -float(score[j]) if there[j] else 0.0, j))
                    chosen = sorted(ranked[:top])
                    out[a + i, g] = torch.tensor(chosen + [-1] * (top - len(chosen)), dtype=torch.int32)
        return out

    def check(self, first, last, top):
        got = self.call(first, last, top).cpu()
        assert torch.equal(got, self.expected(first, last, top)), (first, last, top)


@pytest.mark.parametrize("name,q_name", [("f16", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("heads,kv_heads,head_dim", [(8, 1, 256), (4, 4, 64), (6, 2, 128), (3, 1, 80), (14, 2, 96),
                                                     (2, 1, 8), (32, 1, 64), (20, 2, 24)])
def test_select(torch_cuda, name, q_name, heads, kv_heads, head_dim):
    call = Select(1, name, q_name, heads, kv_heads, head_dim, 16, [1, 0, 3, 1, 20], [1000, 5, 130, 0, 300],
                  before=2, behind=1, extra=8)
    for first, last, top in ((0, 1, 1), (1, 2, 8), (2, 3, 17), (0, 4, 64), (1, 1, 100)):
        call.check(first, last, top)


def test_ties_go_to_the_lower_page(torch_cuda):
    call = Select(2, "f16", "f16", 4, 2, 64, 8, [1, 2], [4000, 2500])
    call.least[:, :, :, 0] = call.least[:, :1, :, 0]  # one score for all pages of a KV head
    call.largest[:, :, :, 0] = call.largest[:, :1, :, 0]
    call.upload()
    for first, last, top in ((0, 1, 5), (2, 2, 64), (0, 7, 300)):
        call.check(first, last, top)
    # zeros of either sign are equal
    call.q_host.zero_()
    call.q_host[:, ::3] = -0.0
    call.q.copy_(call.q_host)
    call.check(0, 1, 9)


def test_pages_that_are_not_there_come_last(torch_cuda):
    call = Select(3, "bf16", "f32", 8, 1, 64, 16, [1, 4], [900, 300])
    call.host_table[0, 3::2] = -1
    call.host_table[1, 5] = call.cache.keys.shape[1]
    call.host_table[1, 6] = 2 ** 31 - 1
    call.table.copy_(call.host_table)
    for first, last, top in ((0, 1, 16), (4, 1, 40), (1, 6, 12)):
        call.check(first, last, top)


def test_scores_that_are_not_finite_come_first(torch_cuda):
    call = Select(4, "f16", "f32", 4, 1, 128, 16, [1, 1], [1600, 1600])
    for slot, value in ((50, math.nan), (71, math.inf), (20, -math.inf)):
        for s in range(2):
            call.least[1, int(call.host_table[s, slot]), 0, 0, 5] = value
            call.largest[1, int(call.host_table[s, slot]), 0, 0, 5] = value
    call.upload()
    for top in (2, 3, 4, 30):
        call.check(0, 1, top)
    # past fp32: 128 products of up to 65504 x 1e38
    call = Select(5, "f16", "f32", 4, 1, 128, 16, [1], [1600], spread=1e36)
    big = call.largest[1, :, 0, 0] > 2.5
    call.largest[1, :, 0, 0] = torch.where(big, 60000.0, call.largest[1, :, 0, 0])
    call.upload()
    call.check(0, 1, 12)


@pytest.mark.parametrize("cached", [0, 15, 16, 31, 32, 47, 1023, 1024])
def test_borders_of_pages(torch_cuda, cached):
    call = Select(6, "f16", "f16", 2, 1, 32, 16, [2], [cached])
    for first, last, top in ((0, 1, 1), (0, 1, 2), (1, 1, 2), (3, 2, 5), (0, 64, 64)):
        call.check(first, last, top)


def test_no_cached_rows_and_many_sequences(torch_cuda):
    call = Select(7, "bf16", "bf16", 4, 2, 64, 4, [1 + s % 3 for s in range(150)], [17 * s % 200 for s in range(150)])
    call.check(1, 1, 6)
    call = Select(8, "f16", "f16", 4, 2, 64, 4, [60], [0])
    call.batch.c.cached = None
    call.check(1, 1, 6)


def test_lengths_past_the_table(torch_cuda):
    """A row that lies past the table chooses among the pages that the table holds."""
    call = Select(9, "f16", "f16", 2, 1, 32, 16, [1], [800])
    call.batch.cached.copy_(ints([2 ** 31 - 1]))
    call.batch.cached_host = [2 ** 31 - 1]
    call.check(2, 3, 9)


def test_long_sequences_and_wide_tables(torch_cuda):
    call = Select(10, "f16", "f16", 8, 2, 128, 8, [1, 1], [70000, 3])
    call.check(1, 4, 256)
    call.check(0, 1, 2000)


def test_streams_and_graphs(torch_cuda):
    call = Select(11, "f16", "f32", 8, 1, 128, 16, [2, 1], [900, 2000])
    out = torch.zeros((3, 1, 24), dtype=torch.int32, device="cuda")
    stream = torch.cuda.Stream()
    call.call(1, 2, 24, out, stream.cuda_stream)
    stream.synchronize()
    assert torch.equal(out.cpu(), call.expected(1, 2, 24))
    graph = torch.cuda.CUDAGraph()
    size = call.workspace.numel()
    with torch.cuda.graph(graph, stream=stream):
        G.page_select(call.cache.c, 1, call.batch.c, call.bounds.c, call.q.data_ptr(), KIND[call.q.dtype],
                      call.q_stride, 8, 1, 2, 24, out.data_ptr(), call.workspace.data_ptr(), size,
                      torch.cuda.current_stream().cuda_stream)
    for cached in ([900, 2000], [10, 1999], [0, 500]):
        call.batch.cached.copy_(ints(cached))
        call.batch.cached_host = cached
        call.q_host = torch.randn(call.q_host.shape)
        call.q.copy_(call.q_host)
        out.fill_(5)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.cpu(), call.expected(1, 2, 24)), cached


def test_the_bound_is_one(torch_cuda):
    """No key's product with a query passes its page's score: the page of the largest
    product of all is among any two pages that are chosen, first or not."""
    g = torch.Generator().manual_seed(12)
    pages, page_rows, d = 64, 16, 64
    cache = Cache(torch.float16, 1, pages, page_rows, 1, d)
    keys = normal(g, cache.keys.shape, torch.float16, 0.05)
    table = torch.randperm(pages, generator=g)[None].to(torch.int32)
    q = normal(g, (1, d), torch.float16)
    best = 23
    keys[0, int(table[0, best]), 5, 0] = q[0] * 0.5  # far above the other products
    cache.keys.copy_(keys)
    bounds = Cache(torch.float16, 1, pages, 1, 1, d)
    device_table, dq = table.cuda(), q.cuda()
    whole = Batch([pages * page_rows], [0], device_table)
    page_bounds(cache, 0, whole, bounds)
    batch = Batch([1], [pages * page_rows - 1], device_table)
    out = torch.zeros((1, 1, 2), dtype=torch.int32, device="cuda")
    workspace = torch.zeros(G.page_select_workspace_bytes(1, 1, pages), dtype=torch.uint8, device="cuda")
    G.page_select(cache.c, 0, batch.c, bounds.c, dq.data_ptr(), KIND[torch.float16], d, 1, 0, 1, 2,
                  out.data_ptr(), workspace.data_ptr(), workspace.numel())
    assert out.cpu().tolist() == [[[best, pages - 1]]]
