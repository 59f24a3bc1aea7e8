"""Attention of packed sequences over a paged cache against its definition in
64 bits: causal prompts and drafted trees, over types, head layouts, page sizes,
lengths from nothing to several units, strides and places that hold no rows."""
import math

import pytest
import torch

from huggingfaceeacp_amd import gemma_q8 as G
from paged_helpers import (KIND, SENTINEL, TYPES, Batch, Cache, assert_near, definition, definition_fast,
                           ints, kv_type, normal, random_cache)

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator().manual_seed(seed)


class Call:
    """A batch's inputs on both sides and a call of either attention."""

    def __init__(self, torch_cuda, seed, name, heads, kv_heads, head_dim, page_rows, rows, cached,
                 before=0, behind=0, extra=0, layers=1, layer=0):
        g = gen(seed)
        self.dtype, self.heads, self.layer = TYPES[name], heads, layer
        self.kv_heads, self.head_dim = kv_heads, head_dim
        self.cache, self.held, self.table = random_cache(g, kv_type(name), cached, page_rows, kv_heads,
                                                         head_dim, layers, layer)
        self.batch = Batch(rows, cached, self.table, before, behind)
        total = self.batch.total
        self.q_stride, self.kv_stride = heads * head_dim + extra, kv_heads * head_dim + extra
        self.q_host = normal(g, (total, self.q_stride), self.dtype, 1.5)
        self.k_host = normal(g, (total, self.kv_stride), kv_type(name))
        self.v_host = normal(g, (total, self.kv_stride), kv_type(name))
        self.scale = 1.0 / math.sqrt(head_dim)
        self.masks = None
        self.upload()

    def upload(self):
        self.q, self.k, self.v = self.q_host.cuda(), self.k_host.cuda(), self.v_host.cuda()
        size = G.packed_attention_workspace_bytes(self.heads, self.kv_heads, self.head_dim)
        self.workspace = torch.full((size // 4,), math.nan, device="cuda")

    def fresh_out(self):
        return torch.full((self.batch.total, self.q_stride), SENTINEL, dtype=self.dtype, device="cuda")

    def causal(self, out=None, stream=0):
        out = self.fresh_out() if out is None else out
        G.packed_attention(self.cache.c, self.layer, self.batch.c, self.q.data_ptr(), KIND[self.dtype],
                           self.q_stride, self.heads, self.k.data_ptr(), self.v.data_ptr(),
                           self.kv_stride, self.scale, out.data_ptr(), self.q_stride,
                           self.workspace.data_ptr(), self.workspace.numel() * 4, stream)
        return out

    def tree(self, out=None, own=True, stream=0):
        out = self.fresh_out() if out is None else out
        G.tree_attention(self.cache.c, self.layer, self.batch.c, self.q.data_ptr(), KIND[self.dtype],
                         self.q_stride, self.heads, self.k.data_ptr() if own else None,
                         self.v.data_ptr() if own else None, self.kv_stride,
                         self.masks.data_ptr() if own else None, self.masks.shape[1] if own else 0,
                         self.scale, out.data_ptr(), self.q_stride, self.workspace.data_ptr(),
                         self.workspace.numel() * 4, stream)
        return out

    def allowed(self, s, how, hidden=()):
        n, c = self.batch.rows[s], self.batch.cached_host[s]
        seen = torch.ones((n, c + n), dtype=torch.bool)
        for key in hidden:
            seen[:, key] = False
        if how == "causal":
            seen[:, c:] = torch.tril(seen[:, c:])
        elif how == "cached":
            seen[:, c:] = False
        else:
            first = self.batch.spans[s][0]
            words = self.masks_host[first:first + n]
            for j in range(n):
                bit = (words[:, j // 64] >> (j % 64)) & 1 if j // 64 < words.shape[1] else torch.zeros(n)
                seen[:, c + j] = bit != 0
        return seen

    def rows_of(self, s):
        a, b = self.batch.spans[s]
        h, g, d = self.heads, self.kv_heads, self.head_dim
        return (self.q_host[a:b, :h * d].reshape(-1, h, d),
                torch.cat([self.held[s][0], self.k_host[a:b, :g * d].reshape(-1, g, d)]),
                torch.cat([self.held[s][1], self.v_host[a:b, :g * d].reshape(-1, g, d)]))

    def check(self, out, how, what, by=definition_fast, hidden=()):
        out = out.cpu()
        width = self.heads * self.head_dim
        touched = torch.zeros(self.batch.total, dtype=torch.bool)
        for s, (a, b) in enumerate(self.batch.spans):
            touched[a:b] = True
            if a == b:
                continue
            q, k, v = self.rows_of(s)
            expected = by(q, k, v, self.allowed(s, how, hidden), self.scale)
            peak = v[torch.isfinite(v)].abs().max().item() if v.numel() else 1.0
            assert_near(out[a:b, :width].reshape(b - a, self.heads, -1), expected, peak, self.dtype,
                        (what, s))
        # rows of no sequence and the columns past the heads are as they were
        assert (out[~touched] == SENTINEL).all(), what
        assert (out[:, width:] == SENTINEL).all(), what

    def draw_masks(self, seed, words=1, empty=()):
        g = gen(seed)
        masks = torch.zeros((self.batch.total, words), dtype=torch.int64)
        for a, b in self.batch.spans:
            bits = []
            for i in range(b - a):
                parent = int(torch.randint(0, i, (1,), generator=g)) if i else -1
                own = [False] * (64 * words)
                if parent >= 0:
                    own = list(bits[parent])
                if i < 64 * words:
                    own[i] = True
                bits.append(own)
            for i, own in enumerate(bits):
                for w in range(words):
                    value = sum(1 << j for j in range(64) if own[64 * w + j])
                    masks[a + i, w] = value - (1 << 64) if value >> 63 else value
        for row in empty:
            masks[row] = 0
        self.masks_host, self.masks = masks, masks.cuda()


HEADS = [(8, 1, 256), (4, 4, 64), (6, 2, 128), (3, 1, 80), (14, 2, 96), (2, 1, 8), (32, 1, 64)]


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,head_dim", HEADS)
def test_causal_ragged_batch(torch_cuda, name, heads, kv_heads, head_dim):
    rows = [1, 0, 64, 17, 130, 2, 65]
    cached = [0, 5, 64, 63, 1, 129, 0]
    call = Call(torch_cuda, 1, name, heads, kv_heads, head_dim, 16, rows, cached, before=2, behind=3,
                extra=8, layers=2, layer=1)
    call.check(call.causal(), "causal", (name, heads, kv_heads, head_dim))


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,head_dim", HEADS)
def test_trees(torch_cuda, name, heads, kv_heads, head_dim):
    rows = [1, 5, 0, 33, 64, 2]
    cached = [100, 0, 7, 64, 65, 200]
    call = Call(torch_cuda, 2, name, heads, kv_heads, head_dim, 32, rows, cached, before=1, behind=2,
                extra=16)
    # the second sequence's third row attends nothing at all
    call.draw_masks(3, empty=[1 + 1 + 2])
    out = call.tree()
    call.check(out, "tree", (name, heads, kv_heads, head_dim))
    assert (out[4, :heads * head_dim] == 0).all()


@pytest.mark.parametrize("name,heads,kv_heads,head_dim",
                         [("f32", 8, 1, 256), ("f16", 8, 2, 128), ("bf16", 4, 4, 64)])
def test_single_tokens(torch_cuda, name, heads, kv_heads, head_dim):
    cached = [0, 1, 63, 64, 65, 513, 1000, 0, 129, 31]
    call = Call(torch_cuda, 4, name, heads, kv_heads, head_dim, 8, [1] * len(cached), cached)
    call.draw_masks(5)
    call.check(call.tree(), "tree", name)
    # over the cache alone: the sequences with nothing cached get zeros
    out = call.tree(own=False)
    call.check(out, "cached", name)
    assert (out[0] == 0).all() and (out[7] == 0).all()


@pytest.mark.parametrize("page_rows", [1, 2, 16, 64, 256])
@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_page_sizes(torch_cuda, page_rows, name):
    call = Call(torch_cuda, 6, name, 4, 2, 128, page_rows, [40, 1, 9], [150, 77, 256])
    call.check(call.causal(), "causal", page_rows)


@pytest.mark.parametrize("sequences", [1, 65, 200])
def test_many_sequences(torch_cuda, sequences):
    """Over 64 sequences the place of a unit is found in several steps."""
    g = gen(7)
    rows = torch.randint(0, 4, (sequences,), generator=g).tolist()
    rows[-1] = 3
    cached = torch.randint(0, 90, (sequences,), generator=g).tolist()
    call = Call(torch_cuda, 8, "f32", 4, 1, 64, 16, rows, cached)
    call.check(call.causal(), "causal", sequences)
    call.draw_masks(9)
    call.check(call.tree(), "tree", sequences)


@pytest.mark.parametrize("name,heads,kv_heads,head_dim",
                         [("f32", 8, 1, 256), ("f16", 8, 2, 128), ("bf16", 3, 3, 64)])
def test_long(torch_cuda, name, heads, kv_heads, head_dim):
    """Tiles that many workgroups share, and workgroups that hold many tiles."""
    call = Call(torch_cuda, 10, name, heads, kv_heads, head_dim, 64, [700, 1, 1300], [333, 4000, 0])
    call.check(call.causal(), "causal", name)


@pytest.mark.parametrize("words", [1, 2, 3])
def test_mask_words(torch_cuda, words):
    """Rows past the words' bits are attended by none."""
    call = Call(torch_cuda, 11, "f16", 8, 2, 64, 16, [150, 70], [10, 0])
    call.draw_masks(12, words)
    call.check(call.tree(), "tree", words)


@pytest.mark.parametrize("name,head_dim", [("f32", 256), ("f32", 64), ("f16", 256), ("bf16", 128)])
@pytest.mark.parametrize("rows", [3, 40])
def test_values_that_are_not_finite_stay_with_their_rows(torch_cuda, name, head_dim, rows):
    """A NaN or infinity among the keys and values of a row reaches the rows that
    attend it, in its own channel alone, and no others."""
    call = Call(torch_cuda, 13, name, 4, 2, head_dim, 16, [rows, rows], [20, 0])
    for s, (a, b) in enumerate(call.batch.spans):
        call.v_host[a + 1, 3] = math.nan
        call.v_host[a + 2, head_dim + 5] = math.inf
        call.k_host[b - 1, 7] = math.nan
    call.upload()
    out = call.causal().cpu()
    for s, (a, b) in enumerate(call.batch.spans):
        q, k, v = call.rows_of(s)
        expected = definition(q, k, v, call.allowed(s, "causal"), call.scale)
        got = out[a:b].reshape(rows, 4, head_dim).double()
        assert torch.equal(torch.isnan(got), torch.isnan(expected)), s
        assert torch.equal(torch.isinf(got), torch.isinf(expected)), s
        fine = torch.isfinite(expected)
        assert fine[0].all() and fine[1, :, :3].all()
        peak = v[torch.isfinite(v)].abs().max().item()
        assert_near(got[fine], expected[fine], peak, call.dtype, s)
    # a tree whose second row attends itself alone, and its third neither
    call.draw_masks(14)
    for a, b in call.batch.spans:
        call.masks_host[a + 1], call.masks_host[a + 2] = 2, 1
        call.masks_host[a + 3:b] &= 1
    call.masks = call.masks_host.cuda()
    out = call.tree().cpu()
    for s, (a, b) in enumerate(call.batch.spans):
        q, k, v = call.rows_of(s)
        expected = definition(q, k, v, call.allowed(s, "tree"), call.scale)
        got = out[a:b].reshape(rows, 4, head_dim).double()
        assert torch.equal(torch.isnan(got), torch.isnan(expected)), s
        fine = torch.isfinite(expected)
        assert_near(got[fine], expected[fine], 5.0, call.dtype, s)


@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_pages_that_are_not_there(torch_cuda, name):
    """Rows in a page outside the pool are attended by none; lengths past the
    table are cut to it."""
    call = Call(torch_cuda, 15, name, 4, 1, 128, 16, [5, 70], [100, 100])
    table = call.table.clone()
    table[0, 2], table[0, 5] = -1, call.cache.c.pages
    table[1, 0] = 2 ** 31 - 1
    call.table.copy_(table)
    out = call.causal().cpu()
    for s, hidden in ((0, [*range(32, 48), *range(80, 96)]), (1, range(16))):
        a, b = call.batch.spans[s]
        q, k, v = call.rows_of(s)
        expected = definition_fast(q, k, v, call.allowed(s, "causal", hidden), call.scale)
        assert_near(out[a:b].reshape(b - a, 4, -1), expected, v.abs().max().item(), call.dtype, s)
    # every page gone: the rows are left with their own
    call.table.fill_(-1)
    call.batch.cached.fill_(2 ** 31 - 1)
    out = call.causal().cpu()
    for s in range(2):
        a, b = call.batch.spans[s]
        q, k, v = call.rows_of(s)
        expected = definition_fast(q, k, v, call.allowed(s, "causal", range(100)), call.scale)
        assert_near(out[a:b].reshape(b - a, 4, -1), expected, v.abs().max().item(), call.dtype, s)


def test_no_cache_at_all(torch_cuda):
    call = Call(torch_cuda, 16, "f16", 8, 2, 64, 16, [70, 3], [0, 0])
    call.cache.c = G.PageCache(None, None, KIND[torch.float16], 1, 0, 16, 2, 64)
    call.batch.c = G.Sequences(2, call.batch.total, call.batch.starts.data_ptr(), None, None, 0)
    call.check(call.causal(), "causal", "no cache")


@pytest.mark.parametrize("scale", [-0.1, 0.0, 3.0])
@pytest.mark.parametrize("name", ["f32", "f16"])
def test_scales(torch_cuda, scale, name):
    call = Call(torch_cuda, 17, name, 2, 1, 64, 16, [30], [90])
    call.scale = scale
    out = call.causal().cpu()
    q, k, v = call.rows_of(0)
    expected = definition_fast(q, k, v, call.allowed(0, "causal"), scale)
    # scores of up to 3 sqrt(64) 1.5 x 4 ~ 150 instead of 15: their errors grow alike
    grown = max(1.0, scale * 8)
    got = out.reshape(30, 2, 64).double()
    step = 0 if name == "f32" else 2 * torch.finfo(torch.float16).eps / 2
    assert (got - expected).abs().max() <= (step + 1e-4 * grown) * v.abs().max()


def test_scores_that_grow(torch_cuda):
    """Each unit's scores pass the last's by far more than the margin: every one
    moves the reference, in both directions of the row."""
    call = Call(torch_cuda, 18, "f32", 2, 1, 64, 16, [1, 3], [500, 500])
    for s in range(2):
        k = call.held[s][0]
        ramp = torch.linspace(0.1, 6, 500) if s == 0 else torch.linspace(6, 0.1, 500)
        k *= ramp[:, None, None].half()
        for j in range(-(-500 // 16)):
            n = min(16, 500 - 16 * j)
            call.cache.keys[0, int(call.table[s, j]), :n] = k[16 * j:16 * j + n].cuda()
    out = call.causal().cpu()
    for s, (a, b) in enumerate(call.batch.spans):
        q, k, v = call.rows_of(s)
        expected = definition_fast(q, k, v, call.allowed(s, "causal"), call.scale)
        got = out[a:b].reshape(b - a, 2, 64).double()
        # six times the score, six times its error
        assert (got - expected).abs().max() <= 6e-4 * v.abs().max()


@pytest.mark.parametrize("size", [1e-30, 1e-6, 1e5, 1e20])
def test_queries_of_any_size(torch_cuda, size):
    """fp32 queries far outside fp16's range: scores as small as nothing, or one
    key that takes all."""
    call = Call(torch_cuda, 19, "f32", 2, 1, 64, 16, [4], [60])
    call.q_host = (call.q_host * size).contiguous()
    call.upload()
    out = call.causal().cpu()
    q, k, v = call.rows_of(0)
    expected = definition_fast(q, k, v, call.allowed(0, "causal"), call.scale)
    got = out.reshape(4, 2, 64).double()
    assert torch.isfinite(got).all()
    # with scores of 1e4 and more the largest takes all but e^-10 or so: ties closer
    # than that are not among these inputs (their gaps exceed 1e-4 of the score)
    tolerance = 1e-4 if size <= 1 else 1e-2
    assert (got - expected).abs().max() <= tolerance * v.abs().max()


def test_offsets_past_32_bits(torch_cuda):
    """A pool of 6 GB a side, of which the last pages are read and written."""
    pages, page_rows = 25000, 128
    c = G.PageCache()
    keys = torch.empty((pages, page_rows, 4, 256), dtype=torch.float16, device="cuda")
    values = torch.empty_like(keys)
    assert keys.numel() * 2 > 6 << 30
    c = G.PageCache(keys.data_ptr(), values.data_ptr(), KIND[torch.float16], 1, pages, page_rows, 4, 256)
    call = Call(torch_cuda, 20, "f16", 8, 4, 256, page_rows, [3], [300])
    table = ints([[pages - 1, pages - 7, pages - 3]])
    for j in range(3):
        page = int(call.table[0, j])
        keys[int(table[0, j])] = call.cache.keys[0, page]
        values[int(table[0, j])] = call.cache.values[0, page]
    call.cache.c = c
    call.batch.c.page_table = table.data_ptr()
    call.check(call.causal(), "causal", "far pages")


def test_streams_and_graphs(torch_cuda):
    """Captured calls replay with new lengths, queries and pages, other work
    between the replays; a call on another stream gives the same bits."""
    torch.cuda.synchronize()
    call = Call(torch_cuda, 21, "f32", 8, 1, 256, 16, [40, 3, 1], [200, 0, 900])
    call.draw_masks(22)
    causal, tree = call.fresh_out(), call.fresh_out()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        call.causal(causal, stream.cuda_stream)
        call.tree(tree, stream=stream.cuda_stream)
    stream.synchronize()
    assert torch.equal(causal, call.causal()) and torch.equal(tree, call.tree())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        call.causal(causal, torch.cuda.current_stream().cuda_stream)
        call.tree(tree, stream=torch.cuda.current_stream().cuda_stream)
    for starts, cached in (([0, 40, 43, 44], [200, 0, 900]), ([0, 1, 1, 44], [3, 200, 897]),
                           ([5, 6, 7, 30], [0, 0, 0])):
        call.batch.starts.copy_(ints(starts))
        call.batch.cached.copy_(ints(cached))
        call.q.copy_(torch.randn_like(call.q))
        causal.fill_(SENTINEL)
        tree.fill_(SENTINEL)
        graph.replay()
        torch.cuda.synchronize()
        expected = call.causal(), call.tree()
        torch.cuda.synchronize()
        assert torch.equal(causal, expected[0]) and torch.equal(tree, expected[1]), starts


def test_nothing_to_do(torch_cuda):
    """No rows, no sequences: the calls return and write nothing."""
    call = Call(torch_cuda, 23, "f16", 4, 1, 64, 16, [2], [5])
    for sequences, rows in ((0, 2), (1, 0), (0, 0)):
        call.batch.c = G.Sequences(sequences, rows, call.batch.starts.data_ptr(),
                                   call.batch.cached.data_ptr(), call.table.data_ptr(),
                                   call.table.shape[1])
        out = call.causal()
        assert (out == SENTINEL).all()
    # sequences that are all empty
    empty = ints([1, 1])
    call.batch.c = G.Sequences(1, 2, empty.data_ptr(), call.batch.cached.data_ptr(),
                               call.table.data_ptr(), call.table.shape[1])
    assert (call.causal() == SENTINEL).all()
