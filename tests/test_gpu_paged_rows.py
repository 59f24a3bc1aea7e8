"""The paged cache's rows on the GPU: per-head norms with rotation, appends and
page copies against plain indexing and 64-bit arithmetic, and a run of all of
the cache's operators together as a server uses them."""
import math

import numpy as np
import pytest
import torch

from huggingfaceeacp_amd import gemma_q8 as G
from paged_helpers import (KIND, SENTINEL, TYPES, Batch, Cache, assert_near, definition_fast, half_step, ints,
                           kv_type, normal, random_cache)

pytestmark = pytest.mark.gpu

EPSILON = 1e-6


def gen(seed):
    return torch.Generator().manual_seed(seed)


def tables(positions, head_dim):
    c, s = G.rotary_table_host(positions, head_dim)
    return torch.from_numpy(c), torch.from_numpy(s)


def norm_rope_definition(x, weight, cos, sin):
    """x [rows, heads, d] in 64 bits; cos and sin [rows, d / 2]."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + np.float64(np.float32(EPSILON)))
        x = x * (1 + weight.double())
    a, b = x.chunk(2, -1)
    c, s = cos.double()[:, None], sin.double()[:, None]
    return torch.cat([a * c - b * s, a * s + b * c], -1)


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,heads,kv_heads,head_dim",
                         [(1, 8, 1, 256), (5, 4, 2, 64), (33, 7, 7, 96), (2, 3, 1, 8), (300, 32, 8, 128),
                          (9, 6, 3, 80)])
def test_norm_and_rotation(torch_cuda, name, rows, heads, kv_heads, head_dim):
    g = gen(rows)
    dtype, kv = TYPES[name], kv_type(name)
    columns = (heads + 2 * kv_heads) * head_dim
    x = normal(g, (rows, columns + 8), dtype, 3.0)
    x[0, :head_dim] = 0  # a head of zeros
    weights = [normal(g, (head_dim,), torch.float32, 0.5) for _ in range(2)]
    cos, sin = tables(50, head_dim)
    positions = torch.randint(0, 50, (rows,), generator=g)
    live = torch.ones(rows, dtype=torch.bool)
    if rows > 4:  # rows outside the tables are left as they were
        positions[1], positions[3] = -1, 50
        live[1] = live[3] = False
    dev = [t.cuda() for t in (x, *weights, ints(positions, "cpu"), cos, sin)]
    dx, dq, dk, dp, dc, ds = dev
    parts = x[:, :columns].reshape(rows, -1, head_dim)
    at = positions.clamp(0, 49)
    for weighted in (True, False):
        q = torch.full((rows, heads * head_dim + 8), SENTINEL, dtype=dtype, device="cuda")
        k = torch.full((rows, kv_heads * head_dim + 16), SENTINEL, dtype=kv, device="cuda")
        v = torch.full_like(k, SENTINEL)
        G.head_norm_rope(dx.data_ptr(), KIND[dtype], rows, columns + 8, heads, kv_heads, head_dim,
                         dq.data_ptr() if weighted else None, dk.data_ptr() if weighted else None,
                         EPSILON, dp.data_ptr(), dc.data_ptr(), ds.data_ptr(), 50, q.data_ptr(),
                         KIND[dtype], heads * head_dim + 8, k.data_ptr(), v.data_ptr(), KIND[kv],
                         kv_heads * head_dim + 16)
        for got, first, count, weight, out_type in ((q, 0, heads, weights[0], dtype),
                                                    (k, heads, kv_heads, weights[1], kv)):
            expected = norm_rope_definition(parts[:, first:first + count], weight if weighted else None,
                                            cos[at], sin[at])
            got = got.cpu()
            width = count * head_dim
            assert (got[:, width:] == SENTINEL).all() and (got[~live] == SENTINEL).all()
            got, expected = got[live][:, :width].double(), expected[live].reshape(-1, width)
            # rounded once from fp32: half a step of its type and of fp32's; fp16's
            # subnormals end at 2^-24
            bound = (half_step(out_type) + 2 ** -24) * expected.abs() * 1.0001 + (
                0 if out_type == torch.bfloat16 else 2 ** -25 if out_type == torch.float16 else 1e-40)
            assert ((got - expected).abs() <= bound + 1e-13).all()
        expected = parts[live][:, heads + kv_heads:].reshape(-1, kv_heads * head_dim).to(kv)
        got = v.cpu()
        assert torch.equal(got[live][:, :kv_heads * head_dim], expected)
        assert (got[~live] == SENTINEL).all() and (got[:, kv_heads * head_dim:] == SENTINEL).all()
        # without the values, then without keys or values: the same queries
        for k_to, v_to in ((k, None), (None, v), (None, None)):
            again = torch.full_like(q, SENTINEL)
            other = [torch.full_like(t, SENTINEL) if t is not None else None for t in (k_to, v_to)]
            G.head_norm_rope(dx.data_ptr(), KIND[dtype], rows, columns + 8, heads, kv_heads, head_dim,
                             dq.data_ptr() if weighted else None, dk.data_ptr() if weighted else None,
                             EPSILON, dp.data_ptr(), dc.data_ptr(), ds.data_ptr(), 50, again.data_ptr(),
                             KIND[dtype], heads * head_dim + 8,
                             other[0].data_ptr() if other[0] is not None else None,
                             other[1].data_ptr() if other[1] is not None else None, KIND[kv],
                             kv_heads * head_dim + 16)
            assert torch.equal(again, q)
            for t, full in zip(other, (k, v)):
                assert t is None or torch.equal(t, full)


def test_norm_and_rotation_in_place(torch_cuda):
    g = gen(3)
    heads, kv_heads, d, rows = 4, 2, 128, 17
    stride = (heads + 2 * kv_heads) * d
    x = normal(g, (rows, stride), torch.bfloat16, 2.0).cuda()
    w = normal(g, (d,), torch.float32, 0.5).cuda()
    cos, sin = (t.cuda() for t in tables(40, d))
    positions = ints(np.arange(rows) + 5)
    q = torch.empty((rows, heads * d), dtype=torch.bfloat16, device="cuda")
    k, v = (torch.empty((rows, kv_heads * d), dtype=torch.bfloat16, device="cuda") for _ in range(2))

    def call(x, q, q_stride, k, v, kv_stride):
        G.head_norm_rope(x.data_ptr(), KIND[x.dtype], rows, stride, heads, kv_heads, d, w.data_ptr(),
                         w.data_ptr(), EPSILON, positions.data_ptr(), cos.data_ptr(), sin.data_ptr(), 40,
                         q, KIND[x.dtype], q_stride, k, v, KIND[x.dtype], kv_stride)

    call(x, q.data_ptr(), heads * d, k.data_ptr(), v.data_ptr(), kv_heads * d)
    y = x.clone()
    base = y.data_ptr()
    call(y, base, stride, base + heads * d * 2, base + (heads + kv_heads) * d * 2, stride)
    assert torch.equal(y, torch.cat([q, k, v], 1))


@pytest.mark.parametrize("name", ["f16", "bf16"])
@pytest.mark.parametrize("kv_heads,head_dim,page_rows", [(1, 256, 16), (3, 8, 1), (4, 80, 64), (2, 64, 4)])
def test_append(torch_cuda, name, kv_heads, head_dim, page_rows):
    g = gen(7)
    dtype = TYPES[name]
    rows, cached = [5, 0, 70, 1, 9], [0, 3, 30, 64, 15]
    width = max(-(-(n + c) // page_rows) for n, c in zip(rows, cached))
    pages = width * len(rows) + 3
    order = torch.randperm(pages, generator=g).to(torch.int32)
    host_table = order[:width * len(rows)].reshape(len(rows), width).clone()
    host_table[3] = -1                # a sequence without pages
    host_table[4, 0] = pages          # and one whose first page is outside the pool
    table = host_table.cuda()
    cache = Cache(dtype, 2, pages, page_rows, kv_heads, head_dim)
    cache.keys.fill_(SENTINEL)
    cache.values.fill_(SENTINEL)
    batch = Batch(rows, cached, table, before=2, behind=3)
    stride = kv_heads * head_dim + 24
    k, v = (normal(g, (batch.total, stride), dtype) for _ in range(2))
    dk, dv = k.cuda(), v.cuda()
    places = torch.full((batch.total,), 3, dtype=torch.int32)
    for a, b in batch.spans:
        order = torch.randperm(b - a, generator=g).to(torch.int32)
        places[a:b] = torch.where(order % 3 == 1, -1, order)  # a third is left out
    for chosen in (None, places):
        expected = [torch.full(cache.keys.shape, SENTINEL, dtype=dtype) for _ in range(2)]
        cache.keys.fill_(SENTINEL)
        cache.values.fill_(SENTINEL)
        for s, (a, b) in enumerate(batch.spans):
            for i in range(b - a):
                place = i if chosen is None else int(chosen[a + i])
                row = cached[s] + place
                if place < 0 or row // page_rows >= width:
                    continue
                page = int(host_table[s, row // page_rows])
                if 0 <= page < pages:
                    for full, new in zip(expected, (k, v)):
                        full[1, page, row % page_rows] = new[a + i, :kv_heads * head_dim].reshape(
                            kv_heads, head_dim)
        device_places = chosen.cuda() if chosen is not None else None
        G.page_append(cache.c, 1, batch.c, dk.data_ptr(), dv.data_ptr(), stride,
                      device_places.data_ptr() if chosen is not None else None)
        assert torch.equal(cache.keys.cpu(), expected[0]) and torch.equal(cache.values.cpu(), expected[1])


def test_append_of_many_sequences(torch_cuda):
    """More sequences than lanes, most of them empty; a length past the table is
    stored nowhere."""
    rows = [1 if s % 3 == 0 else 0 for s in range(200)]
    cached = [s % 7 for s in range(200)]
    cached[3] = 8
    table = ints(np.arange(200)[:, None])
    cache = Cache(torch.float16, 1, 200, 8, 1, 16)
    cache.keys.fill_(SENTINEL)
    batch = Batch(rows, cached, table)
    k = normal(gen(9), (batch.total, 16), torch.float16).cuda()
    G.page_append(cache.c, 0, batch.c, k.data_ptr(), k.data_ptr(), 16)
    expected = torch.full(cache.keys.shape, SENTINEL, dtype=torch.float16)
    for s in range(0, 200, 3):
        if s != 3:
            expected[0, s, cached[s], 0] = k[batch.spans[s][0]].cpu()
    assert torch.equal(cache.keys.cpu(), expected)


@pytest.mark.parametrize("layers,page_rows,kv_heads,head_dim", [(1, 1, 1, 8), (18, 16, 1, 256), (3, 64, 5, 80)])
def test_page_copy(torch_cuda, layers, page_rows, kv_heads, head_dim):
    pages = 23
    cache = Cache(torch.float16, layers, pages, page_rows, kv_heads, head_dim)
    cache.keys.copy_(torch.randn(cache.keys.shape, generator=gen(1)))
    cache.values.copy_(torch.randn(cache.values.shape, generator=gen(2)))
    pairs = [[0, 22], [0, 5], [7, 1], [-1, 3], [4, 23], [9, 2], [6, -5], [30, 8]]
    keys, values = cache.keys.clone(), cache.values.clone()
    for a, b in pairs:
        if 0 <= a < pages and 0 <= b < pages:
            keys[:, b], values[:, b] = keys[:, a], values[:, a]
    device_pairs = ints(pairs)
    G.page_copy(cache.c, device_pairs.data_ptr(), len(pairs))
    assert torch.equal(cache.keys, keys) and torch.equal(cache.values, values)


def test_a_server_s_run(torch_cuda):
    """Prompts, forks, drafted trees with their accepted paths, single tokens and a
    compaction over one pool, at every step against each sequence's own rows
    kept apart on the host; two layers, one of them untouched by the appends."""
    g = gen(11)
    heads, kv_heads, d, page_rows, layer = 8, 1, 256, 16, 1
    pool = G.PagePool(64, page_rows, 6, 12)
    cache = Cache(torch.float16, 2, 64, page_rows, kv_heads, d)
    cos, sin = tables(200, d)
    dcos, dsin = cos.cuda(), sin.cuda()
    weights = [normal(g, (d,), torch.float32, 0.3) for _ in range(2)]
    dweights = [w.cuda() for w in weights]
    workspace = torch.empty(G.packed_attention_workspace_bytes(heads, kv_heads, d), dtype=torch.uint8,
                            device="cuda")
    scale = 1 / math.sqrt(d)
    held = {}  # sequence -> (keys, values) on the host, as stored

    def copies():
        pairs = torch.from_numpy(pool.take_copies()).cuda()
        G.page_copy(cache.c, pairs.data_ptr(), len(pairs))
        torch.cuda.synchronize()

    def step(ids, new_rows, parents=None):
        """Norms, rotation and attention of new rows (a tree where parents are
        given), checked; returns the batch and its keys and values."""
        host_table, lengths = pool.tables(ids)
        table = torch.from_numpy(host_table).cuda()
        batch = Batch(new_rows, lengths.tolist(), table, behind=1)
        x = normal(g, (batch.total, (heads + 2 * kv_heads) * d), torch.float32, 2.0)
        positions = torch.full((batch.total,), -1, dtype=torch.int32)
        masks = torch.zeros((batch.total, 1), dtype=torch.int64)
        for s, (a, b) in enumerate(batch.spans):
            for i in range(b - a):
                parent = parents[s][i] if parents else i - 1
                positions[a + i] = positions[a + parent] + 1 if parent >= 0 else int(lengths[s])
                if parents:
                    own = (1 << i) - (1 << 64 if i == 63 else 0)
                    masks[a + i] = (masks[a + parent] if parent >= 0 else 0) | own
        dx, dpos, dmasks = x.cuda(), positions.cuda(), masks.cuda()
        q = torch.zeros((batch.total, heads * d), device="cuda")
        k, v = (torch.zeros((batch.total, kv_heads * d), dtype=torch.float16, device="cuda")
                for _ in range(2))
        G.head_norm_rope(dx.data_ptr(), KIND[torch.float32], batch.total, x.shape[1], heads, kv_heads, d,
                         dweights[0].data_ptr(), dweights[1].data_ptr(), EPSILON, dpos.data_ptr(),
                         dcos.data_ptr(), dsin.data_ptr(), 200, q.data_ptr(), KIND[torch.float32],
                         heads * d, k.data_ptr(), v.data_ptr(), KIND[torch.float16], kv_heads * d)
        out = torch.full((batch.total, heads * d), SENTINEL, device="cuda")
        head = (cache.c, layer, batch.c, q.data_ptr(), KIND[torch.float32], heads * d, heads, k.data_ptr(),
                v.data_ptr(), kv_heads * d)
        tail = (scale, out.data_ptr(), heads * d, workspace.data_ptr(), workspace.numel())
        if parents:
            G.tree_attention(*head, dmasks.data_ptr(), 1, *tail)
        else:
            G.packed_attention(*head, *tail)
        torch.cuda.synchronize()
        assert (out[-1] == SENTINEL).all()
        for s, (a, b) in enumerate(batch.spans):
            if a == b:
                continue
            parts = x[a:b].reshape(b - a, -1, d)
            at = positions[a:b].long()
            expected_q = norm_rope_definition(parts[:, :heads], weights[0], cos[at], sin[at])
            assert (q[a:b].cpu().double().reshape(-1, heads, d) - expected_q).abs().max() < 2e-6
            old_k, old_v = held[ids[s]]
            keys = torch.cat([old_k, k[a:b].cpu().reshape(-1, kv_heads, d)])
            values = torch.cat([old_v, v[a:b].cpu().reshape(-1, kv_heads, d)])
            n, c = b - a, len(old_k)
            allowed = torch.ones((n, c + n), dtype=torch.bool)
            for j in range(n):
                allowed[:, c + j] = (masks[a:b, 0] >> j) & 1 != 0 if parents else torch.arange(n) >= j
            expected = definition_fast(q[a:b].cpu().reshape(-1, heads, d), keys, values, allowed, scale)
            assert_near(out[a:b].reshape(n, heads, d), expected, values.abs().max().item(), torch.float32, s)
        return batch, k, v

    def store(ids, batch, k, v, taken):
        """The taken rows of each sequence, in order, go into its pages."""
        places = torch.full((batch.total,), -1, dtype=torch.int32)
        for s, (a, b) in enumerate(batch.spans):
            for place, i in enumerate(taken[s]):
                places[a + i] = place
            pool.extend(ids[s], len(taken[s]))
            old_k, old_v = held[ids[s]]
            at = torch.tensor([a + i for i in taken[s]], dtype=torch.long)
            held[ids[s]] = (torch.cat([old_k, k.cpu()[at].reshape(-1, kv_heads, d)]),
                            torch.cat([old_v, v.cpu()[at].reshape(-1, kv_heads, d)]))
        copies()
        table = torch.from_numpy(pool.tables(ids)[0]).cuda()
        batch.c.page_table = table.data_ptr()  # the lengths are those before the step
        dplaces = places.cuda()
        G.page_append(cache.c, layer, batch.c, k.data_ptr(), v.data_ptr(), kv_heads * d,
                      dplaces.data_ptr())
        torch.cuda.synchronize()

    empty = torch.zeros((0, kv_heads, d), dtype=torch.float16)
    ids = [pool.open() for _ in range(3)]
    held.update({s: (empty, empty) for s in ids})
    rows = [37, 1, 70]
    batch, k, v = step(ids, rows)
    store(ids, batch, k, v, [range(n) for n in rows])
    child = pool.fork(ids[0])
    held[child] = held[ids[0]]
    ids.append(child)
    for turn in range(3):
        count = [9, 0, 30, 5] if turn % 2 == 0 else [1, 17, 2, 64]
        parents = [[-1] + [int(torch.randint(max(0, i - 3), i, (1,), generator=g)) for i in range(1, n)]
                   if n else [] for n in count]
        batch, k, v = step(ids, count, parents)
        taken = []
        for p in parents:  # the path to the last node
            path, node = [], len(p) - 1
            while node >= 0:
                path.insert(0, node)
                node = p[node]
            taken.append(path)
        store(ids, batch, k, v, taken)
    # one sequence ends, the rest move to the front of the pool
    pool.close(ids[1])
    del held[ids[1]]
    ids = [ids[0], ids[2], ids[3]]
    pool.truncate(ids[1], 40)
    held[ids[1]] = tuple(t[:40] for t in held[ids[1]])
    assert pool.compact() > 0
    copies()
    used = int((pool.tables(ids)[0] >= 0).sum())
    assert pool.tables(ids)[0].max() < used
    for _ in range(2):
        batch, k, v = step(ids, [1, 1, 1], [[-1]] * 3)
        store(ids, batch, k, v, [[0]] * 3)
    assert torch.isnan(cache.keys[0]).all() and torch.isnan(cache.values[0]).all()
