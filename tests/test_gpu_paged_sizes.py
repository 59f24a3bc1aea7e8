"""Calls of more rows or pairs than one grid's threads number."""

import numpy as np
import pytest
import torch

from huggingfaceeacp_amd import gemma_q8 as G
from paged_helpers import KIND, SENTINEL, ints

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def test_append_of_more_rows_than_a_grid_has_waves(torch_cuda):
    """2^26 rows take 2^32 threads: a first sequence of nearly all of them, a second
    that begins before the end of the first launch and ends behind it."""
    rows, page_rows, width = (1 << 26) + 5, 1 << 16, 8
    split = (1 << 26) - 100
    pages = rows // page_rows + 3
    keys = torch.full((1, pages, page_rows, width), SENTINEL, dtype=BF16, device="cuda")
    values = torch.full_like(keys, SENTINEL)
    k = torch.arange(rows * width, device="cuda", dtype=torch.int32).remainder_(251).to(BF16).reshape(rows, width)
    v = -k
    cache = G.PageCache(keys.data_ptr(), values.data_ptr(), KIND[BF16], 1, pages, page_rows, 1, width)
    table = np.full((2, pages), -1, dtype=np.int32)
    used = -(-split // page_rows)
    table[0, :used] = np.arange(used)[::-1]
    table[1, 0] = pages - 1
    table, starts, cached = ints(table), ints([0, split, rows]), ints([0, 7])
    batch = G.Sequences(2, rows, starts.data_ptr(), cached.data_ptr(), table.data_ptr(), pages)
    G.page_append(cache, 0, batch, k.data_ptr(), v.data_ptr(), width)
    for pool, new in ((keys[0], k), (values[0], v)):
        stored = pool[:used].flip(0).reshape(-1, width)
        assert torch.equal(stored[:split], new[:split])
        assert (stored[split:] == SENTINEL).all()
        assert (pool[used:pages - 1] == SENTINEL).all()
        assert torch.equal(pool[pages - 1, 7:7 + rows - split], new[split:])
        assert (pool[pages - 1, :7] == SENTINEL).all() and (pool[pages - 1, 7 + rows - split:] == SENTINEL).all()


def test_norms_of_more_rows_than_a_grid_has_blocks(torch_cuda):
    """Rows of three heads of 8 take a block each."""
    rows, d = (1 << 24) + 3, 8
    x = torch.empty((rows, 3 * d), dtype=BF16, device="cuda")
    x.copy_(torch.arange(1, 12346, device="cuda").repeat(rows * 3 * d // 12345 + 1)[:rows * 3 * d].reshape(
        rows, 3 * d).remainder(97) - 48)
    q, k, v = (torch.full((rows, d), SENTINEL, dtype=BF16, device="cuda") for _ in range(3))
    positions = torch.arange(rows, device="cuda", dtype=torch.int32).remainder_(31)
    cos, sin = (torch.from_numpy(t).cuda() for t in G.rotary_table_host(31, d))

    def call(first, count, q, k, v):
        G.head_norm_rope(x[first:].data_ptr(), KIND[BF16], count, 3 * d, 1, 1, d, None, None, 1e-6,
                         positions[first:].data_ptr(), cos.data_ptr(), sin.data_ptr(), 31, q.data_ptr(),
                         KIND[BF16], d, k.data_ptr(), v.data_ptr(), KIND[BF16], d)

    call(0, rows, q, k, v)
    # the same rows in calls of one launch
    first = 0
    while first < rows:
        count = min(1 << 22, rows - first)
        parts = [torch.full((count, d), SENTINEL, dtype=BF16, device="cuda") for _ in range(3)]
        call(first, count, *parts)
        for whole, part in zip((q, k, v), parts):
            assert torch.equal(whole[first:first + count], part)
        first += count
    assert torch.equal(v, x[:, 2 * d:])


def test_copies_of_more_pages_than_a_grid_has_blocks(torch_cuda):
    count, width = (1 << 24) + 3, 8
    keys = torch.arange(2 * count * width, device="cuda", dtype=torch.int32).remainder_(253).to(BF16).reshape(
        1, 2 * count, 1, width)
    values = -keys
    cache = G.PageCache(keys.data_ptr(), values.data_ptr(), KIND[BF16], 1, 2 * count, 1, 1, width)
    pairs = torch.stack([torch.arange(count, device="cuda"), 2 * count - 1 - torch.arange(count, device="cuda")],
                        1).to(torch.int32).contiguous()
    expected = [torch.cat([t[:, :count], t[:, :count].flip(1)], 1) for t in (keys, values)]
    G.page_copy(cache, pairs.data_ptr(), count)
    assert torch.equal(keys, expected[0]) and torch.equal(values, expected[1])
