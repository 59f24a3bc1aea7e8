"""Selection, bounds and attention over listed pages for more rows than one grid has blocks."""

import pytest
import torch

from huggingfaceeacp_amd import gemma_q8 as G
from paged_helpers import KIND, SENTINEL, ints

pytestmark = pytest.mark.gpu

F16 = torch.float16
ROWS, D = (1 << 24) + 3, 8


def whole(rows, factor, modulus):
    """Rows of small whole numbers, none of them zero."""
    x = torch.arange(rows * D, device="cuda", dtype=torch.int32).mul_(factor).remainder_(modulus)
    return x.sub_(modulus // 2).to(F16).add_(0.5).reshape(rows, D)


def test_select_of_more_rows_than_a_grid_has_blocks(torch_cuda):
    """All rows but the first two choose between two pages."""
    bounds = torch.tensor([[1, -2, 3, 0, 2, -1, 1, 2], [2, 1, -1, 3, -2, 2, 0, -1]], dtype=F16, device="cuda")
    highs = bounds + torch.tensor([0, 1, 2, 1, 0, 1, 3, 0], dtype=F16, device="cuda")
    keys = torch.zeros((2, D), dtype=F16, device="cuda")
    cache = G.PageCache(keys.data_ptr(), keys.data_ptr(), KIND[F16], 1, 2, 1, 1, D)
    held = G.PageCache(bounds.data_ptr(), highs.data_ptr(), KIND[F16], 1, 2, 1, 1, D)
    table, starts = ints([[0, 1]]), ints([0, ROWS])
    batch = G.Sequences(1, ROWS, starts.data_ptr(), None, table.data_ptr(), 2)
    q = whole(ROWS, 37, 23)
    size = G.page_select_workspace_bytes(ROWS, 1, 2)
    workspace = torch.empty(size, dtype=torch.uint8, device="cuda")
    pages = torch.full((ROWS,), -7, dtype=torch.int32, device="cuda")
    G.page_select(cache, 0, batch, held, q.data_ptr(), KIND[F16], D, 1, 0, 1, 1, pages.data_ptr(),
                  workspace.data_ptr(), size)
    x = q.float() # sums of halves far below 2^23: exact
    scores = [torch.maximum(x * bounds[i].float(), x * highs[i].float()).sum(1) for i in range(2)]
    expected = (scores[1] > scores[0]).to(torch.int32)
    expected[0], expected[1] = 0, 1
    assert torch.equal(pages, expected)
    assert 0 < expected.sum().item() < ROWS


def test_bounds_and_listed_rows_of_more_rows_than_a_grid_has_blocks(torch_cuda):
    """Pages of one row, in reverse: their bounds are their keys, and row i attends row i / 2."""
    k, v = whole(ROWS, 41, 251), whole(ROWS, 43, 257)
    cache = G.PageCache(k.data_ptr(), v.data_ptr(), KIND[F16], 1, ROWS, 1, 1, D)
    table = torch.arange(ROWS - 1, -1, -1, dtype=torch.int32, device="cuda")
    starts = ints([0, ROWS])
    batch = G.Sequences(1, ROWS, starts.data_ptr(), None, table.data_ptr(), ROWS)
    lows, highs = torch.full_like(k, SENTINEL), torch.full_like(k, SENTINEL)
    held = G.PageCache(lows.data_ptr(), highs.data_ptr(), KIND[F16], 1, ROWS, 1, 1, D)
    G.page_bounds(cache, 0, batch, held)
    assert torch.equal(lows, k) and torch.equal(highs, k)

    q = whole(ROWS, 37, 23)
    listed = torch.arange(ROWS, dtype=torch.int32, device="cuda") // 2
    out = torch.full_like(q, SENTINEL)
    size = G.sparse_attention_workspace_bytes(ROWS, 1, 1, D)
    workspace = torch.empty(size, dtype=torch.uint8, device="cuda")
    G.sparse_attention(cache, 0, batch, q.data_ptr(), KIND[F16], D, 1, listed.data_ptr(), 1, 0.25, out.data_ptr(), D,
                       workspace.data_ptr(), size)
    expected = v[table[listed.long()].long()].float()
    # the one weight and the output are rounded to fp16, by 2^-11 each; fp32's roundings are below the rest
    assert ((out.float() - expected).abs() <= expected.abs() * (2.0 ** -10 + 2.0 ** -20)).all()
