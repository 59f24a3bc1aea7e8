"""Scores that are large and close to each other, all exact in fp32: the weights are
those of their differences, in whichever unit, workgroup or order the keys come."""

import numpy as np
import pytest
import torch

from huggingfaceeacp_amd import gemma_q8 as G
from paged_helpers import KIND, TYPES, Cache, definition_fast, half_step, ints, kv_type

pytestmark = pytest.mark.gpu

HEADS, HEAD_DIM, PAGE_ROWS, KEYS = 4, 64, 16, 300
# (first channel of the query, of the keys, the query's second channel): scores of
# +- the product of the first two plus 0 .. 6 times the third.  In powers of two
# those of 5e4 lie on both sides of 2^16, where the reference's rounding is taken
# account of.
SIZES = {"1e2": (8, 12, 0.5), "5e4": (272, 167, 1), "2e5": (512, 384, 0.5), "5e6": (2048, 2560, 0.5), "1e8": (8192, 12288, 8),
         "2e8": (16384, 12288, 16)}


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("size", list(SIZES))
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("sequences,rows", [(1, 1), (300, 1), (1, 20), (120, 20)])
def test_differences_of_large_scores(torch_cuda, name, size, sign, sequences, rows):
    dtype, kv = TYPES[name], kv_type(name)
    g = torch.Generator().manual_seed(51)
    a, b, step = SIZES[size]
    steps = torch.randint(0, 6, (KEYS,), generator=g)
    steps[[10, 70, 150, 290]] = torch.tensor([5, 6, 4, 6])
    pages = -(-KEYS // PAGE_ROWS)
    cache = Cache(kv, 1, pages, PAGE_ROWS, 1, HEAD_DIM)
    keys = torch.zeros((pages * PAGE_ROWS, 1, HEAD_DIM), dtype=kv)
    keys[:KEYS, 0, 0], keys[:KEYS, 0, 1] = sign * b, steps.to(kv)
    keys[:KEYS, 0, 2] = torch.randn(KEYS, generator=g).to(kv)
    values = torch.randn((pages * PAGE_ROWS, 1, HEAD_DIM), generator=g).to(kv)
    cache.keys.copy_(keys.reshape(cache.keys.shape))
    cache.values.copy_(values.reshape(cache.values.shape))
    # heads 1 and 3 have small scores: large and small rows lie in one wave
    q = torch.zeros((rows, HEADS, HEAD_DIM), dtype=dtype)
    q[:, ::2, 0], q[:, ::2, 1] = a, step
    q[:, 1::2, 2] = torch.randn((rows, 2), generator=g).to(dtype)
    total = sequences * rows
    dq = q.repeat(sequences, 1, 1).cuda()
    own = torch.zeros((total, HEAD_DIM), dtype=kv, device="cuda")
    masks = torch.zeros((total, 1), dtype=torch.int64, device="cuda")
    starts, cached = ints(np.arange(sequences + 1) * rows), ints(np.full(sequences, KEYS))
    table = ints(np.tile(np.arange(pages), (sequences, 1)))
    batch = G.Sequences(sequences, total, starts.data_ptr(), cached.data_ptr(), table.data_ptr(), pages)
    size_of = G.packed_attention_workspace_bytes(HEADS, 1, HEAD_DIM)
    workspace = torch.empty(size_of, dtype=torch.uint8, device="cuda")
    out = torch.zeros_like(dq)
    G.tree_attention(cache.c, 0, batch, dq.data_ptr(), KIND[dtype], HEADS * HEAD_DIM, HEADS, own.data_ptr(),
                     own.data_ptr(), HEAD_DIM, masks.data_ptr(), 1, 1.0, out.data_ptr(), HEADS * HEAD_DIM,
                     workspace.data_ptr(), size_of)
    seen = torch.ones((rows, KEYS), dtype=torch.bool)
    expected = definition_fast(q, keys[:KEYS], values[:KEYS], seen, 1.0).repeat(sequences, 1, 1)
    # The scores are exact, and their differences too.  A weight: half a step of its
    # type (fp32: two fp16 pieces, 2^-22), and of the output's; the exponents of the
    # weights that count (up to 25) are off by 2^-22 of themselves, the scale's and
    # the product's rounding, as are small rows' scores of up to 12; sums and factors
    # between references 2^-20.
    weight = half_step(kv) if name != "f32" else 2.0 ** -22
    bound = (weight + half_step(dtype) + 25 * 2.0 ** -22 + 2.0 ** -20) * values.abs().max().item()
    worst = ((out.double().cpu() - expected).abs().max() / bound).item()
    assert worst <= 1, worst
