"""One workspace, sized for the largest step, for steps of fewer rows after it; nothing
behind its end is written."""
import math

import pytest
import torch

from huggingfaceeacp_amd import gemma_q8 as G
from test_gpu_paged_prefix import Prefix
from test_gpu_paged_sparse import Sparse

pytestmark = pytest.mark.gpu

SENTINEL = -7.5
SHAPES = [("f32", 8, 1, 256), ("f16", 32, 8, 128), ("bf16", 4, 4, 64), ("f16", 6, 2, 80)]


def guarded(size):
    whole = torch.full((size // 4 + 4096,), math.nan, device="cuda")
    whole[size // 4:] = SENTINEL
    return whole, whole[:size // 4]


@pytest.mark.parametrize("name,heads,kv_heads,head_dim", SHAPES)
def test_listed_pages(torch_cuda, name, heads, kv_heads, head_dim):
    most = 300
    whole, space = guarded(G.sparse_attention_workspace_bytes(most, heads, kv_heads, head_dim))
    for n in (most, 255, 64, 31, 5, 1):
        call = Sparse(1, name, heads, kv_heads, head_dim, 16, [n], [200], 9)
        call.workspace = space
        call.check(call.call(), (name, n))
        assert (whole[space.numel():] == SENTINEL).all()
        space.fill_(math.nan)


@pytest.mark.parametrize("name,heads,kv_heads,head_dim", SHAPES)
def test_behind_prefixes(torch_cuda, name, heads, kv_heads, head_dim):
    most = 64
    whole, space = guarded(G.prefix_attention_workspace_bytes(most, heads, kv_heads, head_dim))
    for count in (most, 63, 33, 17, 5, 4, 1):
        call = Prefix(torch_cuda, 2, name, heads, kv_heads, head_dim, 16, [1] * count, [130 + s % 7 for s in range(count)],
                      [0, count], [130])
        call.space = space
        for prefixes in (True, False):
            call.check(call.call("causal", prefixes=prefixes), "causal", (name, count, prefixes))
            assert (whole[space.numel():] == SENTINEL).all()
            space.fill_(math.nan)
