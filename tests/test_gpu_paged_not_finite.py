"""Values that are not finite in units of keys that every row attends whole."""
import math

import pytest
import torch

from test_gpu_paged_attention import Call
from paged_helpers import assert_near, definition_fast

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name,head_dim", [("f32", 256), ("f32", 64), ("f16", 128), ("bf16", 256)])
@pytest.mark.parametrize("rows", [2, 40])
def test_values_that_are_not_finite_reach_their_channels_alone(torch_cuda, name, head_dim, rows):
    """Every row attends all of the cache: the channels with an infinity or a NaN
    are not finite, all others as if there were none."""
    call = Call(torch_cuda, 41, name, 4, 2, head_dim, 64, [rows], [320])
    held = call.held[0][1].clone()
    for key, channel, value in ((5, 3, math.inf), (70, 9, -math.inf), (200, 11, math.nan),
                                (319, head_dim - 1, math.inf)):
        page = int(call.table[0, key // 64])
        call.cache.values[0, page, key % 64, 0, channel] = value
        held[key, 0, channel] = 0  # for the other channels' expectation
    call.draw_masks(42)
    odd = [3, 9, 11, head_dim - 1]
    rest = [c for c in range(head_dim) if c not in odd]
    q, k, v = call.rows_of(0)
    v = torch.cat([held, v[320:]])
    for how, out in (("causal", call.causal()), ("tree", call.tree())):
        out = out.cpu().reshape(rows, 4, head_dim)
        expected = definition_fast(q, k, v, call.allowed(0, how), call.scale)
        assert not torch.isfinite(out[:, :2][..., odd]).any(), how
        for got, want in ((out[:, :2][..., rest], expected[:, :2][..., rest]), (out[:, 2:], expected[:, 2:])):
            assert_near(got, want, v.abs().max().item(), call.dtype, how)


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
def test_a_key_that_is_not_a_number_reaches_its_head(torch_cuda, name):
    call = Call(torch_cuda, 43, name, 4, 2, 128, 16, [3, 3], [200, 200])
    page = int(call.table[0, 6])
    call.cache.keys[0, page, 1, 1, 5] = math.nan
    out = call.causal().cpu().reshape(2, 3, 4, 128)
    assert torch.isnan(out[0, :, 2:]).all()
    for s, heads in ((0, slice(0, 2)), (1, slice(0, 4))):
        q, k, v = call.rows_of(s)
        k = torch.nan_to_num(k)
        expected = definition_fast(q, k, v, call.allowed(s, "causal"), call.scale)
        assert_near(out[s, :, heads], expected[:, heads], v.abs().max().item(), call.dtype, s)
