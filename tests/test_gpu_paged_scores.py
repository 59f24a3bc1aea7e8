"""The score of a page is the sum of its definition, max(q low, q high) over the channels,
also where one channel's bounds are far larger than everything that is added."""
import math

import pytest
import torch

from test_gpu_paged_select import Select

pytestmark = pytest.mark.gpu

# types of the bounds and the queries; the far channel's query and bound; what whole
# numbers in the others are multiplied by, queries and bounds
FAR = {"bf16_f32": ("bf16", "f32", 1.0, 1e30, 1.0, 1.0), "bf16": ("bf16", "bf16", 1.0, 1e30, 1.0, 1.0),
       "f16_f32": ("f16", "f32", 1e30, 60000.0, 1.0, 1.0),
       "f16": ("f16", "f16", 60000.0, 60000.0, 2.0 ** -14, 2.0 ** -12)}


def whole_numbers(seed, types, heads, kv_heads, head_dim):
    """Whole numbers of up to 8 in all but a channel of each KV head, whose bounds reach from
    zero to where its queries' sign takes the zero: every sum is exact, in any order (whole
    numbers of at most 256 x 64), and so are the ranks."""
    name, q_name, far_q, far_bound, q_unit, unit = FAR[types]
    call = Select(seed, name, q_name, heads, kv_heads, head_dim, 16, [1, 3], [2000, 900])
    g = torch.Generator().manual_seed(seed)
    shape = call.least.shape
    a, b = (torch.randint(-8, 9, shape, generator=g) * unit for _ in range(2))
    q = torch.randint(-8, 9, call.q_host.shape, generator=g) * q_unit
    q = q.reshape(-1, kv_heads, heads // kv_heads, head_dim)
    least, largest = torch.minimum(a, b), torch.maximum(a, b)
    for of in range(kv_heads):
        channel, sign = int(torch.randint(0, head_dim, (1,), generator=g)), (-1.0) ** of
        q[:, of, :, channel] = sign * far_q
        least[:, :, :, of, channel] = -far_bound if sign > 0 else 0.0
        largest[:, :, :, of, channel] = 0.0 if sign > 0 else far_bound
    call.least, call.largest = least.to(call.least.dtype), largest.to(call.largest.dtype)
    call.upload()
    call.q_host = q.reshape(call.q_host.shape).to(call.q_host.dtype)
    call.q.copy_(call.q_host)
    return call


@pytest.mark.parametrize("types", FAR)
@pytest.mark.parametrize("heads,kv_heads,head_dim", [(2, 2, 64), (4, 2, 128), (6, 2, 80), (8, 2, 256), (8, 1, 256),
                                                     (20, 2, 24), (32, 1, 64)])
def test_bounds_of_very_different_size(torch_cuda, types, heads, kv_heads, head_dim):
    call = whole_numbers(1, types, heads, kv_heads, head_dim)
    for first, last, top in ((0, 1, 2), (1, 2, 9), (0, 1, 40)):
        call.check(first, last, top)


def test_small_scores_beside_a_large_bound(torch_cuda):
    """0.5 of one page above the 0.1 of others, behind a bound of 1e30 that adds nothing."""
    call = Select(2, "bf16", "f32", 1, 1, 8, 16, [1], [16 * 40 - 1])
    call.least.zero_()
    call.largest.fill_(0.0)
    call.largest[..., 0] = 0.1
    page = int(call.host_table[0, 23])
    call.least[1, page, 0, 0, 0], call.largest[1, page, 0, 0, 0] = 0.25, 0.5
    call.largest[1, page, 0, 0, 1] = 1e30
    call.upload()
    call.q_host = torch.tensor([[1.0, -1.0, 0, 0, 0, 0, 0, 0]])
    call.q.copy_(call.q_host)
    assert call.call(0, 1, 2).cpu().tolist() == [[[23, 39]]]


@pytest.mark.parametrize("value", [math.inf, -math.inf])
@pytest.mark.parametrize("head_dim", [64, 80])
def test_pages_with_an_infinite_bound_come_first(torch_cuda, value, head_dim):
    """Whether queries take that bound, the other one or neither."""
    call = Select(3, "f16", "f32", 4, 2, head_dim, 16, [1], [1600])
    pools = (call.largest,) if value > 0 else (call.least,)
    call.q_host[:, 5::head_dim] = 0.0  # of all heads
    call.q_host[:, 6::head_dim] = 2.0
    call.q_host[:, 7::head_dim] = -2.0
    call.q.copy_(call.q_host)
    for slot, channel in ((20, 5), (50, 6), (71, 7)):
        for pool in pools:
            pool[1, int(call.host_table[0, slot]), 0, 0, channel] = value
    call.upload()
    for top in (4, 5, 30):
        call.check(0, 1, top)
    assert {20, 50, 71} <= set(call.call(0, 1, 4).cpu()[0, 0].tolist())
