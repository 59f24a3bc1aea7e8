"""How the norms and rotation round to 16 bits: of four neighbours the first through
fp32, the others once, in every kernel that makes them."""
import pytest
import torch

from huggingfaceeacp_amd import gemma_q8 as G
from paged_helpers import KIND, TYPES, ints, normal
from test_gpu_paged_rows import EPSILON, norm_rope_definition, tables

pytestmark = pytest.mark.gpu

ROWS, HEADS, D, WINDOW = 8000, 8, 64, 500


@pytest.mark.parametrize("name", ["f16", "bf16"])
def test_roundings(torch_cuda, name):
    g = torch.Generator().manual_seed(1)
    dtype = TYPES[name]
    x = normal(g, (ROWS, (HEADS + 2) * D), dtype, 3.0).cuda()
    weights = [normal(g, (D,), torch.float32, 0.3).cuda() for _ in range(2)]
    cos, sin = (t.cuda() for t in tables(WINDOW, D))
    positions = ints([i % WINDOW for i in range(ROWS)])
    q = torch.empty((ROWS, HEADS * D), dtype=dtype, device="cuda")
    k, v = (torch.empty((ROWS, D), dtype=dtype, device="cuda") for _ in range(2))
    kind = KIND[dtype]
    G.head_norm_rope(x.data_ptr(), kind, ROWS, (HEADS + 2) * D, HEADS, 1, D, weights[0].data_ptr(),
                     weights[1].data_ptr(), EPSILON, positions.data_ptr(), cos.data_ptr(), sin.data_ptr(), WINDOW,
                     q.data_ptr(), kind, HEADS * D, k.data_ptr(), v.data_ptr(), kind, D)
    at = positions.long()
    for got, first, weight in ((q.reshape(ROWS, HEADS, D), 0, weights[0]), (k.reshape(ROWS, 1, D), HEADS, weights[1])):
        heads = x.reshape(ROWS, HEADS + 2, D)[:, first:first + got.shape[1]]
        exact = norm_rope_definition(heads, weight, cos[at], sin[at])
        # Both sides' doubles are off by some 20 roundings of 2^-53, relative to the larger of
        # a rotation's two products: far below 2^-45 of the values, of which sums that cancel
        # to less than 2^-6 of the head's largest are left out.
        slack = 2.0 ** -45 * exact.abs()
        clear = exact.abs() > 2.0 ** -6 * exact.abs().amax(-1, keepdim=True)
        bits, y = got.view(torch.int16), got.double()
        off = (y - exact).abs()
        nearer = sum(((bits + step).view(dtype).double() - exact).abs() < off - 2 * slack for step in (1, -1))
        through = [(exact + sign * slack).float().to(dtype) for sign in (1, -1)]
        one, two = (clear & (torch.arange(D, device="cuda") % 4 != 0)), (clear & (torch.arange(D, device="cuda") % 4 == 0))
        assert not (nearer.bool() & one).any()
        settled = through[0] == through[1]
        assert torch.equal(got[two & settled], through[0][two & settled])
        if first == 0: # roundings through fp32 that the nearest would not be
            assert (one & settled & (got != through[0])).any()
            assert (two & nearer.bool()).any() or name == "bf16"
