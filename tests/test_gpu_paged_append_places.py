"""What an append with rotation does with rows whose place is negative, row by row."""
import pytest
import torch

from paged_helpers import SENTINEL
from test_gpu_paged_append_rope import Append

pytestmark = pytest.mark.gpu

PLACES = [1, -1, 0, -5, -2 ** 31, 2]
TAKEN = [0, 2, 5]  # rows whose place is not negative
CACHED = 99        # so cached plus a negative place is a row of the cache, and in the tables


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("given", [False, True])
def test_rows_of_negative_place(torch_cuda, name, given):
    """Without positions they have none and are left out whole; with them their query is
    written.  Neither stores a key or a value."""
    call = Append(torch_cuda, 1, name, 4, 2, 64, 16, [len(PLACES)], [CACHED])
    places = torch.tensor(PLACES, dtype=torch.int32, device="cuda")
    positions = torch.arange(7, 7 + len(PLACES), dtype=torch.int32, device="cuda") if given else None
    q, keys, values = (t.cpu() for t in call.one(positions, places))
    width = call.heads * call.d
    for row in range(len(PLACES)):
        written = (q[row, :width] != SENTINEL).any()
        assert written == (given or row in TAKEN), row
        assert (q[row, width:] == SENTINEL).all()
    stored = {CACHED + PLACES[row] for row in TAKEN}
    for pool in (keys, values):
        assert (pool[0] == SENTINEL).all()
        for slot, page in enumerate(call.host_table[0].tolist()):
            for r in range(16):
                assert (pool[1, page, r] != SENTINEL).any() == (slot * 16 + r in stored), (slot, r)
        for page in set(range(pool.shape[1])) - set(call.host_table[0].tolist()):
            assert (pool[1, page] == SENTINEL).all()
