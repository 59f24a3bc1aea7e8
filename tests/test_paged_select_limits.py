"""Numbers of pages at the ends of their type are refused on the host (no GPU needed: a
refused call launches nothing)."""
import pytest

from huggingfaceeacp_amd import gemma_q8 as G
from test_page_pool import refused
from test_paged_streams_refusals import SELECT, bounds, call

MOST, LEAST = 2 ** 31 - 1, -2 ** 31


@pytest.mark.parametrize("first,last,top", [(0, MOST, -5), (0, 1, LEAST), (0, MOST, LEAST), (1, MOST, -1), (0, MOST, 0),
                                            (MOST, 1, LEAST), (LEAST, 1, 8), (0, LEAST, 8), (MOST, MOST, MOST),
                                            (0, 1, 0), (0, 9, 8), (8, 1, 8)])
def test_pages_to_take(first, last, top):
    refused(G.ERR_SHAPE, lambda: call(G.page_select, {**SELECT, "bounds": bounds()}, first=first, last=last, top=top))
