"""What the appends with rotation, the prefixes, the bounds, the selection and the
attention over selected pages refuse on the host, and the pool's groups (no GPU
needed: a refused call launches nothing)."""
import ctypes

import numpy as np
import pytest

from huggingfaceeacp_amd import gemma_q8 as G
from test_page_pool import BF16, F16, F32, PTR, cache, refused, sequences


def bounds(**change):
    return cache(**{**dict(page_rows=1), **change})


CACHES = (dict(type=F32), dict(layers=0), dict(page_rows=12), dict(pages=-1), dict(head_dim=12),
          dict(head_dim=264), dict(kv_heads=0), dict(pages=1 << 28, page_rows=16))
SEQUENCES = (dict(sequences=-1), dict(rows=-1), dict(starts=None), dict(page_table=None), dict(table_width=0))


def call(function, values, c=None, s=None, **change):
    a = {**values, **change}
    return function(c or cache(), a.pop("layer"), s or sequences(), *a.values())


APPEND = dict(layer=0, x=PTR, x_type=F32, x_stride=512, heads=4, q_weight=PTR, k_weight=PTR, epsilon=1e-6,
              positions=None, cosines=PTR, sines=PTR, max_positions=10, places=None, q=PTR, q_type=F32,
              q_stride=256)
SELECT = dict(layer=0, bounds=None, q=PTR, q_type=F16, q_stride=256, heads=4, first=1, last=2, top=8, pages=PTR,
              workspace=PTR, size=1 << 30)
SPARSE = dict(layer=0, q=PTR, q_type=F16, q_stride=256, heads=4, pages=PTR, top=8, scale=1.0, out=PTR,
              out_stride=256, workspace=PTR, size=1 << 30)
PREFIX = dict(layer=0, prefixes=None, q=PTR, q_type=F16, q_stride=256, heads=4, k=PTR, v=PTR, kv_stride=128,
              ancestors=None, words=0, scale=1.0, out=PTR, out_stride=256, workspace=PTR, size=1 << 30)


def everything():
    select = {**SELECT, "bounds": bounds()}
    prefix = {**PREFIX, "prefixes": G.Prefixes(1, PTR, PTR)}
    yield lambda **a: call(G.page_append_rope, APPEND, **a)
    yield lambda **a: call(G.page_bounds, dict(layer=0, bounds=bounds(), taken=None), **a)
    yield lambda **a: call(G.page_select, select, **a)
    yield lambda **a: call(G.sparse_attention, SPARSE, **a)
    yield lambda **a: call(G.prefix_attention, prefix, **a)


def test_caches_and_sequences():
    for function in everything():
        for change in CACHES:
            refused(G.ERR_SHAPE, lambda: function(c=cache(**change)))
        for change in (dict(keys=None), dict(values=PTR + 2)):
            refused(G.ERR_ARGUMENT, lambda: function(c=cache(**change)))
        for change in SEQUENCES:
            refused(G.ERR_ARGUMENT, lambda: function(s=sequences(**change)))
        refused(G.ERR_SHAPE, lambda: function(s=sequences(table_width=1 << 28)))
        refused(G.ERR_SHAPE, lambda: function(s=sequences(rows=(1 << 30) + 1)))
        for layer in (-1, 2):
            refused(G.ERR_ARGUMENT, lambda: function(layer=layer))
        assert function(s=sequences(rows=0)) == G.OK  # nothing to do is no refusal
        assert function(s=sequences(sequences=0)) == G.OK


def test_append_rope_refusals():
    append = lambda **a: call(G.page_append_rope, APPEND, **a)
    for change in (dict(x_type=2), dict(q_type=0), dict(heads=5), dict(heads=66), dict(heads=0)):
        refused(G.ERR_SHAPE, lambda: append(**change))
    for change in (dict(x=None), dict(x=PTR + 8), dict(x_stride=508), dict(x_stride=510), dict(q=None),
                   dict(q=PTR + 4), dict(q_stride=252), dict(cosines=None), dict(sines=PTR + 4),
                   dict(max_positions=0), dict(epsilon=float("nan")), dict(epsilon=-1.0), dict(q_weight=PTR + 4),
                   dict(c=cache(pages=0)), dict(s=sequences(page_table=None, cached=None))):
        refused(G.ERR_ARGUMENT, lambda: append(**change))


def test_bounds_and_select_refusals():
    for function, values in ((G.page_bounds, dict(layer=0, bounds=bounds(), taken=None)),
                             (G.page_select, {**SELECT, "bounds": bounds()})):
        for other in (cache(), bounds(type=BF16), bounds(layers=1), bounds(pages=3), bounds(kv_heads=1),
                      bounds(head_dim=128), bounds(page_rows=2)):
            refused(G.ERR_SHAPE, lambda: call(function, values, bounds=other))
        refused(G.ERR_ARGUMENT, lambda: call(function, values, bounds=bounds(keys=None)))
        for change in (dict(c=cache(pages=0), bounds=bounds(pages=0)),
                       dict(s=sequences(page_table=None, cached=None))):
            refused(G.ERR_ARGUMENT, lambda: call(function, values, **change))
    select = lambda **a: call(G.page_select, {**SELECT, "bounds": bounds()}, **a)
    for change in (dict(heads=3), dict(heads=66), dict(q_type=BF16), dict(q_type=1), dict(first=-1), dict(last=0),
                   dict(top=2), dict(top=0), dict(top=-5), dict(first=2 ** 31 - 1, last=2 ** 31 - 1),
                   dict(top=1 << 27)):
        refused(G.ERR_SHAPE, lambda: select(**change))
    for change in (dict(q=None), dict(q=PTR + 8), dict(q_stride=248), dict(q_stride=260), dict(pages=None),
                   dict(pages=PTR + 4), dict(workspace=None), dict(workspace=PTR + 4), dict(size=100)):
        refused(G.ERR_ARGUMENT, lambda: select(**change))
    assert G.page_select_workspace_bytes(5, 2, 100) >= 4 * 5 * 2 * 100
    for sizes in ((-1, 1, 1), (1, 0, 1), (1, 1, -1), ((1 << 30) + 1, 1, 1)):
        assert G.page_select_workspace_bytes(*sizes) == 0


def test_attention_refusals():
    prefix = {**PREFIX, "prefixes": G.Prefixes(1, PTR, PTR)}
    for function, values in ((G.sparse_attention, SPARSE), (G.prefix_attention, prefix)):
        run = lambda **a: call(function, values, **a)
        for change in (dict(heads=3), dict(heads=66), dict(heads=0), dict(q_type=BF16), dict(q_type=1),
                       dict(c=cache(type=BF16), q_type=F32)):
            refused(G.ERR_SHAPE, lambda: run(**change))
        for change in (dict(q=None), dict(q=PTR + 8), dict(out=None), dict(workspace=None), dict(q_stride=248),
                       dict(q_stride=260), dict(out_stride=8), dict(scale=float("nan")),
                       dict(scale=float("inf")), dict(size=100)):
            refused(G.ERR_ARGUMENT, lambda: run(**change))
    sparse = lambda **a: call(G.sparse_attention, SPARSE, **a)
    for change in (dict(pages=None), dict(pages=PTR + 4), dict(c=cache(pages=0)),
                   dict(s=sequences(page_table=None, cached=None))):
        refused(G.ERR_ARGUMENT, lambda: sparse(**change))
    for top in (0, -1, 1 << 27):
        refused(G.ERR_SHAPE, lambda: sparse(top=top))
    run = lambda **a: call(G.prefix_attention, prefix, **a)
    for change in (dict(k=None), dict(v=None), dict(k=PTR + 2), dict(kv_stride=120), dict(kv_stride=132),
                   dict(ancestors=PTR, words=0), dict(ancestors=PTR, words=1025),
                   dict(prefixes=G.Prefixes(-1, PTR, PTR)), dict(prefixes=G.Prefixes(1, None, PTR)),
                   dict(prefixes=G.Prefixes(1, PTR, None)), dict(s=sequences(cached=None))):
        refused(G.ERR_ARGUMENT, lambda: run(**change))
    for change in (dict(kv_stride=(1 << 26) + 8), dict(prefixes=G.Prefixes(4, PTR, PTR))):
        refused(G.ERR_SHAPE, lambda: run(**change))
    for size in (G.sparse_attention_workspace_bytes, G.prefix_attention_workspace_bytes):
        assert size(1, 8, 3, 64) == 0 and size(-1, 8, 1, 64) == 0 and size((1 << 30) + 1, 8, 1, 64) == 0
        assert size(16, 8, 1, 256) > 0
    assert ctypes.sizeof(G.Prefixes) == 24


def test_groups_of_a_pool():
    pool = G.PagePool(40, 4, 8, 10)
    a, alone = pool.open(), pool.open()
    pool.extend(a, 18)
    pool.extend(alone, 9)
    b, c = pool.fork(a), pool.fork(a)
    first, rows = pool.prefixes([a, b, c, alone])  # nothing written since: the part of a page counts
    assert first.tolist() == [0, 3, 4] and rows.tolist() == [18, 0]
    pool.extend(b, 1)  # its own copy of the last page
    first, rows = pool.prefixes([a, b, c, alone])
    assert first.tolist() == [0, 3, 4] and rows.tolist() == [16, 0]
    pool.truncate(c, 5)
    assert [x.tolist() for x in pool.prefixes([a, b, c])] == [[0, 3], [5]]
    assert [x.tolist() for x in pool.prefixes([a, b, c], least=6)] == [[0, 2, 3], [16, 0]]
    assert [x.tolist() for x in pool.prefixes([a, alone, b])] == [[0, 1, 2, 3], [0, 0, 0]]
    assert [x.tolist() for x in pool.prefixes([])] == [[0], []]
    assert [x.tolist() for x in pool.prefixes([b])] == [[0, 1], [0]]
    d = pool.fork(alone)
    assert [x.tolist() for x in pool.prefixes([alone, d, a, b], 9)] == [[0, 2, 4], [9, 16]]
    for bad in (lambda: pool.prefixes([a, 7]), lambda: pool.prefixes([a], least=0), lambda: pool.prefixes([-1])):
        refused(G.ERR_ARGUMENT, bad)
    refused(G.ERR_ARGUMENT, lambda: G.check(G.library().gq8_page_pool_prefixes(None, None, 0, 1, PTR, None)))


@pytest.mark.parametrize("seed", range(4))
def test_groups_against_the_tables(seed):
    """Over forks, extensions and truncations: the rows of a group are in the same pages
    for all of it, one more page is not, and neighbours that share are in one group."""
    rng = np.random.default_rng(seed)
    pool = G.PagePool(300, 8, 12, 20)
    open_ids = [pool.open()]
    pool.extend(open_ids[0], 40)
    for _ in range(60):
        s = int(rng.choice(open_ids))
        action = rng.integers(0, 4)
        if action == 0 and len(open_ids) < 12:
            open_ids.append(pool.fork(s))
        elif action == 1 and pool.rows(s) < 130:
            pool.extend(s, int(rng.integers(1, 20)))
        elif action == 2:
            pool.truncate(s, int(rng.integers(pool.rows(s) // 2, pool.rows(s) + 1)))
        elif len(open_ids) > 4:
            pool.close(s)
            open_ids.remove(s)
    order = rng.permutation(open_ids)
    table, held = pool.tables(order)
    first, rows = pool.prefixes(order)
    assert first[0] == 0 and first[-1] == len(order) and (np.diff(first) > 0).all()

    def common(a, b):
        same = 0
        while same < table.shape[1] and table[a, same] == table[b, same] >= 0:
            same += 1
        return min(same * 8, held[a], held[b])

    for i, n in enumerate(rows):
        a, b = first[i], first[i + 1]
        assert n == (min(common(a, s) for s in range(a + 1, b)) if b - a > 1 else 0)
        assert b - a == 1 or n >= 1
        assert b == len(order) or common(a, b) == 0
