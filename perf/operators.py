"""The operators of a paged cache that many sequences share, as timed cases: the
norms and rotation of a step's queries and keys, the cache's appends and page
copies, causal attention over packed prompts, and attention of drafted trees
(single tokens among them) over the cache.

Sequences are packed: sequence s owns the rows starts[s] .. starts[s + 1] - 1 of
the packed tensors, behind cached[s] rows that lie in the pages its row of the
page table names.  `run` is one call of one operator: in plain torch where `own`
is false, through huggingfaceeacp_amd where it is true.  Lengths and the shape
of the drafted trees come from the case; values, pages and positions from the
seed.
"""
import math
import random

import torch

own = False

EPSILON, THETA = 1e-6, 10000.0
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
# the heads that the repository's decoder has (8 query heads of 256 over one),
# and generic ones: grouped, as many keys' heads as queries', odd groups
HEADS = [(8, 1, 256), (8, 1, 256), (32, 8, 128), (16, 16, 64), (12, 4, 80), (6, 2, 256), (7, 7, 96)]


def listed():
    return [
        # one decoded token's fused q|k|v row: the smallest call
        {"name": "norm_rope_1", "op": "norm_rope", "type": "f32", "heads": 8, "kv_heads": 1,
         "head_dim": 256, "rows": 1},
        # a prompt block of grouped heads in bf16
        {"name": "norm_rope_2048_bf16", "op": "norm_rope", "type": "bf16", "heads": 32,
         "kv_heads": 8, "head_dim": 128, "rows": 2048},
        # the accepted paths of 16 drafted trees go into the cache
        {"name": "append_accepted_16", "op": "append", "type": "f16", "kv_heads": 1,
         "head_dim": 256, "page_rows": 16, "sequences": 16, "rows_low": 8, "rows_high": 32,
         "cached_low": 100, "cached_high": 1100, "accept": True, "spread": 3},
        # a batch of ragged prompts goes into the cache
        {"name": "append_prompts_16", "op": "append", "type": "f16", "kv_heads": 1,
         "head_dim": 256, "page_rows": 64, "sequences": 16, "rows_low": 64, "rows_high": 1024,
         "cached_low": 0, "cached_high": 700, "accept": False, "spread": 4},
        # sixteen forks write: their shared last pages are copied in all layers
        {"name": "copy_forked_16", "op": "copy", "type": "f16", "kv_heads": 1, "head_dim": 256,
         "page_rows": 16, "layers": 18, "pages": 400, "count": 16},
        # a compaction moves most of what a long conversation holds
        {"name": "copy_compacted_500", "op": "copy", "type": "f16", "kv_heads": 1,
         "head_dim": 256, "page_rows": 16, "layers": 18, "pages": 1100, "count": 500},
        # a prompt of 2048 tokens at the decoder's heads and types
        {"name": "packed_2048", "op": "packed", "type": "f32", "heads": 8, "kv_heads": 1,
         "head_dim": 256, "page_rows": 64, "sequences": 1, "rows_low": 2048, "rows_high": 2048,
         "cached_low": 0, "cached_high": 0, "spread": 0},
        # ragged prompts of a batch, some behind cached turns, grouped heads
        {"name": "packed_ragged_16_f16", "op": "packed", "type": "f16", "heads": 32, "kv_heads": 8,
         "head_dim": 128, "page_rows": 32, "sequences": 16, "rows_low": 33, "rows_high": 1024,
         "cached_low": 0, "cached_high": 1000, "spread": 5},
        # a whole window in bf16
        {"name": "packed_8192_bf16", "op": "packed", "type": "bf16", "heads": 8, "kv_heads": 1,
         "head_dim": 256, "page_rows": 64, "sequences": 1, "rows_low": 8192, "rows_high": 8192,
         "cached_low": 0, "cached_high": 0, "spread": 0},
        # one token of one sequence after a 512-token prompt
        {"name": "tree_1x1_512", "op": "tree", "type": "f32", "heads": 8, "kv_heads": 1,
         "head_dim": 256, "page_rows": 16, "sequences": 1, "rows_low": 1, "rows_high": 1,
         "cached_low": 512, "cached_high": 512, "spread": 0},
        # one token each of 16 sequences around 1024 tokens
        {"name": "tree_16x1_1024", "op": "tree", "type": "f32", "heads": 8, "kv_heads": 1,
         "head_dim": 256, "page_rows": 16, "sequences": 16, "rows_low": 1, "rows_high": 1,
         "cached_low": 900, "cached_high": 1150, "spread": 6},
        # drafted trees over long conversations, grouped heads
        {"name": "tree_8x32_f16", "op": "tree", "type": "f16", "heads": 32, "kv_heads": 8,
         "head_dim": 128, "page_rows": 32, "sequences": 8, "rows_low": 16, "rows_high": 48,
         "cached_low": 1000, "cached_high": 8000, "spread": 7},
    ]


def _spread(rng, low, high):
    """A whole number spread over the logarithm of [low, high]."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng):
    op = rng.choice(["norm_rope", "append", "copy", "packed", "packed", "packed", "tree", "tree", "tree"])
    heads, kv_heads, head_dim = rng.choice(HEADS)
    case = {"op": op, "type": rng.choice(["f32", "f16", "bf16"]), "kv_heads": kv_heads,
            "head_dim": head_dim}
    if op in ("norm_rope", "packed", "tree"):
        case["heads"] = heads
    if op == "norm_rope":
        return {**case, "rows": _spread(rng, 1, 4096)}
    case["page_rows"] = rng.choice([8, 16, 16, 32, 64, 128])
    if op == "copy":
        case["type"] = rng.choice(["f16", "bf16"])
        pages = _spread(rng, 8, 16384 // case["page_rows"])
        return {**case, "layers": rng.randint(1, 18), "pages": pages,
                "count": rng.randint(1, pages // 2)}
    sequences = _spread(rng, 1, 32)
    case.update(sequences=sequences, spread=rng.randrange(1 << 20))
    if op == "append":
        case["type"] = rng.choice(["f16", "bf16"])
        high = _spread(rng, 1, 1024)
        return {**case, "rows_low": rng.randint(0, high), "rows_high": high,
                "cached_low": 0, "cached_high": rng.randint(0, 1024), "accept": rng.random() < 0.5}
    if op == "packed":
        # the scores of the padded batch stay below those of one whole window
        most = max(64, int(math.sqrt(8 * 4096 * 4096 / (sequences * heads) / 2)))
        high = _spread(rng, 16, min(4096, most))
        return {**case, "rows_low": rng.randint(0, high), "rows_high": high,
                "cached_low": 0, "cached_high": rng.choice([0, rng.randint(0, min(4096, most))])}
    high = rng.choice([1, 1, _spread(rng, 2, 64)])
    cached = _spread(rng, 1, 8100)
    return {**case, "rows_low": rng.randint(1, high), "rows_high": high,
            "cached_low": rng.randint(0, cached), "cached_high": cached}


# ---- what the case fixes: lengths and trees -----------------------------------
def _lengths(case):
    """(rows, cached) of each sequence."""
    rng = random.Random(case["spread"])
    rows = [rng.randint(case["rows_low"], case["rows_high"]) for _ in range(case["sequences"])]
    cached = [rng.randint(case["cached_low"], case["cached_high"]) for _ in rows]
    rows[-1] = max(rows[-1], 1)
    return rows, cached


def _parents(case):
    """The parent of each drafted node in its sequence, -1 for the first."""
    rng = random.Random(case["spread"] + 1)
    return [[-1] + [rng.randint(max(0, (i - 1) // 4), i - 1) for i in range(1, n)] if n else []
            for n in _lengths(case)[0]]


def _depths(parents):
    depths = []
    for parent in parents:
        depths.append(1 + (depths[parent] if parent >= 0 else 0))
    return depths


def _accepted(case):
    """The place among the appended rows of each row, -1 for one not taken:
    of a drafted tree the path to its last node."""
    places = []
    for parents in _parents(case):
        place = [-1] * len(parents)
        node = len(parents) - 1
        depths = _depths(parents)
        while node >= 0:
            place[node] = depths[node] - 1
            node = parents[node]
        places += place
    return places


def work(case):
    g, d = case["kv_heads"], case["head_dim"]
    if case["op"] == "norm_rope":
        h, rows, e = case["heads"], case["rows"], SIZE[case["type"]]
        read = rows * ((h + 2 * g) * d * e + 4 + d * 4) + 2 * d * 4
        return {"bytes": read + rows * (h * d * e + 2 * g * d * 2), "flops": 7 * rows * (h + g) * d}
    if case["op"] == "copy":
        return {"bytes": 4 * case["count"] * case["layers"] * case["page_rows"] * g * d * 2, "flops": 0}
    rows, cached = _lengths(case)
    if case["op"] == "append":
        taken = sum(p >= 0 for p in _accepted(case)) if case["accept"] else sum(rows)
        return {"bytes": 4 * taken * g * d * 2 + 4 * sum(rows), "flops": 0}
    h, e = case["heads"], SIZE[case["type"]]
    if case["op"] == "packed":
        pairs = sum(n * c + n * (n + 1) // 2 for n, c in zip(rows, cached))
    else:
        pairs = sum(n * c + sum(_depths(p)) for n, c, p in zip(rows, cached, _parents(case)))
    moved = 2 * sum(rows) * h * d * e + 2 * (sum(rows) + sum(c for n, c in zip(rows, cached) if n)) * g * d * 2
    return {"bytes": moved, "flops": 4 * h * d * pairs}


# ---- inputs -------------------------------------------------------------------
def _generator(seed):
    generator = torch.Generator(device="cuda")
    generator.manual_seed(int(seed))
    return generator


def _normal(generator, shape, dtype, sigma=1.0):
    return (torch.randn(shape, generator=generator, device="cuda") * sigma).to(dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _kv_type(case):
    return TYPES["bf16" if case["type"] == "bf16" else "f16"]


def prepare(case, seed):
    gen = _generator(seed)
    g, d, kv_type = case["kv_heads"], case["head_dim"], _kv_type(case)
    s = {"case": case}
    if case["op"] == "norm_rope":
        h, rows, dtype = case["heads"], case["rows"], TYPES[case["type"]]
        window = 8192
        angles = torch.arange(window, device="cuda", dtype=torch.float64)[:, None] * THETA ** (
            -torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d)
        s.update(x=_normal(gen, (rows, (h + 2 * g) * d), dtype, 2.0),
                 q_weight=_normal(gen, (d,), torch.float32, 0.3),
                 k_weight=_normal(gen, (d,), torch.float32, 0.3),
                 cos=angles.cos().float(), sin=angles.sin().float(),
                 positions=torch.randint(0, window, (rows,), generator=gen, device="cuda",
                                         dtype=torch.int32),
                 q=torch.zeros((rows, h, d), dtype=dtype, device="cuda"),
                 k=torch.zeros((rows, g, d), dtype=kv_type, device="cuda"),
                 v=torch.zeros((rows, g, d), dtype=kv_type, device="cuda"))
        return s
    page_rows = case["page_rows"]
    if case["op"] == "copy":
        pages, layers = case["pages"], case["layers"]
        order = torch.randperm(pages, generator=gen, device="cuda")[:2 * case["count"]]
        s["pairs"] = order.reshape(-1, 2).to(torch.int32).contiguous()
    else:
        layers = 1
        rows, cached = _lengths(case)
        starts = [0]
        for n in rows:
            starts.append(starts[-1] + n)
        widths = [-(-(n + c) // page_rows) for n, c in zip(rows, cached)]
        width = max(1, max(widths))
        pages = max(1, sum(widths)) + 3
        # every sequence's pages lie anywhere in the pool; entries past them are -1
        order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
        table = torch.full((len(rows), width), -1, dtype=torch.int32, device="cuda")
        first = 0
        for i, w in enumerate(widths):
            table[i, :w] = order[first:first + w]
            first += w
        s.update(starts=_ints(starts), cached=_ints(cached), table=table,
                 most_rows=max(rows), most_cached=max(cached),
                 k=_normal(gen, (starts[-1], g, d), kv_type), v=_normal(gen, (starts[-1], g, d), kv_type))
        if case["op"] == "append":
            s["places"] = _ints(_accepted(case)) if case["accept"] else None
        else:
            s.update(q=_normal(gen, (starts[-1], case["heads"], d), TYPES[case["type"]], 1.5),
                     out=torch.zeros((starts[-1], case["heads"], d), dtype=TYPES[case["type"]],
                                     device="cuda"))
        if case["op"] == "tree":
            masks = []
            for parents in _parents(case):
                mask = []
                for i, parent in enumerate(parents):
                    mask.append((1 << i) | (mask[parent] if parent >= 0 else 0))
                masks += mask
            s["ancestors"] = torch.tensor([m - (1 << 64) if m >> 63 else m for m in masks],
                                          dtype=torch.int64, device="cuda")
    s["keys"] = _normal(gen, (layers, pages, page_rows, g, d), kv_type)
    s["values"] = _normal(gen, (layers, pages, page_rows, g, d), kv_type)
    if own:
        _plan(s)
    return s


# ---- the framework's operators -------------------------------------------------
def _plan(s):
    """What a program keeps between calls: the cache's and the batch's
    descriptions and the attention's workspace."""
    from huggingfaceeacp_amd import gemma_q8 as G
    case = s["case"]
    layers, pages, page_rows, g, d = s["keys"].shape
    kind = G.DTYPES.index("BF16" if s["keys"].dtype == torch.bfloat16 else "F16")
    s["cache"] = G.PageCache(s["keys"].data_ptr(), s["values"].data_ptr(), kind, layers, pages,
                             page_rows, g, d)
    if case["op"] != "copy":
        s["batch"] = G.Sequences(len(s["cached"]), len(s["k"]), s["starts"].data_ptr(),
                                 s["cached"].data_ptr(), s["table"].data_ptr(), s["table"].shape[1])
    if case["op"] in ("packed", "tree"):
        size = G.packed_attention_workspace_bytes(case["heads"], g, d)
        s["workspace"] = torch.empty(size, dtype=torch.uint8, device="cuda")


def _run_own(s):
    from huggingfaceeacp_amd import gemma_q8 as G
    case = s["case"]
    stream = torch.cuda.current_stream().cuda_stream
    g, d = case["kv_heads"], case["head_dim"]
    if case["op"] == "norm_rope":
        h = case["heads"]
        kind = G.DTYPES.index(case["type"].upper())
        kv_kind = G.DTYPES.index("BF16" if case["type"] == "bf16" else "F16")
        G.head_norm_rope(s["x"].data_ptr(), kind, case["rows"], (h + 2 * g) * d, h, g, d,
                         s["q_weight"].data_ptr(), s["k_weight"].data_ptr(), EPSILON,
                         s["positions"].data_ptr(), s["cos"].data_ptr(), s["sin"].data_ptr(),
                         s["cos"].shape[0], s["q"].data_ptr(), kind, h * d, s["k"].data_ptr(),
                         s["v"].data_ptr(), kv_kind, g * d, stream)
        return [s["q"], s["k"], s["v"]]
    if case["op"] == "copy":
        G.page_copy(s["cache"], s["pairs"].data_ptr(), len(s["pairs"]), stream)
        return [s["keys"], s["values"]]
    if case["op"] == "append":
        places = s["places"].data_ptr() if s["places"] is not None else None
        G.page_append(s["cache"], 0, s["batch"], s["k"].data_ptr(), s["v"].data_ptr(), g * d, places,
                      stream)
        return [s["keys"], s["values"]]
    h, kind = case["heads"], G.DTYPES.index(case["type"].upper())
    workspace, scale = s["workspace"], 1.0 / math.sqrt(d)
    if case["op"] == "packed":
        G.packed_attention(s["cache"], 0, s["batch"], s["q"].data_ptr(), kind, h * d, h,
                           s["k"].data_ptr(), s["v"].data_ptr(), g * d, scale, s["out"].data_ptr(),
                           h * d, workspace.data_ptr(), workspace.numel(), stream)
    else:
        G.tree_attention(s["cache"], 0, s["batch"], s["q"].data_ptr(), kind, h * d, h,
                         s["k"].data_ptr(), s["v"].data_ptr(), g * d, s["ancestors"].data_ptr(), 1,
                         scale, s["out"].data_ptr(), h * d, workspace.data_ptr(),
                         workspace.numel(), stream)
    return [s["out"]]


# ---- the plain forms -------------------------------------------------------------
def run(s):
    if own:
        return _run_own(s)
    op = s["case"]["op"]
    if op == "norm_rope":
        return _plain_norm_rope(s)
    if op == "copy":
        source, target = s["pairs"][:, 0].long(), s["pairs"][:, 1].long()
        s["keys"][:, target] = s["keys"][:, source]
        s["values"][:, target] = s["values"][:, source]
        return [s["keys"], s["values"]]
    if op == "append":
        return _plain_append(s)
    return _plain_attention(s)


def _plain_norm_rope(s):
    case = s["case"]
    h, g, d = case["heads"], case["kv_heads"], case["head_dim"]
    x = s["x"].float().reshape(-1, h + 2 * g, d)
    weight = torch.cat([s["q_weight"].expand(h, d), s["k_weight"].expand(g, d)])
    both = x[:, :h + g]
    both = both / torch.sqrt((both * both).mean(-1, keepdim=True) + EPSILON) * (1.0 + weight)
    cos, sin = s["cos"][s["positions"].long()][:, None], s["sin"][s["positions"].long()][:, None]
    a, b = both[..., :d // 2], both[..., d // 2:]
    both = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    s["q"].copy_(both[:, :h])
    s["k"].copy_(both[:, h:])
    s["v"].copy_(x[:, h + g:])
    return [s["q"], s["k"], s["v"]]


def _row_sequences(s):
    """(sequence, row in it) of each packed row."""
    at = torch.arange(len(s["k"]), device="cuda")
    sequence = torch.searchsorted(s["starts"][1:].long(), at, right=True)
    return sequence, at - s["starts"].long()[sequence]


def _plain_append(s):
    sequence, place = _row_sequences(s)
    if s["places"] is not None:
        place = s["places"].long()
    taken = place >= 0
    sequence, place = sequence[taken], place[taken]
    row = s["cached"].long()[sequence] + place
    page_rows = s["case"]["page_rows"]
    page = s["table"][sequence, row // page_rows].long()
    s["keys"][0, page, row % page_rows] = s["k"][taken]
    s["values"][0, page, row % page_rows] = s["v"][taken]
    return [s["keys"], s["values"]]


def _plain_attention(s):
    """Scores of the whole padded batch, in 32 bits: keys are the cached rows,
    padded to the longest, then the new rows, padded to the longest."""
    case = s["case"]
    h, g, d, page_rows = case["heads"], case["kv_heads"], case["head_dim"], case["page_rows"]
    most_rows, most_cached, count = s["most_rows"], s["most_cached"], len(s["cached"])
    starts, cached = s["starts"].long(), s["cached"].long()
    row = torch.arange(most_rows, device="cuda")
    old = torch.arange(most_cached, device="cuda")
    live_row = row < (starts[1:] - starts[:-1])[:, None]
    live_old = old < cached[:, None]
    at = torch.where(live_row, starts[:-1, None] + row, 0)
    page = s["table"].long()[:, old // page_rows] * page_rows + old % page_rows
    page = torch.where(live_old, page, 0)

    def keys_of(pool, new):
        both = torch.cat([pool[0].reshape(-1, g, d)[page], new[at]], 1).float()
        live = torch.cat([live_old, live_row], 1)[..., None, None]
        return torch.where(live, both, 0.0).transpose(1, 2)

    k, v = keys_of(s["keys"], s["k"]), keys_of(s["values"], s["v"])
    q = s["q"][at].float().transpose(1, 2).reshape(count, g, h // g * most_rows, d)
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()) / math.sqrt(d)
    if case["op"] == "tree":
        seen = (s["ancestors"][at][..., None] >> row) & 1 > 0
    else:
        seen = (row <= row[:, None]).expand(count, -1, -1)
    seen = torch.cat([live_old[:, None].expand(-1, most_rows, -1), seen & live_row[:, None]], 2)
    scores = scores.reshape(count, h, most_rows, -1)
    scores = torch.where(seen[:, None], scores, -math.inf)
    peak = scores.amax(-1, keepdim=True)
    weight = torch.exp(scores - torch.where(peak == -math.inf, 0.0, peak))
    total = weight.sum(-1, keepdim=True)
    weight = weight.reshape(count, g, h // g * most_rows, -1)
    out = torch.matmul(weight, v).reshape(count, h, most_rows, d) / torch.where(total > 0, total, 1.0)
    s["out"][at[live_row]] = out.transpose(1, 2)[live_row].to(s["out"].dtype)
    return [s["out"]]


# ---- the definition in 64 bits ----------------------------------------------------
def exact(case, seed):
    if case["op"] in ("append", "copy"):
        return None  # rows are moved, nothing is computed
    s = prepare(case, seed)
    h, g, d = case["heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "norm_rope":
        x = s["x"].double().reshape(-1, h + 2 * g, d)
        outs = []
        for first, count, weight in ((0, h, s["q_weight"]), (h, g, s["k_weight"])):
            part = x[:, first:first + count]
            norm = part.square().sum(-1, keepdim=True) / d + EPSILON
            part = part * norm.rsqrt() * (weight.double() + 1.0)
            turn = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"].long()]
            turned = torch.complex(part[..., :d // 2], part[..., d // 2:]) * turn[:, None]
            outs.append(torch.cat([turned.real, turned.imag], -1))
        return outs + [x[:, h + g:].contiguous()]
    rows, cached = _lengths(case)
    out = torch.zeros((sum(rows), h, d), dtype=torch.float64, device="cuda")
    first = 0
    page_rows = case["page_rows"]
    for i, (n, c) in enumerate(zip(rows, cached)):
        used = s["table"][i, :-(-c // page_rows)].long()
        old_k = s["keys"][0, used].reshape(-1, g, d)[:c]
        old_v = s["values"][0, used].reshape(-1, g, d)[:c]
        k = torch.cat([old_k, s["k"][first:first + n]]).double()
        v = torch.cat([old_v, s["v"][first:first + n]]).double()
        allowed = torch.ones((n, c + n), dtype=torch.bool, device="cuda")
        if case["op"] == "tree":
            bits = s["ancestors"][first:first + n]
            for j in range(n):
                allowed[:, c + j] = (bits >> j) & 1 != 0
        else:
            allowed[:, c:] = torch.tril(allowed[:, c:])
        for head in range(h):
            other = head // (h // g)
            score = s["q"][first:first + n, head].double() @ k[:, other].T.contiguous()
            score = (score * (1.0 / math.sqrt(d))).masked_fill(~allowed, -math.inf)
            out[first:first + n, head] = torch.softmax(score, -1) @ v[:, other].contiguous()
        first += n
    return [out]
