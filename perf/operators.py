"""Speculative decoding over the paged INT8 cache: a tree of drafted tokens is
verified in one attention launch, the accepted path is committed to the cache,
and the pages behind it are forked, freed and compacted.

A case is a dict of plain values.  prepare() makes the inputs on the GPU from
a seed (and, where `own` is true, the operator that a serving program keeps);
run() is one pass; exact() is the attention in 64 bits.

kind "tree"     PreparedTreeAttention: `batch` requests, `nodes_lo` .. `nodes_hi`
                drafted tokens each, committed lengths `ctx_lo` .. `ctx_hi`,
                `heads` query heads, ratio 1 (window only) or 128 (and every
                compressed row), `window` original rows (0: all of them),
                `layers` 16 KiB pages that share one page stride, `lse`
kind "commit"   PreparedPathCommit: after verification `depth` tokens at most of
                each request's tree are kept; their rows move behind the
                committed rows in each of `layers` caches
kind "fork"     PreparedPageFork: `batch` rows of a block table go on as
                `children` rows (parallel samples, beams, ended requests), with
                room for `room` more tokens; partly filled pages are copied
kind "compact"  PreparedPageCompact: the pages in use (`live` of `pages`, as a
                share) move to the front of the pool
"""
import math
import sys
from pathlib import Path

import torch

own = False

ROOT = Path(__file__).resolve().parents[1]
DIM, BLOCK = 512, 32
PAGE = BLOCK * DIM
DEVICE = "cuda"
ALL = 1 << 30                    # a window that holds every row
SOFTMAX_SCALE = 1 / math.sqrt(DIM)


def tree(name, batch, nodes, ctx, *, heads=8, ratio=128, window=128, layers=38, lse=False):
    return dict(name=name, kind="tree", batch=batch, nodes_lo=nodes[0], nodes_hi=nodes[1], ctx_lo=ctx[0], ctx_hi=ctx[1],
                heads=heads, ratio=ratio, window=window, layers=layers, lse=lse)


def commit(name, batch, nodes, ctx, *, depth=8, layers=38):
    return dict(name=name, kind="commit", batch=batch, nodes_lo=nodes[0], nodes_hi=nodes[1], ctx_lo=ctx[0],
                ctx_hi=ctx[1], depth=depth, layers=layers)


def fork(name, batch, children, ctx, *, room=16, layers=38):
    return dict(name=name, kind="fork", batch=batch, children=children, ctx_lo=ctx[0], ctx_hi=ctx[1], room=room,
                layers=layers)


def compact(name, pages, live, *, batch=32, layers=38):
    return dict(name=name, kind="compact", pages=pages, live=live, batch=batch, layers=layers)


def listed():
    return [
        # A lone request's tree of eight drafted tokens on a C128 layer: the smallest call, all latency.
        tree("tree_1x8", 1, (8, 8), (4096, 4096)),
        # A decode batch on a C128 layer with trees of 4 to 16 tokens and mixed contexts.
        tree("tree_32_ragged", 32, (4, 16), (2048, 65536)),
        # A window-only layer under larger trees, log-sum-exp asked for too.
        tree("tree_window_48x25", 48, (25, 25), (1500, 65536), ratio=1, lse=True),
        # All 64 heads on one GPU (data-parallel attention), long contexts: many query rows for each key.
        tree("tree_64_heads", 16, (24, 24), (65536, 131072), heads=64),
        # A layer that attends its whole INT8 context: 16 heads, trees of about 61 tokens.  The largest products.
        tree("tree_whole_context", 4, (57, 61), (20011, 32768), heads=16, ratio=1, window=0, layers=1),
        # One request's accepted tokens in every layer.
        commit("commit_1", 1, (8, 8), (4096, 4096)),
        # A batch's accepted tokens in every layer of the pool.
        commit("commit_64", 64, (9, 25), (300, 4096)),
        # One request goes on as four samples: the smallest change of a block table.
        fork("fork_1_to_4", 1, 4, (1900, 1900), layers=3),
        # Sixty-four beams reordered, tails of all layers copied.
        fork("fork_64_beams", 64, 64, (200, 1000)),
        # A large batch: most rows go on alone, some end, some fork; one layer's pool.
        fork("fork_256", 256, 277, (500, 8000), room=64, layers=1),
        # A small one-layer pool with few holes.
        compact("compact_512", 509, 0.9, batch=8, layers=1),
        # The serving pool of all layers after a burst of requests has ended.
        compact("compact_1536", 1536, 0.55),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the same ranges, none larger than the listed ones."""
    kind = rng.choice(["tree", "tree", "tree", "commit", "fork", "compact"])
    if kind == "tree":
        whole = rng.random() < 0.25
        heads = rng.choice([1, 4, 8, 8, 16]) if whole else rng.choice([4, 8, 8, 8, 12, 16, 64])
        nodes_hi = _log(rng, 1, 64)
        nodes_lo = rng.randint(max(1, nodes_hi // 2), nodes_hi)
        if whole:
            ctx_hi = _log(rng, 500, 32768)
            most = max(1, min(16, int(4 * 61 * 16 * 32768 * 0.9) // (ctx_hi * nodes_hi * heads), 100000 // ctx_hi))
            return _unnamed(tree("", _log(rng, 1, most), (nodes_lo, nodes_hi), (max(1, ctx_hi // 2), ctx_hi), heads=heads,
                                 ratio=1, window=0, layers=rng.choice([1, 3]), lse=rng.random() < 0.3))
        ratio = rng.choice([128, 128, 1])
        ctx_lo = _log(rng, 1, 65536)
        ctx_hi = min(131072, int(ctx_lo * rng.uniform(1.0, 8.0)) + 1)
        most = max(1, min(64, 24000 // (nodes_hi * heads)))
        return _unnamed(tree("", _log(rng, 1, most), (nodes_lo, nodes_hi), (ctx_lo, ctx_hi), heads=heads, ratio=ratio,
                             window=rng.choice([128, 128, 128, 1024, 33]), layers=rng.choice([1, 3, 38]),
                             lse=rng.random() < 0.3))
    if kind == "commit":
        nodes_hi = _log(rng, 1, 64)
        ctx_lo = _log(rng, 1, 2000)
        return _unnamed(commit("", _log(rng, 1, 64), (rng.randint(1, nodes_hi), nodes_hi), (ctx_lo, 2 * ctx_lo),
                               depth=rng.randint(1, 17), layers=rng.choice([1, 3, 38])))
    if kind == "fork":
        layers = rng.choice([1, 3, 38])
        batch = _log(rng, 1, 256 if layers == 1 else 64)
        ctx_lo = _log(rng, 1, 8000 if layers == 1 else 500)
        return _unnamed(fork("", batch, max(1, int(batch * rng.uniform(0.5, 1.2)) + rng.randint(0, 3)),
                             (ctx_lo, min(8000 if layers == 1 else 1000, 2 * ctx_lo)), room=rng.choice([0, 1, 16, 64]),
                             layers=layers))
    layers = rng.choice([1, 3, 38])
    return _unnamed(compact("", _log(rng, 40, 1536 if layers == 38 else 8192), rng.uniform(0.2, 0.98),
                            batch=rng.randint(1, 64), layers=layers))


def _unnamed(case):
    return {k: v for k, v in case.items() if k != "name"}


def _spread(lo, hi, n, shift=0):
    """n whole numbers spread over lo .. hi (both met from two on), in a mixed order."""
    if n == 1:
        return [hi]
    ends = [lo + (hi - lo) * i // (n - 1) for i in range(n)]
    step = next(s for s in range(max(1, int(n * 0.618)), 2 * n + 2) if math.gcd(s, n) == 1)
    return [ends[(shift + i * step) % n] for i in range(n)]


def _requests(case):
    """(drafted tokens, committed lengths) of the requests."""
    n = case["batch"]
    return _spread(case["nodes_lo"], case["nodes_hi"], n), _spread(case["ctx_lo"], case["ctx_hi"], n, n // 3)


def _window(case):
    return case["window"] or ALL


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _pool(gen, pages, layers, layer):
    """INT8 pages of one layer at the pool's common stride: normal values in steps of the channel scale."""
    pool = torch.empty(pages * layers * PAGE, dtype=torch.int8, device=DEVICE)
    view = pool.as_strided((pages, BLOCK, 1, DIM), (layers * PAGE, DIM, DIM, 1), layer * PAGE)
    for at in range(0, pages, 4096):
        part = view[at:at + 4096]
        part.copy_((torch.randn(part.shape, generator=gen, device=DEVICE) * 28).round_().clamp_(-127, 127))
    return view


def _scale(gen):
    """Channel scales of such a cache: sixteen channels are eight times as large."""
    scale = 0.03 + 0.01 * torch.rand(DIM, generator=gen, device=DEVICE)
    scale[torch.randperm(DIM, generator=gen, device=DEVICE)[:16]] *= 8
    return scale


def _table(gen, counts, width):
    """A block table whose rows hold `counts` pages each, in mixed order; (table, pages)."""
    total = sum(counts)
    pages = total + total // 8 + 1
    order = torch.randperm(pages, generator=gen, device=DEVICE)[:max(1, total)].to(torch.int32)
    ends = torch.tensor([0] + counts, device=DEVICE).cumsum(0)
    col = torch.arange(width, device=DEVICE)[None]
    held = col < _ints(counts)[:, None]
    return torch.where(held, order[(ends[:-1, None] + col).clamp(max=max(0, total - 1))], -1).contiguous(), pages


def _trees(gen, nodes):
    """Parents of each request's drafted tokens (-1: the last committed token), lower nodes first."""
    host = torch.Generator().manual_seed(torch.randint(1 << 30, (1,), generator=gen, device=DEVICE).item())
    parents = []
    for n in nodes:
        pick = torch.rand(n, generator=host)
        back = (torch.rand(n, generator=host) * 6).long() + 1
        parents += [-1 if i < 2 or pick[i] < 0.04 else max(0, i - int(back[i])) for i in range(n)]
    return _ints(parents)


def _bounds(nodes):
    at = [0]
    for n in nodes:
        at.append(at[-1] + n)
    return at


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    state = {"case": case}
    {"tree": _prepare_tree, "commit": _prepare_commit, "fork": _prepare_fork,
     "compact": _prepare_compact}[case["kind"]](case, gen, state)
    if own:
        state["op"] = _operator(state)
    return state


def _operator(s):
    """The framework's operator for these inputs, as a serving program keeps it."""
    if str(ROOT / "ascend-int8-attention_amd") not in sys.path:
        sys.path.insert(0, str(ROOT / "ascend-int8-attention_amd"))
    import npu_sparse_attn_sharedkv_int8 as sharedkv
    case = s["case"]
    if case["kind"] == "tree":
        launch = sharedkv.SharedKVCase(s["q"], s["ori"], s["ori_table"], s["cu_q"], s["seq_lens"], s["sink"], s["cmp"],
                                       s["cmp_table"], None, ratio=case["ratio"], window=_window(case),
                                       softmax_scale=SOFTMAX_SCALE)
        return sharedkv.PreparedTreeAttention(launch, s["parents"], s["ori_scale"], s["cmp_scale"],
                                              return_lse=case["lse"])
    if case["kind"] == "commit":
        return sharedkv.PreparedPathCommit(s["caches"], s["table"], s["cu_q"], s["seq_lens"], s["paths"],
                                           s["path_lens"])
    if case["kind"] == "fork":
        return sharedkv.PreparedPageFork([s["backing"]], s["table"], s["seq_lens"], s["refs"], s["parents"],
                                         room=case["room"])
    return sharedkv.PreparedPageCompact([s["backing"]], s["table"], s["refs"])


def run(s):
    kind = s["case"]["kind"]
    if own:
        s["op"].run()
        if kind == "tree":
            return [s["op"].out, s["op"].lse] if s["case"]["lse"] else [s["op"].out]
        if kind == "commit":
            return [s["op"].seq_lens] + s["caches"]
        if kind == "fork":
            return [s["op"].block_table, s["op"].seq_lens, s["op"].refs, s["op"].missing, s["backing"]]
        return [s["op"].block_table, s["op"].refs, s["op"].moved, s["op"].live, s["backing"]]
    return {"tree": _plain_tree, "commit": _plain_commit, "fork": _plain_fork, "compact": _plain_compact}[kind](s)


# ------------------------------------------------------------ a tree of drafted tokens

def _prepare_tree(case, gen, s):
    nodes, committed = _requests(case)
    ratio, layers = case["ratio"], case["layers"]
    s["cu_q"] = _ints(_bounds(nodes))
    s["seq_lens"] = _ints([c + n for c, n in zip(committed, nodes)])
    s["parents"] = _trees(gen, nodes)
    s["q"] = torch.randn(sum(nodes), case["heads"], DIM, generator=gen, device=DEVICE).to(torch.bfloat16)
    s["sink"] = torch.linspace(-2, 2, case["heads"], device=DEVICE)
    # Pages behind the window have been given back: their table entries are -1.
    first = [max(0, c - _window(case) + 1) // BLOCK for c in committed]
    last = [-(-(c + n) // BLOCK) for c, n in zip(committed, nodes)]
    held, pages = _table(gen, [b - a for a, b in zip(first, last)], max(b - a for a, b in zip(first, last)))
    col = torch.arange(max(last), device=DEVICE)[None] - _ints(first)[:, None]
    inside = (col >= 0) & (col < held.shape[1])
    s["ori_table"] = torch.where(inside, held.gather(1, col.clamp(0, held.shape[1] - 1)), -1).to(torch.int32).contiguous()
    s["ori"], s["ori_scale"] = _pool(gen, pages, layers, layers // 2), _scale(gen)
    s["cmp"] = s["cmp_table"] = s["cmp_scale"] = None
    s["first"] = [a * BLOCK for a in first]
    s["keys"] = max((b - a) * BLOCK for a, b in zip(first, last))
    s["cmp_keys"] = max(c // ratio for c in committed) if ratio > 1 else 0
    if ratio > 1:
        counts = [-(-(c // ratio) // BLOCK) for c in committed]
        s["cmp_table"], pages = _table(gen, counts, max(1, max(counts)))
        s["cmp"], s["cmp_scale"] = _pool(gen, pages, layers, layers // 2), _scale(gen)
    s["most"] = max(nodes)
    # Where each token sits in a [batch, most nodes] block, and back.
    s["token"] = torch.tensor([i * s["most"] + k for i, n in enumerate(nodes) for k in range(n)], device=DEVICE)


def _gather(pool, table, rows):
    """Codes of logical `rows` [B, K] as [B, K, 512] in 32 bits."""
    page = table.gather(1, (rows // BLOCK).clamp(max=table.shape[1] - 1)).long().clamp(min=0)
    return pool[page, (rows % BLOCK), 0].float()


def _plain_tree(s):
    case, most, heads = s["case"], s["most"], s["case"]["heads"]
    batch, window = case["batch"], _window(case)
    cu, tokens = s["cu_q"].long(), s["q"].shape[0]
    nodes = cu[1:] - cu[:-1]
    committed = (s["seq_lens"].long() - nodes)[:, None]
    block = lambda x, fill: torch.full((batch * most,) + x.shape[1:], fill, dtype=x.dtype,  # noqa: E731
                                       device=x.device).index_copy_(0, s["token"], x).view(batch, most, *x.shape[1:])
    # Ancestors, the node itself among them: the closure of the parent relation.
    parent = block(s["parents"].long(), -1)
    index = torch.arange(most, device=DEVICE)
    above = ((index == parent[..., None]) | (index == index[:, None])).float()
    for _ in range(max(1, (most - 1).bit_length())):
        above = (torch.bmm(above, above.contiguous()) > 0).float()
    depth = above.sum(-1).long() - 1
    position = committed + depth
    rows = torch.tensor(s["first"], device=DEVICE)[:, None] + torch.arange(s["keys"], device=DEVICE)
    key = _gather(s["ori"], s["ori_table"], rows) * s["ori_scale"]
    node = (rows - committed).clamp(0, most - 1)
    spread = node[:, None].expand(batch, most, s["keys"])
    near = depth[..., None] - depth[:, None].expand(batch, most, most).gather(2, spread) < window
    drafted = (rows - committed >= 0) & (rows - committed < nodes[:, None])
    sees = torch.where(rows[:, None] < committed[:, None], rows[:, None] > position[..., None] - window,
                       (above.gather(2, spread) > 0) & near & drafted[:, None])
    if case["ratio"] > 1 and s["cmp_keys"]:
        rows = torch.arange(s["cmp_keys"], device=DEVICE)[None].expand(batch, -1)
        key = torch.cat([_gather(s["cmp"], s["cmp_table"], rows) * s["cmp_scale"], key], 1)
        sees = torch.cat([(rows < committed // case["ratio"])[:, None].expand(batch, most, -1), sees], 2)
    q = block(s["q"], 0).float().view(batch, most * heads, DIM)
    scores = torch.bmm(q, key.transpose(1, 2).contiguous()).mul_(SOFTMAX_SCALE).view(batch, most, heads, -1)
    scores.masked_fill_(~sees[:, :, None], -math.inf)
    peak = torch.maximum(scores.amax(-1), s["sink"])
    weight = scores.sub_(peak[..., None]).exp_()
    total = weight.sum(-1) + (s["sink"] - peak).exp()
    out = torch.bmm(weight.view(batch, most * heads, -1), key).view(batch, most, heads, DIM) / total[..., None]
    out = out.view(batch * most, heads, DIM)[s["token"]].to(torch.bfloat16)
    if not case["lse"]:
        return [out]
    return [out, (peak + total.log()).view(batch * most, heads)[s["token"]]]


# ------------------------------------------------------------ an accepted path

def _prepare_commit(case, gen, s):
    nodes, committed = _requests(case)
    layers, depth = case["layers"], case["depth"]
    counts = [-(-(c + n) // BLOCK) for c, n in zip(committed, nodes)]
    s["table"], pages = _table(gen, counts, max(counts))
    backing = torch.randint(-127, 128, (pages * layers * PAGE,), generator=gen, device=DEVICE, dtype=torch.int8)
    s["caches"] = [backing.as_strided((pages, BLOCK, 1, DIM), (layers * PAGE, DIM, DIM, 1), k * PAGE)
                   for k in range(layers)]
    s["backing"] = backing
    s["cu_q"], s["seq_lens"] = _ints(_bounds(nodes)), _ints([c + n for c, n in zip(committed, nodes)])
    # The path: rising node indices; how long it is differs from request to request.
    most = max(nodes)
    keys = torch.rand(case["batch"], most, generator=gen, device=DEVICE)
    keys[torch.arange(most, device=DEVICE)[None] >= _ints(nodes)[:, None]] = 2.0
    chosen = keys.argsort(1)[:, :depth]
    lens = torch.minimum(1 + (torch.rand(case["batch"], generator=gen, device=DEVICE) * depth).int(), _ints(nodes))
    lens = lens.clamp(max=depth)
    chosen = torch.where(torch.arange(chosen.shape[1], device=DEVICE)[None] < lens[:, None], chosen, most).sort(1).values
    paths = torch.full((case["batch"], depth), -1, dtype=torch.int32, device=DEVICE)
    paths[:, :chosen.shape[1]] = torch.where(chosen < most, chosen, -1).int()
    s["paths"], s["path_lens"] = paths, lens.int()


def _plain_commit(s):
    table, paths, lens = s["table"].long(), s["paths"].long(), s["path_lens"].long()
    cu = s["cu_q"].long()
    committed = (s["seq_lens"].long() - (cu[1:] - cu[:-1]))[:, None]
    step = torch.arange(paths.shape[1], device=DEVICE)[None]
    kept = step < lens[:, None]
    source, target = (committed + paths)[kept], (committed + step)[kept]
    row = torch.arange(paths.shape[0], device=DEVICE)[:, None].expand_as(kept)[kept]
    at = lambda r: (table[row, r // BLOCK], r % BLOCK)  # noqa: E731
    source, target = at(source), at(target)
    layers = s["case"]["layers"]
    pages = s["backing"].view(-1, layers, BLOCK, DIM)
    pages[target[0], :, target[1]] = pages[source[0], :, source[1]]
    return [(committed[:, 0] + lens).int()] + s["caches"]


# ------------------------------------------------------------ pages of a pool

def _prepare_fork(case, gen, s):
    lengths = _spread(case["ctx_lo"], case["ctx_hi"], case["batch"], case["batch"] // 3)
    counts = [-(-n // BLOCK) for n in lengths]
    width = -(-(case["ctx_hi"] + case["room"]) // BLOCK)
    table, pages = _table(gen, counts, width)
    pages += case["children"] * (2 + case["room"] // BLOCK)      # and free ones for the forked rows
    # Requests with a common prompt: row i shares the whole pages of its group's first row up to a point.
    group = torch.arange(case["batch"], device=DEVICE) // 4 * 4
    whole = _ints([min(lengths[i // 4 * 4], n) // BLOCK // 2 for i, n in enumerate(lengths)])
    shared = torch.arange(width, device=DEVICE)[None] < whole[:, None]
    s["table"] = torch.where(shared, table[group], table).contiguous()
    s["refs"] = torch.zeros(pages, dtype=torch.int32, device=DEVICE)
    held = s["table"][s["table"] >= 0].long()
    s["refs"].index_add_(0, held, torch.ones_like(held, dtype=torch.int32))
    s["seq_lens"] = _ints(lengths)
    parents = torch.randint(case["batch"], (case["children"],), generator=gen, device=DEVICE)
    if case["children"] >= case["batch"] > 64:                   # a large batch: most rows go on alone
        parents[:case["batch"]] = torch.arange(case["batch"], device=DEVICE)
        parents[:case["batch"]][torch.rand(case["batch"], generator=gen, device=DEVICE) < 0.1] = -1
    s["parents"] = parents.int()
    stride = case["layers"] * PAGE
    s["backing"] = torch.randint(-127, 128, (pages, stride), generator=gen, device=DEVICE, dtype=torch.int8)


def _plain_fork(s):
    table, refs, parents = s["table"].long(), s["refs"].long(), s["parents"].long()
    (batch, width), pages, room = table.shape, refs.shape[0], s["case"]["room"]
    alive = (parents >= 0) & (parents < batch)
    safe = parents.clamp(0, batch - 1)
    length = torch.where(alive, s["seq_lens"].long()[safe], 0)
    count = parents.shape[0]
    column = torch.arange(width, device=DEVICE)[None]
    old = torch.where(alive[:, None], table[safe], -1)
    held = (table >= 0) & (table < pages)
    # A parent's first child keeps the parent's own pages.
    order = torch.arange(count, device=DEVICE)
    first = torch.full((batch,), count, device=DEVICE).scatter_reduce_(0, safe[alive], order[alive], "amin")
    whole = (length // BLOCK)[:, None]
    needed = torch.where(alive, (length + room + BLOCK - 1) // BLOCK, 0).clamp(max=width)[:, None]
    good = (old >= 0) & (old < pages)
    keeps = (first[safe] == order)[:, None] & good & (refs[old.clamp(0, pages - 1)] == 1)
    private = (column >= whole) & (column < needed)
    wants = private & ~keeps
    rank = (wants.flatten().long().cumsum(0) - 1).view(count, width)
    free = refs == 0
    spare = torch.full((pages + 1,), -1, device=DEVICE)
    spare[torch.where(free, free.long().cumsum(0) - 1, pages)] = torch.arange(pages, device=DEVICE)
    number = free.sum()
    fresh = torch.where(rank < number, spare[rank.clamp(0, pages - 1)], -1)
    new = torch.where(column < whole, torch.where(good, old, -1), -1)
    new = torch.where(private & keeps, old, torch.where(wants, fresh, new))
    missing = (wants & (rank >= number)).sum()
    tail = whole.clamp(max=width - 1)
    target, source = new.gather(1, tail)[:, 0], old.gather(1, tail)[:, 0]
    partly = alive & (length % BLOCK > 0)
    copies = partly & wants.gather(1, tail)[:, 0] & (target >= 0) & good.gather(1, tail)[:, 0]
    length = torch.where(partly & (target < 0), whole[:, 0] * BLOCK, length)
    s["backing"][target[copies]] = s["backing"][source[copies]]
    change = torch.zeros(pages + 1, dtype=torch.long, device=DEVICE)
    change.index_add_(0, torch.where(held, table, pages).flatten(), torch.full((batch * width,), -1, device=DEVICE))
    change.index_add_(0, torch.where(new >= 0, new, pages).flatten(), torch.ones(count * width, dtype=torch.long,
                                                                                 device=DEVICE))
    return [new.int(), length.int(), (refs + change[:-1]).int(), missing.int().view(1), s["backing"]]


def _prepare_compact(case, gen, s):
    pages, layers, batch = case["pages"], case["layers"], case["batch"]
    used = torch.rand(pages, generator=gen, device=DEVICE) < case["live"]
    s["refs"] = torch.where(used, 1 + (torch.rand(pages, generator=gen, device=DEVICE) < 0.1).int(), 0).int()
    ids = used.nonzero()[:, 0]
    ids = ids[torch.randperm(len(ids), generator=gen, device=DEVICE)]
    width = max(1, int(pages * case["live"]) // batch)
    table = torch.full((batch * width,), -1, dtype=torch.int32, device=DEVICE)
    table[:min(len(ids), batch * width)] = ids[:batch * width].int()
    # Rows of the table differ in length; the pages that none of them names have another owner.
    length = (torch.rand(batch, generator=gen, device=DEVICE) * width).int() + 1
    s["table"] = torch.where(torch.arange(width, device=DEVICE)[None] < length[:, None], table.view(batch, width), -1)
    s["backing"] = torch.randint(-127, 128, (pages, layers * PAGE), generator=gen, device=DEVICE, dtype=torch.int8)


def _plain_compact(s):
    refs, table = s["refs"].long(), s["table"].long()
    pages = refs.shape[0]
    index = torch.arange(pages, device=DEVICE)
    live = refs > 0
    count = live.sum()
    inside = index < count
    source = index[live & ~inside]
    target = index[~live & inside]
    moved = torch.where(live & inside, index, -1)
    moved[source] = target
    s["backing"][target] = s["backing"][source]
    new_refs = torch.where(live & inside, refs, torch.zeros_like(refs))
    new_refs[target] = refs[source]
    good = (table >= 0) & (table < pages)
    new = torch.where(good, moved[table.clamp(0, pages - 1)], -1)
    return [new.int(), new_refs.int(), moved.int(), count.int().view(1), s["backing"]]


# ------------------------------------------------------------ what a pass cannot do without

def work(case):
    """Each input read once, each output written once; for attention one multiplication and addition per query row, key
    that it sees and channel, in Q K and in P V (a tree's nodes are taken at a depth of four)."""
    kind = case["kind"]
    if kind == "tree":
        nodes, committed = _requests(case)
        window, ratio, heads = _window(case), case["ratio"], case["heads"]
        tokens, rows, pairs = sum(nodes), 0, 0
        for n, c in zip(nodes, committed):
            compressed = c // ratio if ratio > 1 else 0
            rows += min(c, window - 1) + n + compressed
            pairs += n * (min(c, max(0, window - 4)) + min(n, 5) + compressed)
        extra = 4 * heads * tokens if case["lse"] else 0
        return {"bytes": rows * DIM + rows // BLOCK * 4 + 4 * tokens * heads * DIM + 4 * tokens + extra
                + 4 * DIM * (2 if ratio > 1 else 1), "flops": 4 * DIM * heads * pairs}
    if kind == "commit":
        nodes, _ = _requests(case)
        kept = sum(min(n, (case["depth"] + 1) / 2) for n in nodes)
        return {"bytes": 2 * kept * DIM * case["layers"] + 16 * case["batch"] + 4 * kept, "flops": 0}
    stride = case["layers"] * PAGE
    if kind == "fork":
        counts = [-(-n // BLOCK) for n in _spread(case["ctx_lo"], case["ctx_hi"], case["batch"])]
        children = case["children"]
        if children >= case["batch"] > 64:
            copies = children - case["batch"]
        else:                                                     # random parents: a child in about 1 - 1/e is the first
            copies = children - case["batch"] * (1 - (1 - 1 / case["batch"]) ** children)
        mean = sum(counts) / len(counts)
        pages = sum(counts) + children * 3
        return {"bytes": 2 * copies * stride + 4 * (sum(counts) + children * mean + 2 * pages), "flops": 0}
    moves = case["pages"] * case["live"] * (1 - case["live"])
    return {"bytes": 2 * moves * stride + 4 * (3 * case["pages"] + 2 * case["pages"] * case["live"]), "flops": 0}


# ------------------------------------------------------------ the definition in 64 bits

def exact(case, seed):
    if case["kind"] != "tree":
        return None                       # page tables, counts and moved bytes: whole numbers
    s = prepare(case, seed)
    cu = s["cu_q"].tolist()
    lengths, parents = s["seq_lens"].tolist(), s["parents"].tolist()
    sink, window, heads = s["sink"].double(), _window(case), case["heads"]
    outs, sums = [], []
    for b in range(case["batch"]):
        n = cu[b + 1] - cu[b]
        before = lengths[b] - n
        chains = []
        for i in range(n):
            chain, at = [], i
            while at >= 0:
                chain.append(at)
                at = parents[cu[b] + at]
            chains.append(chain)
        low = max(0, before - window + 1)
        rows = torch.arange(low, before + n, device=DEVICE)
        at = s["ori_table"][b, rows // BLOCK].long()
        value = s["ori"][at, rows % BLOCK, 0].double() * s["ori_scale"].double()
        seen = torch.zeros(n, len(rows), dtype=torch.bool)
        for i, chain in enumerate(chains):
            seen[i, max(0, before + len(chain) - window - low):before - low] = True
            for k, node in enumerate(chain):
                if k < window:
                    seen[i, before - low + node] = True
        seen = seen.to(DEVICE)
        if case["ratio"] > 1 and before // case["ratio"]:
            rows = torch.arange(before // case["ratio"], device=DEVICE)
            at = s["cmp_table"][b, rows // BLOCK].long()
            value = torch.cat([s["cmp"][at, rows % BLOCK, 0].double() * s["cmp_scale"].double(), value])
            seen = torch.cat([torch.ones(n, len(rows), dtype=torch.bool, device=DEVICE), seen], 1)
        q = s["q"][cu[b]:cu[b + 1]].double()
        logits = torch.matmul(q.reshape(n * heads, DIM), value.t().contiguous()).view(n, heads, -1) / math.sqrt(DIM)
        logits = logits.masked_fill(~seen[:, None], -math.inf)
        top = torch.maximum(logits.amax(-1), sink)
        e = (logits - top[..., None]).exp()
        total = e.sum(-1) + (sink - top).exp()
        outs.append(torch.matmul(e.view(n * heads, -1), value).view(n, heads, DIM) / total[..., None])
        sums.append(top + total.log())
    return [torch.cat(outs), torch.cat(sums)] if case["lse"] else [torch.cat(outs)]
