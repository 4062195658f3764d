"""PreparedTreeAttention against attention in 64 bits.

Bounds (derived, none fitted).  With the row's largest |q scale| = peak, codes
of 8 n bits are whole multiples of step = peak / (127 * 256^(n-1)), off by
half a step at most, so a score is off by
  d = softmax_scale * step / 2 * max_j sum_c |code[j][c]|
(n = 2, and 3 where the log-sum-exp is asked for) and by FP32 roundings of at
most four half steps of its size, 2^-22 max|s|.  A weight relative to the sum
is then off by 2 (d + 2^-22 max|s|) and by FP16's 2^-11, the exponential, the
sums and the scales by less than 2^-18 together, each relative to
A = sum_j p_j |v_j|; the output's rounding adds 2^-8 |out|.  FP16 weights start
at 2^8 for a row's largest and are multiples of 2^-24 at the low end, so each is
off by 2^-25 besides, at most 2^-33 of the largest (which is at most the sum):
2^-33 sum_j |v_j|, all that is left in a channel where every heavy key's code
is 0.  Where a channel's original scale is below 2^-60 of the compressed one, a
unit of both kinds takes 2^-60 of the compressed one, r, for it: with s the
true scale, 0 < s < r, what the original rows add is off by
(r - s) |sum_j p_j code_j| < r sum_j p_j |code_j| over the original rows, times
1 + 2^-8 for the output's rounding and 1 + 2^-9 for the weights' (2^-6
together); no term for other channels.  The log-sum-exp is
off by d + 2^-22 (max|s| + |lse|) + 2^-20.
"""
import math
import sys
import zlib

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
DIM, BLOCK = 512, 32
ALL = 1 << 30


def say(*a):
    print(*a, file=sys.stderr, flush=True)


class Trees:
    """Inputs on the host.  `parents` per request: a list of lists, or None for random trees."""

    def __init__(self, seed, nodes, committed, *, heads=8, ratio=128, window=128, parents=None, stride=BLOCK * DIM,
                 pad_tokens=0, pad_batch=0, softmax_scale=1 / math.sqrt(DIM), q_size=1.0):
        rng = self.rng = np.random.default_rng(seed)
        self.nodes, self.committed, self.heads, self.ratio, self.window = nodes, committed, heads, ratio, window
        self.softmax_scale, self.pad_batch = softmax_scale, pad_batch
        if parents is None:
            parents = [[int(rng.integers(-1, i)) if rng.random() < 0.3 else i - 1 - int(rng.integers(0, min(i, 3) + 1))
                        for i in range(n)] for n in nodes]
        self.parents = parents
        tokens = sum(nodes)
        self.live_tokens, self.tokens = tokens, tokens + pad_tokens
        self.cu = np.array([0] + list(np.cumsum(nodes)) + [tokens] * pad_batch, np.int32)
        self.seq = np.array([c + n for c, n in zip(committed, nodes)] + [0] * pad_batch, np.int32)
        self.q = rng.standard_normal((self.tokens, heads, DIM)).astype(np.float32) * q_size
        self.sink = rng.standard_normal(heads).astype(np.float32)
        self.ori = self._kind(rng, [c + n for c, n in zip(committed, nodes)], stride)
        self.cmp = self._kind(rng, [c // ratio for c in committed], stride) if ratio > 1 else None

    def _kind(self, rng, rows, stride):
        pages = [-(-r // BLOCK) for r in rows]
        total = max(1, sum(pages) + 3)
        order = rng.permutation(total)
        table = np.full((len(rows) + self.pad_batch, max(1, max(pages)) + 1), -1, np.int32)
        at = 0
        for b, n in enumerate(pages):
            table[b, :n] = order[at:at + n]
            at += n
        pool = np.clip(np.rint(rng.standard_normal((total, BLOCK, DIM)) * 40), -127, 127).astype(np.int8)
        scale = (0.02 + 0.02 * rng.random(DIM)).astype(np.float32)
        scale[rng.choice(DIM, 16, replace=False)] *= 8
        return dict(pool=pool, table=table, scale=scale, stride=stride)

    def device(self):
        import torch
        from npu_sparse_attn_sharedkv_int8 import SharedKVCase

        def cache(kind):
            if kind is None:
                return None, None, None
            pages = len(kind["pool"])
            flat = torch.full((pages * kind["stride"],), 77, dtype=torch.int8, device="cuda")
            view = flat.as_strided((pages, BLOCK, 1, DIM), (kind["stride"], DIM, DIM, 1))
            view.copy_(torch.from_numpy(kind["pool"])[:, :, None])
            return view, torch.from_numpy(kind["table"]).cuda(), torch.from_numpy(kind["scale"]).cuda()

        ori, table, scale = cache(self.ori)
        cmp, cmp_table, cmp_scale = cache(self.cmp)
        self.q_dev = torch.from_numpy(self.q).to(torch.bfloat16).cuda()
        case = SharedKVCase(self.q_dev, ori, table, torch.from_numpy(self.cu).cuda(), torch.from_numpy(self.seq).cuda(),
                            torch.from_numpy(self.sink).cuda(), cmp, cmp_table, None, ratio=self.ratio,
                            window=self.window, softmax_scale=self.softmax_scale)
        flat = [p for row in self.parents for p in row] + [-1] * (self.tokens - self.live_tokens)
        parents = torch.tensor(flat, dtype=torch.int32, device="cuda")
        return case, parents, scale, cmp_scale

    def rows(self, kind, b, rows):
        """(codes, readable) of logical rows."""
        entry = rows // BLOCK
        inside = entry < kind["table"].shape[1]
        page = np.where(inside, kind["table"][b, np.minimum(entry, kind["table"].shape[1] - 1)], -1)
        good = (page >= 0) & (page < len(kind["pool"]))
        return kind["pool"][np.where(good, page, 0), rows % BLOCK].astype(np.float64), good

    def expect(self, terms):
        """(out, allowed |difference|, lse, allowed) in 64 bits."""
        import torch
        q = torch.from_numpy(self.q).to(torch.bfloat16).double().numpy()
        out = np.zeros((self.tokens, self.heads, DIM))
        near, lse, lse_near = np.zeros_like(out), np.zeros(out.shape[:2]), np.zeros(out.shape[:2])
        for b, (n, c) in enumerate(zip(self.nodes, self.committed)):
            for i in range(n):
                chain, a = [], i
                while a >= 0:
                    chain.append(a)
                    up = self.parents[b][a]
                    a = up if 0 <= up < a else -1
                depth = len(chain) - 1
                low = max(0, c + depth - self.window + 1)
                mine = np.concatenate([np.arange(min(low, c), c), c + np.array(chain[:self.window], np.int64)])
                kinds = [(self.ori, mine)]
                if self.ratio > 1:
                    kinds.append((self.cmp, np.arange(c // self.ratio)))
                t = self.cu[b] + i
                scores, values, d = [], [], np.zeros(self.heads)
                raised = []                     # |value| of the rows whose scale is raised, as raised
                for kind, rows in kinds:
                    codes, good = self.rows(kind, b, rows)
                    codes, scale = codes[good], kind["scale"].astype(np.float64)
                    if not len(codes):
                        continue
                    qs = q[t] * scale
                    scores.append(qs @ codes.T * self.softmax_scale)
                    values.append(codes * scale)
                    least = self.cmp["scale"].astype(np.float64) * 2.0 ** -60 if self.cmp and kind is self.ori else scale
                    raised.append(np.abs(codes) * np.where(scale < least, least, 0))
                    step = np.abs(qs).max(1) / (127 * 256 ** (terms - 1))
                    d = np.maximum(d, abs(self.softmax_scale) * step / 2 * np.abs(codes).sum(1).max())
                sink = self.sink.astype(np.float64)
                if not scores:
                    lse[t] = sink
                    lse_near[t] = 2 ** -20 + 2 ** -22 * np.abs(sink)
                    continue
                s, v = np.concatenate(scores, 1), np.concatenate(values)
                top = np.maximum(s.max(1), sink)
                e = np.exp(s - top[:, None])
                total = e.sum(1) + np.exp(sink - top)
                p = e / total[:, None]
                out[t] = p @ v
                size = np.abs(s).max(1)
                slack = 2 * (d + 2 ** -22 * size) + 2 ** -11 + 2 ** -18
                near[t] = 2 ** -8 * np.abs(out[t]) + slack[:, None] * (p @ np.abs(v)) + 2 ** -33 * np.abs(v).sum(0) \
                    + (1 + 2 ** -6) * (p @ np.concatenate(raised))
                lse[t] = top + np.log(total)
                lse_near[t] = d + 2 ** -22 * (size + np.abs(lse[t])) + 2 ** -20
        return out, near, lse, lse_near


def check(trees, lse=False, prepare=None):
    import torch
    from npu_sparse_attn_sharedkv_int8 import PreparedTreeAttention
    case, parents, scale, cmp_scale = trees.device()
    op = PreparedTreeAttention(case, parents, scale, cmp_scale, return_lse=lse)
    op.out.fill_(float("nan"))
    if prepare:
        prepare(op)
    assert op.run() is op.out
    torch.cuda.synchronize()
    compare(op, trees, lse)
    return op


def compare(op, trees, lse):
    out, near, want, want_near = trees.expect(3 if lse else 2)
    got = op.out.double().cpu().numpy()
    far = np.abs(got - out) - near
    assert not np.isnan(got).any()
    assert far.max(initial=-1) <= 0, f"out: worst {far.max():.3g} past its bound at {np.unravel_index(far.argmax(), far.shape)}"
    if lse:
        off = np.abs(op.lse.double().cpu().numpy() - want) - want_near
        assert off.max(initial=-1) <= 0, f"lse: worst {off.max():.3g} past its bound"


SHAPES = [
    # nodes, committed, heads, ratio, window
    ([1], [0], 1, 1, 128),                        # one row, nothing committed
    ([1], [1], 8, 128, 1),                        # a window of one: only itself
    ([8], [4096], 8, 128, 128),
    ([3], [33], 5, 1, 128),                       # 15 query rows: less than a wave's
    ([7, 1, 16, 2], [127, 128, 129, 5000], 8, 128, 128),
    ([25, 24], [63, 4001], 12, 128, 128),         # 300 rows of 12 heads: a token's heads in two units
    ([9], [300], 64, 128, 128),
    ([5], [2000], 128, 1, 33),
    ([40], [31], 3, 1, 17),                       # a chain longer than the window
    ([61, 57], [1000, 1531], 16, 1, ALL),
    ([2], [70000], 8, 1, ALL),                    # a long context
    ([130], [95], 2, 1, 128),                     # a tree over three key tiles
    ([64], [16384], 8, 128, 1024),
]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{len(s[0])}x{max(s[0])}_c{max(s[1])}_h{s[2]}_r{s[3]}_w{s[4]}")
@pytest.mark.parametrize("lse", [False, True], ids=["out", "lse"])
def test_matches_64_bits(shape, lse):
    nodes, committed, heads, ratio, window = shape
    say(f"[tree] {shape} lse={lse}")
    check(Trees(zlib.crc32(str(shape).encode()) % 1000, nodes, committed, heads=heads, ratio=ratio, window=window), lse)


LAUNCHES = [
    # split, nodes, committed, heads, ratio, window: units of 16, 32 and 64 rows
    (False, [3] * 24, [0, 5, 127, 128, 200, 9000] * 4, 64, 128, 128),
    (True, [12, 11], [6000, 4100], 128, 128, 1024),
    (False, [14] * 10, [31, 4096, 127, 300, 9000, 1, 0, 640, 129, 8500], 64, 128, 128),
    (True, [61, 57], [2000, 1531], 64, 1, ALL),
    (False, [16] * 30, [0, 17, 128, 500, 9000, 700] * 5, 64, 128, 128),
    (True, [61], [33000], 16, 1, ALL),             # many items of a unit
    (True, [30, 1], [20000, 70], 128, 128, 1000),
]


@pytest.mark.parametrize("launch", LAUNCHES, ids=lambda s: f"{len(s[1])}x{max(s[1])}_c{max(s[2])}_h{s[3]}_r{s[4]}_w{s[5]}")
@pytest.mark.parametrize("lse", [False, True], ids=["out", "lse"])
def test_units_of_every_size(launch, lse):
    """Units split over items and whole ones, which change from the compressed rows' scales to the original ones'."""
    split, nodes, committed, heads, ratio, window = launch
    say(f"[tree] {launch} lse={lse}")
    op = check(Trees(zlib.crc32(str(launch).encode()) % 1000, nodes, committed, heads=heads, ratio=ratio, window=window), lse)
    assert (op.partial is not None) == split


@pytest.mark.parametrize("nodes,heads,batch", [(3, 64, 24), (14, 64, 10), (16, 64, 30)])
def test_scales_far_apart(nodes, heads, batch):
    """Channels whose original scale is far below the compressed one (their quotient passes FP32's range), and the other
    way round, in units that hold both kinds."""
    trees = Trees(22, [nodes] * batch, [200, 9000] * (batch // 2), heads=heads)
    trees.ori["scale"][::7] = 1e-38
    trees.ori["scale"][1::7] = 1e-8
    trees.cmp["scale"][2::7] = 1e-38
    trees.ori["scale"][3::7] = trees.cmp["scale"][3::7] = 1e-38
    say(f"[tree] scales far apart, {batch} requests of {nodes} tokens")
    assert check(trees, False).partial is None


@pytest.mark.parametrize("batch,heads", [(40, 64), (20, 64), (70, 32)])
def test_whole_units_beside_padding(batch, heads):
    """Units of 64 rows in the order of their length (more than 512 of them, fewer, and more requests than a wave has
    lanes, in their own order), with requests that are padding between live ones and tokens behind them."""
    import torch
    from npu_sparse_attn_sharedkv_int8 import PreparedTreeAttention
    committed = [0, 17, 128, 500, 9000, 700, 3, 1290, 8000, 65]
    trees = Trees(24, [16] * batch, [committed[b % 10] for b in range(batch)], heads=heads, pad_tokens=9, pad_batch=2)
    case, parents, scale, cmp_scale = trees.device()
    dead = list(range(3, batch, 7))
    case.seq_lens[dead] = 0
    op = PreparedTreeAttention(case, parents, scale, cmp_scale)
    assert op.partial is None
    op.out.fill_(float("nan"))
    say(f"[tree] {batch} requests of 16 tokens, {heads} heads, {len(dead)} of them padding")
    op.run()
    torch.cuda.synchronize()
    out, near, _, _ = trees.expect(2)
    for b in dead:
        out[16 * b:16 * b + 16], near[16 * b:16 * b + 16] = 0, 0
    got = op.out.double().cpu().numpy()
    assert not np.isnan(got).any() and (np.abs(got - out) <= near).all()
    assert (op.out[16 * batch:] == 0).all()


@pytest.mark.parametrize("softmax_scale", [-0.05, 0.0, 1.5])
def test_softmax_scales(softmax_scale):
    say(f"[tree] softmax scale {softmax_scale}")
    check(Trees(25, [9, 5], [700, 6000], softmax_scale=softmax_scale), True)
    check(Trees(26, [9, 5], [700, 6000], softmax_scale=softmax_scale), False)


def test_chains_and_stars():
    chain = [[i - 1 for i in range(20)], [-1] * 20, [-1] + [0] * 19]
    say("[tree] chain, roots only, star")
    check(Trees(3, [20, 20, 20], [500, 90, 7], parents=chain), True)
    say("[tree] chain of 50 under a window of 20")
    check(Trees(4, [50], [10], parents=[[i - 1 for i in range(50)]], ratio=1, window=20), True)


def test_parents_that_are_no_lower_index_make_roots():
    parents = [[-1, 5, 1, 3, -9, 2 ** 31 - 1, 4, 7]]
    say("[tree] parents out of range")
    check(Trees(5, [8], [200], parents=parents), True)


def test_tree_of_more_than_a_thousand_tokens():
    say("[tree] 1100 tokens, two heads")
    check(Trees(6, [1100, 3], [77, 2000], heads=2, ratio=1), False)


def test_strided_pages_keep_their_neighbours():
    say("[tree] page stride 622592")
    check(Trees(7, [9, 12], [700, 3001], stride=622592), True)


def test_offsets_past_32_bits():
    """Pages 4 GiB and more into a pool: the table names the last of them."""
    import torch
    from npu_sparse_attn_sharedkv_int8 import PreparedTreeAttention
    trees = Trees(8, [6], [100], ratio=1)
    case, parents, scale, _ = trees.device()
    pages, stride = 7300, 622592
    flat = torch.empty(pages * stride, dtype=torch.int8, device="cuda")
    view = flat.as_strided((pages, BLOCK, 1, DIM), (stride, DIM, DIM, 1))
    view[:7].fill_(1)
    shift = pages - case.ori.shape[0]
    view[shift:].copy_(case.ori)
    case.ori = view
    case.ori_block_table = torch.where(case.ori_block_table >= 0, case.ori_block_table + shift, -1)
    say("[tree] a pool of 4.5 GB")
    op = PreparedTreeAttention(case, parents, scale, return_lse=True)
    op.run()
    torch.cuda.synchronize()
    compare(op, trees, True)


def test_bad_pages_are_masked():
    """Entries outside the pool, and rows past the table: masked, down to a
    row that sees nothing (output 0, log-sum-exp the sink)."""
    trees = Trees(9, [4, 4, 4], [200, 40, 5000])
    trees.ori["table"][0, 5] = 2 ** 30
    trees.ori["table"][1, :] = -1
    trees.cmp["table"][1, :] = len(trees.cmp["pool"])
    trees.cmp["table"][2, 0] = -7
    trees.ori["table"] = np.ascontiguousarray(trees.ori["table"][:, :156])     # request 2 needs 157 pages
    say("[tree] bad pages")
    op = check(trees, True)
    assert (op.out[4:8] == 0).all()


def test_infinite_sinks_and_large_scores():
    trees = Trees(10, [6], [300], heads=4, q_size=40.0)
    trees.sink = np.array([-np.inf, 3.0, -1e30, 1e30], np.float32)
    trees.expect_finite = True
    import torch
    from npu_sparse_attn_sharedkv_int8 import PreparedTreeAttention
    case, parents, scale, cmp_scale = trees.device()
    op = PreparedTreeAttention(case, parents, scale, cmp_scale, return_lse=True)
    say("[tree] sinks at their limits")
    op.run()
    torch.cuda.synchronize()
    with np.errstate(invalid="ignore"):
        compare(op, trees, False)
    assert (op.out[:, 3] == 0).all()
    case.sink.fill_(float("inf"))
    op.run()
    torch.cuda.synchronize()
    assert (op.out == 0).all() and (op.lse == float("inf")).all()
    # Neither a key nor a sink: zero, and a log-sum-exp of -infinity.
    case.sink.fill_(-float("inf"))
    case.ori_block_table.fill_(-1)
    case.cmp_block_table.fill_(-1)
    op.run()
    torch.cuda.synchronize()
    assert (op.out == 0).all() and (op.lse == -float("inf")).all()


def test_rows_that_are_not_finite_stay_by_themselves():
    import torch
    from npu_sparse_attn_sharedkv_int8 import PreparedTreeAttention
    trees = Trees(11, [10, 4], [150, 900])
    case, parents, scale, cmp_scale = trees.device()
    op = PreparedTreeAttention(case, parents, scale, cmp_scale, return_lse=True)
    say("[tree] NaN, infinity and zero rows")
    op.run()
    clean, clean_lse = op.out.clone(), op.lse.clone()
    case.q[2, 3, 100] = float("nan")
    case.q[5, 0, 0] = float("inf")
    case.q[7, 7] = 0
    op.run()
    torch.cuda.synchronize()
    same = torch.ones(14, 8, dtype=torch.bool, device="cuda")
    same[2, 3] = same[5, 0] = same[7, 7] = False
    assert torch.equal(op.out[same], clean[same]) and torch.equal(op.lse[same], clean_lse[same])
    assert op.out[2, 3].isnan().all() and op.out[5, 0].isnan().all() and op.lse[2, 3].isnan() and op.lse[5, 0].isnan()
    trees.q[7, 7] = 0
    trees.q[2, 3] = trees.q[5, 0] = 0       # the rows that are compared are the others
    case.q[2, 3] = case.q[5, 0] = 0
    op.run()
    torch.cuda.synchronize()
    compare(op, trees, True)


def test_extreme_codes():
    """Every code -128 or 127 (a foreign cache may hold -128): the integer sums are at their largest."""
    trees = Trees(12, [3], [500], heads=2, q_size=1.0)
    for kind, code in ((trees.ori, -128), (trees.cmp, 127)):
        kind["pool"][:] = code
    trees.q[:] = 1.0
    for kind in (trees.ori, trees.cmp):
        kind["scale"][:] = 0.03125
    say("[tree] codes at their limits")
    check(trees, True)


@pytest.mark.parametrize("pad_tokens,pad_batch", [(1, 0), (0, 3), (70, 5)])
def test_graph_padding_is_zero(pad_tokens, pad_batch):
    say(f"[tree] padding {pad_tokens} tokens, {pad_batch} requests")
    trees = Trees(13, [5, 9], [300, 77], pad_tokens=pad_tokens, pad_batch=pad_batch)
    op = check(trees, True)
    assert (op.out[14:] == 0).all() and (op.lse[14:] == 0).all()


def test_padding_requests_between_live_ones():
    import torch
    from npu_sparse_attn_sharedkv_int8 import PreparedTreeAttention
    trees = Trees(14, [5, 9, 4], [300, 77, 1000])
    case, parents, scale, cmp_scale = trees.device()
    case.seq_lens[1] = 0
    op = PreparedTreeAttention(case, parents, scale, cmp_scale, return_lse=True)
    op.out.fill_(float("nan"))
    op.lse.fill_(float("nan"))
    op.run()
    torch.cuda.synchronize()
    assert (op.out[5:14] == 0).all() and (op.lse[5:14] == 0).all()
    out, near, lse, lse_near = trees.expect(3)
    got = op.out.double().cpu().numpy()
    live = [*range(5), *range(14, 18)]
    assert (np.abs(got - out)[live] <= near[live]).all()


def test_no_tokens():
    import torch
    from npu_sparse_attn_sharedkv_int8 import PreparedTreeAttention
    trees = Trees(15, [2], [10])
    case, parents, scale, cmp_scale = trees.device()
    case.q, case.cu_q = case.q[:0], torch.zeros(2, dtype=torch.int32, device="cuda")
    assert PreparedTreeAttention(case, parents[:0], scale, cmp_scale).run().shape == (0, 8, 512)


def test_many_requests():
    """More requests than a work-group has threads, of one to four tokens."""
    rng = np.random.default_rng(16)
    nodes = [int(n) for n in rng.integers(1, 5, 300)]
    committed = [int(n) for n in rng.integers(0, 400, 300)]
    say("[tree] 300 requests")
    check(Trees(16, nodes, committed, heads=2), False)


def test_graph_replays_and_rebinding():
    """One captured launch replayed over changing inputs, with eager launches between, each against 64 bits."""
    import torch
    from npu_sparse_attn_sharedkv_int8 import PreparedTreeAttention
    first, second = Trees(17, [7, 12], [500, 4000]), Trees(18, [12, 7], [100, 4100])
    size = max(first.ori["table"].shape[1], second.ori["table"].shape[1])
    for t in (first, second):
        for kind in (t.ori, t.cmp):
            kind["table"] = np.pad(kind["table"], ((0, 0), (0, size - kind["table"].shape[1])), constant_values=-1)
        t.ori["pool"] = np.resize(t.ori["pool"], (200, BLOCK, DIM))
        t.cmp["pool"] = np.resize(t.cmp["pool"], (9, BLOCK, DIM))
    case, parents, scale, cmp_scale = first.device()
    other, other_parents, other_scale, other_cmp_scale = second.device()
    op = PreparedTreeAttention(case, parents, scale, cmp_scale, return_lse=True)
    op.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        op.run()
    eager = PreparedTreeAttention(other, other_parents, other_scale, other_cmp_scale, return_lse=True)
    inputs = [(case.q, other.q), (case.ori, other.ori), (case.cmp, other.cmp), (case.ori_block_table, other.ori_block_table),
              (case.cmp_block_table, other.cmp_block_table), (case.cu_q, other.cu_q), (case.seq_lens, other.seq_lens),
              (case.sink, other.sink), (parents, other_parents), (scale, other_scale), (cmp_scale, other_cmp_scale)]
    saved = [a.clone() for a, _ in inputs]
    for k in range(4):
        for (a, b), kept in zip(inputs, saved):
            a.copy_(b if k & 1 else kept)
        op.out.fill_(float("nan"))
        say(f"[tree] replay {k}")
        graph.replay()
        eager.run()
        torch.cuda.synchronize()
        compare(op, second if k & 1 else first, True)
        compare(eager, second, True)
    # New tensors of the same geometry.
    eager._rebind_same_geometry(case, parents)
    case.q.copy_(saved[0])
    eager.run()
    torch.cuda.synchronize()


def test_made_under_capture():
    """Scratch that is not clear, first seen under capture: an eager run and a second graph before the first's replay."""
    import torch
    from npu_sparse_attn_sharedkv_int8 import PreparedTreeAttention
    trees = Trees(23, [7, 12], [500, 4000])
    case, parents, scale, cmp_scale = trees.device()
    PreparedTreeAttention(case, parents, scale, cmp_scale, return_lse=True).run()
    dirty = {"tree_workspace": torch.full((1 << 10,), 7, dtype=torch.int32, device="cuda"),
             "tree_partial": torch.full((1 << 23,), float("nan"), device="cuda")}
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    with torch.cuda.graph(graphs[0]):
        op = PreparedTreeAttention(case, parents, scale, cmp_scale, return_lse=True,
                                   scratch_allocator=lambda name, shape, dtype, device: dirty[name][:shape[0]])
        op.run()
    with torch.cuda.graph(graphs[1]):
        op.run()
    assert op.partial is not None
    for step in (graphs[1].replay, op.run, graphs[0].replay, op.run, graphs[1].replay):
        op.out.fill_(float("nan"))
        say("[tree] a run of an operator made under capture")
        step()
        torch.cuda.synchronize()
        compare(op, trees, True)


def test_another_stream():
    import torch
    from npu_sparse_attn_sharedkv_int8 import PreparedTreeAttention
    trees = Trees(19, [7, 12], [500, 4000])
    case, parents, scale, cmp_scale = trees.device()
    op = PreparedTreeAttention(case, parents, scale, cmp_scale, return_lse=True)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    say("[tree] a second stream")
    with torch.cuda.stream(side):
        op.run()
    side.synchronize()
    compare(op, trees, True)


def test_two_operators_at_once():
    """Split launches of two operators on two streams, over the same caches."""
    import torch
    from npu_sparse_attn_sharedkv_int8 import PreparedTreeAttention
    trees = Trees(27, [7, 12, 16], [500, 4000, 12000])
    case, parents, scale, cmp_scale = trees.device()
    ops = [PreparedTreeAttention(case, parents, scale, cmp_scale, return_lse=True) for _ in range(2)]
    assert all(op.partial is not None for op in ops)
    for op in ops:
        op.out.fill_(float("nan"))
    torch.cuda.synchronize()
    say("[tree] two streams at once")
    streams = [torch.cuda.Stream() for _ in ops]
    for _ in range(20):
        for op, stream in zip(ops, streams):
            with torch.cuda.stream(stream):
                op.run()
    torch.cuda.synchronize()
    for op in ops:
        compare(op, trees, True)


def test_equals_the_window_operator_on_a_chain():
    """A chain is an ordinary multi-token decode.  PreparedAttention is within
    2e-2 of the same attention before rounding (its P codes), and both outputs
    are rounded to BF16, half a step (2^-8 of the value) each: 2^-7 |out|, 0.06
    in the channels of large scale, where |out| reaches 8."""
    import torch
    from npu_sparse_attn_sharedkv_int8 import PreparedAttention, PreparedTreeAttention
    trees = Trees(20, [4, 4], [300, 1000], ratio=1, parents=[[-1, 0, 1, 2]] * 2)
    case, parents, scale, _ = trees.device()
    say("[tree] chain against the window operator")
    tree = PreparedTreeAttention(case, parents, scale).run()
    plain = PreparedAttention(case, scale).run()
    torch.cuda.synchronize()
    assert ((tree.float() - plain.float()).abs() <= 2e-2 + 2 ** -7 * plain.float().abs()).all()


def test_refusals():
    import torch
    from npu_sparse_attn_sharedkv_int8 import PreparedTreeAttention
    trees = Trees(21, [4, 4], [300, 1000])

    def refuse(match, change=None, **kw):
        case, parents, scale, cmp_scale = trees.device()
        args = dict(case=case, parents=parents, ori_scale=scale, cmp_scale=cmp_scale, **kw)
        if change:
            change(args)
        with pytest.raises(ValueError, match=match):
            PreparedTreeAttention(**args)

    def case_field(name, value):
        def change(args):
            setattr(args["case"], name, value(getattr(args["case"], name)))
        return change

    refuse("BF16", case_field("q", lambda q: q.float()))
    refuse("BF16", case_field("q", lambda q: q.cpu()))
    refuse("BF16", case_field("q", lambda q: q[..., :256]))
    refuse("contiguous", case_field("q", lambda q: q.transpose(0, 1).contiguous().transpose(0, 1)))
    refuse("heads", case_field("q", lambda q: torch.cat([q] * 17, 1)))
    refuse("ratio 4", case_field("ratio", lambda r: 4))
    refuse("explicit", case_field("ori_indices", lambda r: torch.zeros(8, 1, 4, dtype=torch.int32, device="cuda")))
    refuse("window", case_field("window", lambda r: 0))
    refuse("window", case_field("window", lambda r: 2 ** 31))
    refuse("INT8", case_field("ori", lambda c: c.float()))
    refuse("INT8", case_field("cmp", lambda c: None))
    refuse("pages of 32", case_field("ori", lambda c: c.reshape(-1, 16, 1, 512)))
    refuse("block table", case_field("ori_block_table", lambda t: t.long()))
    refuse("block table", case_field("cmp_block_table", lambda t: t[:1]))
    refuse("one page", case_field("cmp_block_table", lambda t: t[:, :0].contiguous()))
    refuse("scale", lambda a: a.update(cmp_scale=None))
    refuse("scale", lambda a: a.update(ori_scale=a["ori_scale"][:500]))
    refuse("parents", lambda a: a.update(parents=a["parents"][:7]))
    refuse("metadata", lambda a: a.update(parents=a["parents"].long()))
    refuse("metadata", case_field("seq_lens", lambda t: t.long()))
    refuse("metadata", case_field("cu_q", lambda t: t[:2].contiguous()))
    refuse("output", lambda a: a.update(output=torch.empty(8, 8, 512, device="cuda")))
    refuse("LSE", lambda a: a.update(lse_output=torch.empty(8, 7, device="cuda")))
    refuse("overlap", lambda a: a.update(output=a["case"].q))
    refuse("overlap", lambda a: a.update(lse_output=a["case"].q.view(torch.float32).reshape(-1)[:64].view(8, 8)))
