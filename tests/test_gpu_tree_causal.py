"""PreparedTreeAttention with causal_compressed: a token at position p sees the
(p + 1) // 128 compressed rows that PreparedAttention's queries see there.
Compared with 64 bits (the bounds derived in test_gpu_tree.py, without the term
for scales far apart, which are not drawn here), and a chain with
PreparedAttention itself."""
import sys
import zlib
from types import SimpleNamespace

import numpy as np
import pytest

from tests.test_gpu_tree import BLOCK, DIM, Trees
from tests.test_gpu_tree_rebinding import adapter, call

pytestmark = pytest.mark.gpu
RATIO = 128


def say(*a):
    print(*a, file=sys.stderr, flush=True)


class Causal(Trees):
    """Trees whose compressed pool has room for the rows that the drafted tokens complete, but for those past `room`
    rows of each request's table (None: all)."""

    def __init__(self, seed, nodes, committed, *, room=None, **kw):
        super().__init__(seed, nodes, committed, ratio=RATIO, **kw)
        rows = [(c + n) // RATIO for c, n in zip(committed, nodes)]
        self.cmp = self._kind(self.rng, rows, kw.get("stride", BLOCK * DIM))
        if room is not None:
            self.cmp["table"] = np.ascontiguousarray(self.cmp["table"][:, :-(-room // BLOCK)])

    def chain(self, b, i):
        up, found = i, []
        while up >= 0:
            found.append(up)
            above = self.parents[b][up]
            up = above if 0 <= above < up else -1
        return found

    def expect(self, terms):
        import torch
        q = torch.from_numpy(self.q).to(torch.bfloat16).double().numpy()
        sink = self.sink.astype(np.float64)
        out, near = np.zeros((2, self.tokens, self.heads, DIM))
        lse, lse_near = np.zeros((2, self.tokens, self.heads))
        for b, (n, c) in enumerate(zip(self.nodes, self.committed)):
            for i in range(n):
                chain, t = self.chain(b, i), self.cu[b] + i
                p = c + len(chain) - 1
                window = np.concatenate([np.arange(min(max(0, p - self.window + 1), c), c),
                                         c + np.array(chain[:self.window], np.int64)])
                scores, values, d = [], [], np.zeros(self.heads)
                for kind, rows in ((self.ori, window), (self.cmp, np.arange((p + 1) // RATIO))):
                    codes, good = self.rows(kind, b, rows)
                    codes, scale = codes[good], kind["scale"].astype(np.float64)
                    if len(codes):
                        qs = q[t] * scale
                        scores.append(qs @ codes.T * self.softmax_scale)
                        values.append(codes * scale)
                        step = np.abs(qs).max(1) / (127 * 256 ** (terms - 1))
                        d = np.maximum(d, abs(self.softmax_scale) * step / 2 * np.abs(codes).sum(1).max())
                s, v = np.concatenate(scores, 1), np.concatenate(values)
                top = np.maximum(s.max(1), sink)
                e = np.exp(s - top[:, None])
                total = e.sum(1) + np.exp(sink - top)
                weight = e / total[:, None]
                out[t], size = weight @ v, np.abs(s).max(1)
                slack = 2 * (d + 2 ** -22 * size) + 2 ** -11 + 2 ** -18
                near[t] = 2 ** -8 * np.abs(out[t]) + slack[:, None] * (weight @ np.abs(v)) + 2 ** -33 * np.abs(v).sum(0)
                lse[t] = top + np.log(total)
                lse_near[t] = d + 2 ** -22 * (size + np.abs(lse[t])) + 2 ** -20
        return out, near, lse, lse_near


def compare(trees, out, lse=None):
    want, near, want_lse, lse_near = trees.expect(2 if lse is None else 3)
    off = np.abs(out.double().cpu().numpy() - want) - near
    assert off.max(initial=-1) <= 0, f"out: worst {off.max():.3g} past its bound at {np.unravel_index(off.argmax(), off.shape)}"
    if lse is not None:
        off = np.abs(lse.double().cpu().numpy() - want_lse) - lse_near
        assert off.max(initial=-1) <= 0, f"lse: worst {off.max():.3g} past its bound"


def run(trees, lse, **kw):
    import torch
    from npu_sparse_attn_sharedkv_int8 import PreparedTreeAttention
    case, parents, scale, cmp_scale = trees.device()
    op = PreparedTreeAttention(case, parents, scale, cmp_scale, return_lse=lse, **dict(dict(causal_compressed=True), **kw))
    op.out.fill_(float("nan"))
    op.run()
    torch.cuda.synchronize()
    return op


def chain(*counts):
    return [list(range(-1, n - 1)) for n in counts]


SHAPES = [
    # nodes, committed, heads, window, chains
    ([8], [250], 8, 128, True),                    # row 1 ends within the chain
    ([1], [127], 8, 128, True),                    # and at the only token, the first compressed row there is
    ([1, 1, 1], [126, 127, 128], 3, 128, True),
    ([9, 16, 5], [8185, 8188, 8316], 8, 128, True),    # the last row of a tile of 64, and the first of the next
    ([140], [120], 2, 33, True),                   # two rows in one chain
    ([300], [8180], 1, 128, False),                # a tree of that size, past a tile's end
    ([12, 7, 16], [507, 1020, 2045], 8, 128, False),
    ([24] * 16, [8185 + 128 * b + b % 5 for b in range(16)], 64, 128, False),     # whole units of 64 rows
    ([14] * 10, [128 * 7 * b + 122 + b % 6 for b in range(10)], 64, 128, False),     # of 32
    ([30, 20], [20475, 124], 128, 1000, False),    # units split over items
    ([1100, 3], [90, 126], 1, 128, False),         # more tokens than parents kept in LDS
    ([3] * 300, [121 + 5 * b for b in range(300)], 2, 128, True),        # more requests than threads
]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{len(s[0])}x{max(s[0])}_c{max(s[1])}_h{s[2]}_w{s[3]}")
@pytest.mark.parametrize("lse", [False, True], ids=["out", "lse"])
def test_matches_64_bits(shape, lse):
    nodes, committed, heads, window, chains = shape
    say(f"[causal] {len(nodes)} requests of {max(nodes)} tokens, {heads} heads, lse={lse}")
    trees = Causal(zlib.crc32(str(shape).encode()) % 1000, nodes, committed, heads=heads, window=window,
                   parents=chain(*nodes) if chains else None)
    assert any((c + len(trees.chain(b, i))) // RATIO > c // RATIO
               for b, (n, c) in enumerate(zip(nodes, committed)) for i in range(n))
    op = run(trees, lse)
    compare(trees, op.out, op.lse)


def test_rows_that_the_table_does_not_hold():
    """Compressed rows past the table, and on pages that are none, are masked; the rest of the tile is seen."""
    trees = Causal(70, [10, 10], [4090, 4090], parents=chain(10, 10), room=32)      # row 31 is there, the next is not
    say("[causal] a table of one page")
    op = run(trees, True)
    compare(trees, op.out, op.lse)
    trees = Causal(71, [10, 10], [4100, 4090], parents=chain(10, 10))
    trees.cmp["table"][1, 0] = -1
    say("[causal] no page")
    op = run(trees, True)
    compare(trees, op.out, op.lse)


def test_without_a_row_completed_both_rules_are_one():
    import torch
    trees = Causal(72, [7, 12, 3], [500, 4000, 0])
    assert all((c + n) // RATIO == c // RATIO for c, n in zip(trees.committed, trees.nodes))
    say("[causal] no row ends in the drafts")
    for lse in (False, True):
        assert torch.equal(run(trees, lse).out, run(trees, lse, causal_compressed=False).out)


@pytest.mark.parametrize("committed,tokens", [([250, 127], 8), ([127, 126], 1), ([1000, 8190], 16)])
def test_a_chain_is_the_ordinary_operator(committed, tokens):
    """PreparedAttention is within 2e-2 of the same attention before rounding, and both outputs are rounded to BF16:
    2^-7 |out|.  The committed rows' rule is further off, and is not meant here."""
    import torch
    from npu_sparse_attn_sharedkv_int8 import PreparedAttention
    trees = Causal(73, [tokens] * 2, committed, parents=chain(tokens, tokens))
    case, parents, scale, cmp_scale = trees.device()
    tree = run(trees, True)
    plain = PreparedAttention(case, scale, cmp_scale, return_lse=True)
    say(f"[causal] chain of {tokens} against the ordinary operator")
    plain.run()
    torch.cuda.synchronize()
    assert ((tree.out.float() - plain.out.float()).abs() <= 2e-2 + 2 ** -7 * plain.out.float().abs()).all()


def test_adapter_follows_its_causal_rule():
    """A chain through the serving call, with and without tree_parents; then a captured call."""
    import torch
    trees = Causal(74, [8, 16], [250, 8180], parents=chain(8, 16))
    case, parents, scale, cmp_scale = trees.device()
    layer = adapter(scale, cmp_scale)
    say("[causal] adapter")
    out, lse = layer.attention(case.q, tree_parents=parents, **call(case))
    plain, _ = layer.attention(case.q, **call(case))
    torch.cuda.synchronize()
    compare(trees, out, lse.squeeze(-1))
    assert ((out.float() - plain.float()).abs() <= 2e-2 + 2 ** -7 * plain.float().abs()).all()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = layer.attention(case.q, tree_parents=parents, **call(case))
    for _ in range(3):
        out.fill_(float("nan"))
        graph.replay()
        layer.attention(case.q, **call(case))
        torch.cuda.synchronize()
        compare(trees, out, lse.squeeze(-1))


def test_adapter_without_rows_for_drafted_tokens():
    """tree_causal_compressed=False beside the causal call of the same shape: an operator each."""
    import torch
    from tests.test_gpu_tree import compare as committed_only
    trees = Causal(76, [8, 16], [250, 8180])
    case, parents, scale, cmp_scale = trees.device()
    layer = adapter(scale, cmp_scale)
    for _ in range(2):
        out, lse = layer.attention(case.q, tree_parents=parents, **call(case))
        less, less_lse = layer.attention(case.q, tree_parents=parents, tree_causal_compressed=False, **call(case))
        torch.cuda.synchronize()
        say("[causal] adapter, both rules")
        compare(trees, out, lse.squeeze(-1))
        want = Trees.expect(trees, 3)
        committed_only(SimpleNamespace(out=less, lse=less_lse.squeeze(-1)),
                       SimpleNamespace(expect=lambda terms: want), True)
        assert len(layer.operators.values()) == 2


def test_speculative_chains_over_both_caches():
    """Steps of a decode loop with compressed rows: the drafted rows and those that they complete are written, the
    chains verified, a part of each accepted.  A compressed row is the mean of its 128 original rows here."""
    import torch
    from npu_sparse_attn_sharedkv_int8 import (CacheQuantization, PreparedCacheWrite, PreparedPathCommit,
                                               PreparedTreeAttention, SharedKVCase)
    rng = np.random.default_rng(75)
    batch, nodes, heads, width = 3, 12, 4, 14
    quant = CacheQuantization(torch.full((DIM,), 0.03))
    scale, inverse = quant.scale.cuda(), quant.inverse_scale.cuda()
    lengths = np.array([100, 250, 371])
    pool = torch.from_numpy(rng.integers(-100, 100, (batch * width, BLOCK, 1, DIM)).astype(np.int8)).cuda()
    compressed = torch.zeros((batch + 2, BLOCK, 1, DIM), dtype=torch.int8, device="cuda")
    table = torch.from_numpy(rng.permutation(batch * width).reshape(batch, width).astype(np.int32)).cuda()
    cmp_table = torch.tensor([[2], [4], [1]], dtype=torch.int32, device="cuda")
    ints = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")  # noqa: E731

    def row_slots(where, rows):
        return where[:, rows // BLOCK].long() * BLOCK + rows % BLOCK

    def complete(first, end):
        """Writes the compressed rows that end in rows [first, end) of each request."""
        for b in range(batch):
            for r in range(first[b] // RATIO, end[b] // RATIO):
                rows = torch.arange(r * RATIO, (r + 1) * RATIO, device="cuda")
                codes = pool.view(-1, DIM)[row_slots(table, rows)[b]]
                mean = (codes.float() * scale).mean(0)[None].bfloat16()
                PreparedCacheWrite(compressed, mean, row_slots(cmp_table, torch.tensor([r], device="cuda"))[b], inverse).run()

    complete(np.zeros(batch, int), lengths)
    cu, seq, sink = ints(np.arange(batch + 1) * nodes), ints(lengths), torch.zeros(heads, device="cuda")
    q = torch.zeros((batch * nodes, heads, DIM), dtype=torch.bfloat16, device="cuda")
    paths, path_lens = ints([list(range(nodes))] * batch), ints([0] * batch)
    parents = ints(np.concatenate(chain(*[nodes] * batch)))
    case = SharedKVCase(q, pool, table, cu, seq, sink, compressed, cmp_table, ratio=RATIO, window=128)
    tree = PreparedTreeAttention(case, parents, scale, scale, return_lse=True, causal_compressed=True)
    commit = PreparedPathCommit(pool, table, cu, seq, paths, path_lens)
    for step in range(4):
        drafts = torch.from_numpy(rng.standard_normal((batch * nodes, DIM)).astype(np.float32)).cuda().bfloat16()
        queries = rng.standard_normal((batch * nodes, heads, DIM)).astype(np.float32)
        q.copy_(torch.from_numpy(queries))
        seq.copy_(ints(lengths + nodes))
        slots = torch.cat([row_slots(table, torch.arange(n, n + nodes, device="cuda"))[b] for b, n in enumerate(lengths)])
        PreparedCacheWrite(pool, drafts, slots, inverse).run()
        complete(lengths, lengths + nodes)
        say(f"[causal] step {step} at {lengths.tolist()}")
        tree.run()
        torch.cuda.synchronize()
        expect = Causal(0, [nodes] * batch, lengths.tolist(), heads=heads, parents=chain(*[nodes] * batch))
        expect.q, expect.sink = queries, sink.cpu().numpy()
        expect.ori = dict(pool=pool[:, :, 0].cpu().numpy(), table=table.cpu().numpy(), scale=quant.scale.numpy())
        expect.cmp = dict(pool=compressed[:, :, 0].cpu().numpy(), table=cmp_table.cpu().numpy(), scale=quant.scale.numpy())
        compare(expect, tree.out, tree.lse)
        accepted = rng.integers(1, nodes + 1, batch)
        path_lens.copy_(ints(accepted))
        lengths = lengths + accepted
        assert commit.run().tolist() == lengths.tolist()
