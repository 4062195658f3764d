"""Speculative decoding over one pool, the operators as they are used together:
fork and grow the rows of a block table, write the drafted rows, verify the
trees, commit the accepted paths, compact the pages.  A plain mirror on the
host keeps every sequence's rows; after each step the cache holds exactly them,
and the attention is compared with 64 bits (bounds of test_gpu_tree.py).  Then
the same attention through the serving adapter's call."""
import math
import sys
from types import SimpleNamespace

import numpy as np
import pytest

from tests.test_gpu_pages import ints
from tests.test_gpu_tree import Trees, compare

pytestmark = pytest.mark.gpu
BLOCK, DIM, LAYERS = 32, 512, 2


def say(*a):
    print(*a, file=sys.stderr, flush=True)


def pool_rows(flat, table, row, count):
    """Codes of a row's first `count` tokens in each layer, [LAYERS, count, 512]."""
    pages = flat.cpu().numpy().reshape(-1, LAYERS, BLOCK, DIM)
    at = np.arange(count)
    page = np.asarray(table)[row, at // BLOCK]
    return pages[page, :, at % BLOCK].transpose(1, 0, 2)


@pytest.mark.parametrize("captured", [False, True], ids=["eager", "graph"])
def test_decode_loop(captured):
    import torch
    from npu_sparse_attn_sharedkv_int8 import (CacheQuantization, PreparedCacheWrite, PreparedPageCompact,
                                               PreparedPageFork, PreparedPathCommit, PreparedTreeAttention, SharedKVCase)
    rng = np.random.default_rng(30)
    batch, nodes, heads, width, pages, depth, window = 5, 9, 4, 12, 70, 4, 128
    flat = torch.from_numpy(rng.integers(-127, 128, (pages, LAYERS * BLOCK * DIM)).astype(np.int8)).cuda()
    caches = [flat.view(-1).as_strided((pages, BLOCK, 1, DIM), (LAYERS * BLOCK * DIM, DIM, DIM, 1), k * BLOCK * DIM)
              for k in range(LAYERS)]
    quant = CacheQuantization(torch.from_numpy((0.02 + 0.01 * rng.random(DIM)).astype(np.float32)))
    scale, inverse = quant.scale.cuda(), quant.inverse_scale.cuda()

    # Sequences of different lengths on pages in mixed order.
    lengths = np.array([200, 3, 64, 95, 31])
    table, refs, order, at = np.full((batch, width), -1), np.zeros(pages, int), rng.permutation(pages), 0
    for b, n in enumerate(lengths):
        held = -(-n // BLOCK)
        table[b, :held] = order[at:at + held]
        refs[order[at:at + held]] = 1
        at += held
    mirror = [pool_rows(flat, table, b, n) for b, n in enumerate(lengths)]
    table, lens, refs = ints(table), ints(lengths), ints(refs)

    # One step's buffers; every operator keeps its arguments and works in place.
    children, total = ints(np.arange(batch)), torch.zeros(batch, dtype=torch.int32, device="cuda")
    drafts = [torch.zeros((batch * nodes, DIM), dtype=torch.bfloat16, device="cuda") for _ in range(LAYERS)]
    slots = torch.zeros(batch * nodes, dtype=torch.int64, device="cuda")
    q = torch.zeros((batch * nodes, heads, DIM), dtype=torch.bfloat16, device="cuda")
    parents, sink = ints(np.zeros(batch * nodes)), torch.linspace(-1, 1, heads, device="cuda")
    cu, paths, path_lens = ints(np.arange(batch + 1) * nodes), ints(np.zeros((batch, depth))), ints(np.zeros(batch))
    index = torch.arange(nodes, device="cuda")
    fork = PreparedPageFork(flat, table, lens, refs, children, room=nodes, output=(table, lens, refs))
    writers = [PreparedCacheWrite(cache, draft, slots, inverse) for cache, draft in zip(caches, drafts)]
    case = SharedKVCase(q, caches[1], table, cu, total, sink, window=window)
    tree = PreparedTreeAttention(case, parents, scale, return_lse=True)
    commit = PreparedPathCommit(caches, table, cu, total, paths, path_lens)
    compact = PreparedPageCompact([flat], table, refs, output=(table, refs))

    def draft_step():
        fork.run()
        torch.add(lens, nodes, out=total)
        place = lens[:, None].long() + index
        slots.copy_((table.gather(1, place // BLOCK).long() * BLOCK + place % BLOCK).flatten())
        for writer in writers:
            writer.run()
        tree.run()

    def accept_step():
        commit.run()
        lens.copy_(commit.seq_lens)
        compact.run()

    steps = [draft_step, accept_step]
    if captured:
        torch.cuda.synchronize()
        graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
        for graph, step in zip(graphs, steps):
            with torch.cuda.graph(graph):
                step()
        steps = [graph.replay for graph in graphs]

    for turn in range(6):
        chosen = np.arange(batch) if turn == 0 else rng.integers(0, batch, batch)     # some end, some go on twice
        trees = [[-1 if i == 0 else int(rng.integers(0, i)) for i in range(nodes)] for _ in range(batch)]
        values = rng.standard_normal((LAYERS, batch * nodes, DIM)).astype(np.float32)
        queries = rng.standard_normal((batch * nodes, heads, DIM)).astype(np.float32) * 2
        children.copy_(ints(chosen))
        parents.copy_(ints([p for row in trees for p in row]))
        for draft, value in zip(drafts, values):
            draft.copy_(torch.from_numpy(value))
        q.copy_(torch.from_numpy(queries))
        say(f"[speculative] turn {turn}: parents {chosen.tolist()}")
        steps[0]()
        torch.cuda.synchronize()
        assert fork.missing.item() == 0
        lengths = lengths[chosen]
        new = np.stack([quant.quantize(draft.cpu()).numpy() for draft in drafts]).reshape(LAYERS, batch, nodes, DIM)
        mirror = [np.concatenate([mirror[p], new[:, b]], 1) for b, p in enumerate(chosen)]
        held = table.cpu().numpy()
        for b in range(batch):
            np.testing.assert_array_equal(pool_rows(flat, held, b, lengths[b] + nodes), mirror[b])
        expect = Trees(0, [nodes] * batch, lengths.tolist(), heads=heads, ratio=1, window=window, parents=trees)
        expect.q, expect.sink = queries, sink.cpu().numpy()
        expect.ori = dict(pool=caches[1][:, :, 0].cpu().numpy(), table=held, scale=quant.scale.numpy())
        compare(tree, expect, True)

        # Accept a path from a root down.
        accepted = []
        for row in trees:
            path = [int(rng.integers(0, nodes))]
            while row[path[0]] >= 0:
                path.insert(0, row[path[0]])
            accepted.append(path[:depth])
        paths.copy_(ints([p + [-1] * (depth - len(p)) for p in accepted]))
        path_lens.copy_(ints([len(p) for p in accepted]))
        steps[1]()
        torch.cuda.synchronize()
        mirror = [np.concatenate([m[:, :n], m[:, n:][:, p]], 1) for m, n, p in zip(mirror, lengths, accepted)]
        lengths = lengths + np.array([len(p) for p in accepted])
        np.testing.assert_array_equal(lens.cpu().numpy(), lengths)
        held, counts, live = table.cpu().numpy(), refs.cpu().numpy(), compact.live.item()
        assert (counts[:live] > 0).all() and (counts[live:] == 0).all()
        np.testing.assert_array_equal(np.bincount(held[held >= 0], minlength=pages), counts)
        for b in range(batch):
            np.testing.assert_array_equal(pool_rows(flat, held, b, lengths[b]), mirror[b])


@pytest.mark.parametrize("ratio", [1, 128])
def test_adapter_call(ratio):
    """SharedKVLayer.attention with tree_parents, eager and captured, with an ordinary call on the same layer between."""
    import torch
    from npu_sparse_attn_sharedkv_int8 import vllm_adapter
    trees = Trees(31, [7, 12], [500, 4000], ratio=ratio)
    case, parents, scale, cmp_scale = trees.device()
    impl = SimpleNamespace(swa_cache_layer=SimpleNamespace(prefix="unit.swa_cache"), head_dim=512)
    layer = vllm_adapter.runtime(impl)
    layer.device_scales = {("ori", case.q.device): (scale, None), ("cmp", case.q.device): (cmp_scale, None)}
    kw = dict(ori_kv=case.ori, cmp_kv=case.cmp, ori_block_table=case.ori_block_table,
              cmp_block_table=case.cmp_block_table, cu_seqlens_q=case.cu_q, seqused_kv=case.seq_lens, sinks=case.sink,
              cmp_ratio=ratio, ori_win_left=127, softmax_scale=1 / math.sqrt(DIM), layout_q="TND", layout_kv="PA_ND",
              return_softmax_lse=True)
    say(f"[adapter] trees, ratio {ratio}")
    check = lambda out, lse: compare(SimpleNamespace(out=out, lse=lse.squeeze(-1)), trees, True)  # noqa: E731
    check(*layer.attention(case.q, tree_parents=parents, **kw))
    layer.attention(case.q, **kw)                              # the window operator of the same shape is another one
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = layer.attention(case.q, tree_parents=parents, **kw)
    for _ in range(3):
        out.fill_(float("nan"))
        graph.replay()
        layer.attention(case.q, **kw)
        torch.cuda.synchronize()
        check(out, lse)
    out, lse = layer.attention(case.q, tree_parents=parents, **dict(kw, return_softmax_lse=False))
    assert lse.numel() == 0 and out.shape == case.q.shape
    with pytest.raises(ValueError, match="ratio 4"):
        layer.attention(case.q, tree_parents=parents,
                        **dict(kw, cmp_ratio=4, cmp_kv=case.ori, cmp_block_table=case.ori_block_table,
                               cmp_sparse_indices=torch.zeros(19, 1, 8, dtype=torch.int32, device="cuda")))
