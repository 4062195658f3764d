"""Sinks at their limits and large scores, outputs and log-sum-exps of both kernels (16-bit codes, and 24 bits with the
log-sum-exp), against 64 bits.

The bounds of test_gpu_tree.py hold as they are: a sink enters as sink * log2 e, and a log-sum-exp leaves times ln 2.  The
two constants and the two products are off by half a step each, 2^-24 of the value, 2^-22 |sink| together, which is the
2^-22 |lse| of the bound in rows that the sink dominates.  In others the sink's share is off by 2^-23 |sink| of itself, less
than 2^-20 for a sink that is not negligible beside scores of its own size (|sink| <= 3 here)."""
import sys

import numpy as np
import pytest

from tests.test_gpu_tree import Trees, compare

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, file=sys.stderr, flush=True)


@pytest.mark.parametrize("lse", [False, True], ids=["out", "lse"])
@pytest.mark.parametrize("q_size,nodes,committed", [(40.0, [6], [300]), (1.0, [6, 3], [300, 9000]), (1.0, [1], [0])])
def test_sinks(lse, q_size, nodes, committed):
    import torch
    from npu_sparse_attn_sharedkv_int8 import PreparedTreeAttention
    trees = Trees(90, nodes, committed, heads=6, q_size=q_size)
    trees.sink = np.array([-np.inf, 3.0, -1e30, 1e30, 0.0, -3.0], np.float32)
    case, parents, scale, cmp_scale = trees.device()
    op = PreparedTreeAttention(case, parents, scale, cmp_scale, return_lse=lse)
    op.out.fill_(float("nan"))
    if lse:
        op.lse.fill_(float("nan"))
    say(f"[sinks] {nodes} tokens, q {q_size}, lse={lse}")
    op.run()
    torch.cuda.synchronize()
    compare(op, trees, lse)
    assert (op.out[:, 3] == 0).all()
    if lse:
        assert not op.lse.isnan().any()


@pytest.mark.parametrize("lse", [False, True], ids=["out", "lse"])
def test_neither_key_nor_sink(lse):
    import torch
    from npu_sparse_attn_sharedkv_int8 import PreparedTreeAttention
    trees = Trees(91, [6], [300], heads=2)
    case, parents, scale, cmp_scale = trees.device()
    case.sink = torch.tensor([-float("inf"), 2.0], device="cuda")
    case.ori_block_table.fill_(-1)
    case.cmp_block_table.fill_(-1)
    op = PreparedTreeAttention(case, parents, scale, cmp_scale, return_lse=lse)
    op.out.fill_(float("nan"))
    say(f"[sinks] no keys, lse={lse}")
    op.run()
    torch.cuda.synchronize()
    assert (op.out == 0).all()
    if lse:
        assert (op.lse[:, 0] == -float("inf")).all() and ((op.lse[:, 1] - 2.0).abs() <= 2 ** -20 + 2 ** -21).all()
