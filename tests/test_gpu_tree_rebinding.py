"""Tree operators bound to new tensors: by hand, and as every serving call after
the first of its shape finds one.  Results against 64 bits (bounds of
test_gpu_tree.py)."""
import math
import sys
from types import SimpleNamespace

import numpy as np
import pytest

from tests.test_gpu_tree import BLOCK, DIM, Trees, compare

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, file=sys.stderr, flush=True)


def alike(*trees):
    """Tables and pools of one size, and the first one's scales, so that one operator serves them all."""
    for name in ("ori", "cmp"):
        kinds = [getattr(t, name) for t in trees if getattr(t, name) is not None]
        width = max((k["table"].shape[1] for k in kinds), default=0)
        pages = max((len(k["pool"]) for k in kinds), default=0)
        for kind in kinds:
            kind["table"] = np.pad(kind["table"], ((0, 0), (0, width - kind["table"].shape[1])), constant_values=-1)
            kind["pool"] = np.resize(kind["pool"], (pages, BLOCK, DIM))
            kind["scale"] = kinds[0]["scale"]
    return trees


@pytest.mark.parametrize("ratio", [1, 128])
@pytest.mark.parametrize("lse", [False, True], ids=["out", "lse"])
def test_new_tensors(ratio, lse):
    import torch
    from npu_sparse_attn_sharedkv_int8 import PreparedTreeAttention
    first, second = alike(Trees(40, [7, 12], [500, 4000], ratio=ratio), Trees(41, [12, 7], [100, 4100], ratio=ratio))
    case, parents, scale, cmp_scale = first.device()
    other, other_parents, _, _ = second.device()
    op = PreparedTreeAttention(case, parents, scale, cmp_scale, return_lse=lse)
    say(f"[rebinding] first tensors, ratio {ratio}")
    op.run()
    torch.cuda.synchronize()
    compare(op, first, lse)
    kept, kept_lse = op.out, op.lse
    before = kept.clone()
    out = torch.full_like(other.q, float("nan"))
    out_lse = torch.full(other.q.shape[:2], float("nan"), device="cuda") if lse else None
    op._rebind_same_geometry(other, other_parents, output=out, lse_output=out_lse)
    say("[rebinding] second tensors")
    assert op.run() is out
    torch.cuda.synchronize()
    compare(op, second, lse)
    assert torch.equal(kept, before) and (kept_lse is None or not lse or op.lse is out_lse)
    op._rebind_same_geometry(case, parents)                    # the outputs stay
    op.out.fill_(float("nan"))
    say("[rebinding] first tensors again")
    assert op.run() is out
    torch.cuda.synchronize()
    compare(op, first, lse)


@pytest.mark.parametrize("nodes,committed,heads", [([7, 12], [500, 4000], 8), ([16] * 30, [0, 17, 128, 500, 9000, 700] * 5, 64)])
def test_the_log_sum_exp_comes_and_goes(nodes, committed, heads):
    """Outputs with and without it, bound in turn to one operator: its scratch serves both kernels."""
    import torch
    from npu_sparse_attn_sharedkv_int8 import PreparedTreeAttention
    trees = Trees(42, nodes, committed, heads=heads)
    case, parents, scale, cmp_scale = trees.device()
    op = PreparedTreeAttention(case, parents, scale, cmp_scale)
    for lse in (False, True, False):
        out = torch.full_like(case.q, float("nan"))
        op._rebind_same_geometry(case, parents, output=out, lse_output=torch.full(
            case.q.shape[:2], float("nan"), device="cuda") if lse else None)
        say(f"[rebinding] {len(nodes)} requests, lse={lse}")
        op.run()
        torch.cuda.synchronize()
        compare(op, trees, lse)


def adapter(scale, cmp_scale):
    from npu_sparse_attn_sharedkv_int8 import vllm_adapter
    impl = SimpleNamespace(swa_cache_layer=SimpleNamespace(prefix="unit.swa_cache"), head_dim=512)
    layer = vllm_adapter.runtime(impl)
    layer.device_scales = {("ori", scale.device): (scale, None)}
    if cmp_scale is not None:
        layer.device_scales["cmp", scale.device] = cmp_scale, None
    return layer


def call(case, **more):
    return dict(dict(ori_kv=case.ori, cmp_kv=case.cmp, ori_block_table=case.ori_block_table,
                     cmp_block_table=case.cmp_block_table, cu_seqlens_q=case.cu_q, seqused_kv=case.seq_lens,
                     sinks=case.sink, cmp_ratio=case.ratio, ori_win_left=case.window - 1,
                     softmax_scale=1 / math.sqrt(DIM), layout_q="TND", layout_kv="PA_ND", return_softmax_lse=True), **more)


@pytest.mark.parametrize("ratio", [1, 128])
def test_adapter_calls_of_one_shape(ratio):
    """Calls of one shape on one stream share an operator, with their own queries, trees, lengths, tables and caches."""
    import torch
    trees = alike(*(Trees(50 + i, nodes, committed, ratio=ratio) for i, (nodes, committed) in enumerate(
        [([7, 12], [500, 4000]), ([12, 7], [100, 4100]), ([9, 10], [3000, 0]), ([18, 1], [129, 2000])])))
    calls = [t.device() for t in trees]
    layer = adapter(calls[0][2], calls[0][3])
    for t, (case, parents, _, _) in zip(trees, calls):
        say(f"[rebinding] adapter call over {t.committed} rows, ratio {ratio}")
        out, lse = layer.attention(case.q, tree_parents=parents, **call(case))
        torch.cuda.synchronize()
        compare(SimpleNamespace(out=out, lse=lse.squeeze(-1)), t, True)
        assert len(layer.operators.values()) == 1


def test_adapter_refuses_other_parents_on_every_call():
    import torch
    trees = Trees(60, [7, 12], [500, 4000])
    case, parents, scale, cmp_scale = trees.device()
    layer = adapter(scale, cmp_scale)
    say("[rebinding] adapter, good and bad parents")
    for again in range(2):                                     # on an operator of the first call, then on a bound one
        out, lse = layer.attention(case.q, tree_parents=parents, **call(case))
        for bad in (parents.long(), parents[:-1], parents.cpu(), parents.repeat_interleave(2)[::2], parents[:, None]):
            with pytest.raises(ValueError, match="parents|metadata"):
                layer.attention(case.q, tree_parents=bad, **call(case))
        with pytest.raises(ValueError, match="contiguous"):
            layer.attention(case.q.transpose(0, 1).contiguous().transpose(0, 1), tree_parents=parents, **call(case))
        torch.cuda.synchronize()
        compare(SimpleNamespace(out=out, lse=lse.squeeze(-1)), trees, True)
