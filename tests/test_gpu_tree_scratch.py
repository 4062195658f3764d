"""Scratch that a caller hands to tree operators: cleared in the order of the stream that runs them, without a wait."""
import sys
from types import SimpleNamespace

import pytest

from tests.test_gpu_tree import Trees, compare
from tests.test_gpu_tree_rebinding import adapter, call

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, file=sys.stderr, flush=True)


def test_operators_of_a_serving_loop_wait_for_nothing(monkeypatch):
    """Calls of new shapes build operators; their scratch, shared and dirty, is cleared by the first run."""
    import torch
    from npu_sparse_attn_sharedkv_int8 import vllm_adapter
    trees = [Trees(80 + i, nodes, committed) for i, (nodes, committed) in enumerate(
        [([7, 12], [500, 4000]), ([5], [100]), ([9, 2, 3], [3000, 0, 77])])]
    calls = [t.device() for t in trees]
    layer = adapter(calls[0][2], calls[0][3])
    for t in trees:
        for name in ("ori", "cmp"):
            getattr(t, name)["scale"] = getattr(trees[0], name)["scale"]
    device = calls[0][0].q.device
    vllm_adapter.scratch_allocator("tree_workspace", (1 << 12,), torch.int32, device).fill_(7)
    vllm_adapter.scratch_allocator("tree_partial", (1 << 24,), torch.float32, device).fill_(float("nan"))
    torch.cuda.synchronize()
    results = []
    say("[scratch] three shapes, no wait")
    with monkeypatch.context() as m:
        def waited(*a):
            raise AssertionError("the call waited for the stream")
        m.setattr(torch.cuda.Stream, "synchronize", waited)
        m.setattr(torch.cuda, "synchronize", waited)
        for again in range(2):
            for case, parents, _, _ in calls:
                results.append(layer.attention(case.q, tree_parents=parents, **call(case)))
    torch.cuda.synchronize()
    assert len(layer.operators.values()) == 3 and all(op.partial is not None for op in layer.operators.values())
    for i, (out, lse) in enumerate(results):
        compare(SimpleNamespace(out=out, lse=lse.squeeze(-1)), trees[i % 3], True)


def test_scratch_of_one_allocator_on_its_stream():
    """Two operators that share their scratch, one behind the other on a stream that neither was made on."""
    import torch
    from npu_sparse_attn_sharedkv_int8 import PreparedTreeAttention
    pair = [Trees(83, [7, 12], [500, 4000]), Trees(84, [16], [12000])]
    held = {"tree_workspace": torch.full((1 << 10,), 7, dtype=torch.int32, device="cuda"),
            "tree_partial": torch.full((1 << 23,), float("nan"), device="cuda")}
    ops = []
    for t in pair:
        case, parents, scale, cmp_scale = t.device()
        ops.append(PreparedTreeAttention(case, parents, scale, cmp_scale, return_lse=True,
                                         scratch_allocator=lambda name, shape, dtype, device: held[name][:shape[0]]))
        ops[-1].out.fill_(float("nan"))
    assert all(op.partial is not None for op in ops)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    say("[scratch] two operators in turn")
    with torch.cuda.stream(side):
        for _ in range(3):
            for op in ops:
                op.run()
    torch.cuda.synchronize()
    for op, t in zip(ops, pair):
        compare(op, t, True)
    assert (held["tree_workspace"][:64] == 0).any() and not ops[0]._unclear


@pytest.mark.parametrize("lse", [False, True], ids=["out", "lse"])
def test_repeated_runs_agree_bit_for_bit(lse):
    """Whichever of a unit's items ends last joins them, in the items' order."""
    import torch
    from npu_sparse_attn_sharedkv_int8 import PreparedTreeAttention
    trees = Trees(85, [7, 12, 16], [500, 4000, 12000], ratio=1, window=1 << 30)
    case, parents, scale, cmp_scale = trees.device()
    op = PreparedTreeAttention(case, parents, scale, cmp_scale, return_lse=lse)
    assert op.partial is not None
    say(f"[scratch] twenty runs, lse={lse}")
    op.run()
    first = [x.clone() for x in (op.out, op.lse) if x is not None]
    for _ in range(20):
        op.out.fill_(float("nan"))
        op.run()
        assert all(torch.equal(a, b) for a, b in zip(first, (op.out, op.lse)))
    compare(op, trees, lse)
