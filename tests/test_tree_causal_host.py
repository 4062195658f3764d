"""The rule for compressed rows, without a device: the C entry's field, and the serving call's choice."""
import ctypes

import pytest
import torch

from npu_sparse_attn_sharedkv_int8 import runtime, vllm_adapter
from tests.test_tree_pages_host import INVALID, good_tree
from tests.test_tree_rebinding import HEADS, TOKENS, aligned, inputs


def test_the_field_is_zero_or_one():
    lib, sizes = runtime.library(), (ctypes.c_uint64(), ctypes.c_uint64())
    for value, code in ((0, 0), (1, 0), (2, INVALID), (1 << 31, INVALID)):
        a = good_tree()
        a.causalCompressed = value
        assert lib.sharedkv_tree_scratch(ctypes.addressof(a), *map(ctypes.byref, sizes)) == code
    a.causalCompressed, a.ratio = 1, 1 << 31
    assert lib.sharedkv_tree_scratch(ctypes.addressof(a), *map(ctypes.byref, sizes)) == INVALID


@pytest.mark.parametrize("ratio", [1, 128])
def test_serving_calls_with_trees_are_causal(monkeypatch, ratio):
    """As cmp_mask_mode 3, the only one that the call takes, says of every token."""
    made = []

    class Operator:
        def __init__(self, case, parents, *scales, **kw):
            made.append(kw)

        def run(self):
            pass

    monkeypatch.setattr(vllm_adapter, "PreparedTreeAttention", Operator)
    monkeypatch.setattr(vllm_adapter, "stream_key", lambda device: 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    layer = vllm_adapter.SharedKVLayer(vllm_adapter.LayerDescription(prefix="unit"))
    layer.device_scales = {(kind, torch.device("cpu")): (aligned(torch.ones(512)), None) for kind in ("ori", "cmp")}
    case, parents = inputs(ratio)
    out, _ = layer.attention(case.q, tree_parents=parents, ori_kv=case.ori, cmp_kv=case.cmp,
                             ori_block_table=case.ori_block_table, cmp_block_table=case.cmp_block_table,
                             cu_seqlens_q=case.cu_q, seqused_kv=case.seq_lens, sinks=case.sink, cmp_ratio=ratio,
                             ori_win_left=127, softmax_scale=0.04, layout_q="TND", layout_kv="PA_ND", cmp_mask_mode=3)
    assert out.shape == (TOKENS, HEADS, 512) and len(made) == 1 and made[0]["causal_compressed"] is True
