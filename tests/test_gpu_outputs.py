"""Outputs of the tree and page operators that lie over what the operators read: refused by the constructors."""
import pytest

from tests.test_gpu_pages import ints
from tests.test_gpu_tree import Trees

pytestmark = pytest.mark.gpu


def test_page_operators_refuse_outputs_over_caches():
    import torch
    from npu_sparse_attn_sharedkv_int8 import PreparedPageCompact, PreparedPageFork, PreparedPathCommit
    # A pool of 9 pages of 32 rows, seen as INT32 where an output would lie in it.
    words = torch.zeros(9 * 32 * 128, dtype=torch.int32, device="cuda")
    cache = words.view(torch.int8).view(9, 32, 512)
    table, seq, refs, parents = ints([[0, 1], [2, 3]]), ints([3, 40]), ints([1] * 4 + [0] * 5), ints([0, 1])
    cu, paths, lens = ints([0, 1, 2]), ints([[0], [0]]), ints([1, 1])
    calls = [
        lambda: PreparedPathCommit(cache, table, cu, seq, paths, lens, output=words[100:102]),
        lambda: PreparedPageFork(cache, table, seq, refs, parents, output=(words[:4].view(2, 2), None, None)),
        lambda: PreparedPageFork(cache, table, seq, refs, parents, output=(None, words[-2:], None)),
        lambda: PreparedPageFork(cache, table, seq, refs, parents, output=(None, None, words[64:73])),
        lambda: PreparedPageCompact(cache, table, refs, output=(words[:4].view(2, 2), None)),
        lambda: PreparedPageCompact(cache, table, refs, output=(None, words[64:73])),
    ]
    for call in calls:
        with pytest.raises(ValueError, match="overlap|own"):
            call()


def test_tree_operators_refuse_outputs_over_their_inputs():
    import torch
    from npu_sparse_attn_sharedkv_int8 import PreparedTreeAttention
    trees = Trees(21, [4, 4], [300, 1000])
    case, parents, scale, cmp_scale = trees.device()
    size = 8 * 8 * 512
    for cache in (case.ori, case.cmp):
        with pytest.raises(ValueError, match="overlap"):
            PreparedTreeAttention(case, parents, scale, cmp_scale,
                                  output=cache.view(-1)[:2 * size].view(torch.bfloat16).view(8, 8, 512))
    for one in (scale, cmp_scale):
        with pytest.raises(ValueError, match="overlap"):
            PreparedTreeAttention(case, parents, scale, cmp_scale, lse_output=one[:64].view(8, 8))
    case.ori_block_table = torch.nn.functional.pad(case.ori_block_table, (0, 64 - case.ori_block_table.shape[1]), value=-1)
    with pytest.raises(ValueError, match="overlap"):
        PreparedTreeAttention(case, parents, scale, cmp_scale,
                              lse_output=case.ori_block_table.view(torch.float32).view(-1)[:64].view(8, 8))
