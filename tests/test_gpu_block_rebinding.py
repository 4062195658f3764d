"""Outputs of PreparedBlockAttention._rebind_same_geometry: each new one is taken,
whichever is given, and the others stay."""
import pytest

from tests.block_cases import Attend
from tests.test_gpu_block_attention import compare

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new_out,new_lse", [(False, False), (True, False), (False, True), (True, True)])
def test_outputs_given_one_by_one(new_out, new_lse):
    import torch
    from npu_sparse_attn_sharedkv_int8 import PreparedBlockAttention
    attend, other = Attend(70, [2, 1], [300, 90]), Attend(70, [2, 1], [300, 90])
    other.q += 1
    case, scale, _ = attend.device()
    op = PreparedBlockAttention(case, scale, return_lse=True)
    op.run()
    old, old_lse = op.out, op.lse
    out = torch.full_like(old, 7) if new_out else None
    lse = torch.full_like(old_lse, 7) if new_lse else None
    theirs, scale, _ = other.device()
    op._rebind_same_geometry(theirs, scale, output=out, lse_output=lse)
    op.run()
    assert op.out is (out if new_out else old) and op.lse is (lse if new_lse else old_lse)
    compare(other, op.out, op.lse, other.expect())
    # What was replaced is left as it was.
    want, near, want_lse, lse_near = attend.expect()
    if new_out:
        compare(attend, old, None, (want, near, want_lse, lse_near))
    if new_lse:
        assert (abs(old_lse.double().cpu().numpy() - want_lse) <= lse_near).all()


def test_a_log_sum_exp_where_there_was_none():
    import torch
    from npu_sparse_attn_sharedkv_int8 import PreparedBlockAttention
    attend = Attend(71, [1], [5000])
    case, scale, _ = attend.device()
    op = PreparedBlockAttention(case, scale)
    op.run()
    assert op.lse is None
    lse = torch.zeros(case.q.shape[:2], device="cuda")
    op._rebind_same_geometry(case, lse_output=lse)
    op.run()
    compare(attend, op.out, lse, attend.expect())
    with pytest.raises(ValueError):
        op._rebind_same_geometry(case, lse_output=lse[:, :4])
    with pytest.raises(ValueError):
        op._rebind_same_geometry(case, lse_output=op.out.view(-1)[:16].view(torch.float32).view(1, 8))
