"""PreparedBlockAttention on prompts into empty caches, whose split units differ
most in the rows they see (test_block_plan_host.PROMPTS), against 64 bits."""
import pytest

from tests.block_cases import Attend
from tests.test_block_plan_host import PROMPTS
from tests.test_gpu_block_attention import check, KINDS

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("case", PROMPTS, ids=lambda c: f"{c['new'][0]}x{len(c['new'])}_{c['heads']}_{c['kv_heads']}")
def test_prompts(kind, case):
    op = check(Attend(31, case["new"], case["lengths"], heads=case["heads"], kv_heads=case["kv_heads"],
                      ratio=case["ratio"], window=case["window"], kind=kind))
    assert op.partial is not None
