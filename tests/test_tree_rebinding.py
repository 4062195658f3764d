"""PreparedTreeAttention._rebind_same_geometry on the host, without a device: it
refuses what the constructor refuses, and leaves the operator as it was."""
import pytest
import torch

from npu_sparse_attn_sharedkv_int8 import PreparedTreeAttention, SharedKVCase, runtime, tree

TOKENS, HEADS, BATCH = 6, 2, 2


def aligned(x):
    """A copy of x on a 16-byte boundary."""
    room = torch.empty(x.numel() * x.element_size() + 16, dtype=torch.uint8)
    at = -room.data_ptr() % 16
    return room[at:at + x.numel() * x.element_size()].view(x.dtype).view(x.shape).copy_(x)


def off_by(x, count):
    return aligned(torch.empty(x.numel() + count, dtype=x.dtype))[count:].view(x.shape)


def inputs(ratio=128):
    cache = lambda pages: aligned(torch.zeros((pages, 32, 1, 512), dtype=torch.int8))  # noqa: E731
    table = lambda width: torch.zeros((BATCH, width), dtype=torch.int32)  # noqa: E731
    case = SharedKVCase(aligned(torch.zeros((TOKENS, HEADS, 512), dtype=torch.bfloat16)), cache(4), table(3),
                        torch.tensor([0, 2, TOKENS], dtype=torch.int32), torch.tensor([40, 9], dtype=torch.int32),
                        torch.zeros(HEADS), cache(2) if ratio > 1 else None, table(1) if ratio > 1 else None, None,
                        ratio=ratio, window=128, softmax_scale=0.04)
    return case, torch.full((TOKENS,), -1, dtype=torch.int32)


@pytest.fixture
def bound(monkeypatch):
    """An operator as the constructor leaves it, but for the launcher and the scratch."""
    monkeypatch.setattr(tree, "_check_query", lambda q: None, raising=False)      # asks for a GPU
    case, parents = inputs()
    op = object.__new__(PreparedTreeAttention)
    op.scales = tuple(aligned(torch.ones(512)) for _ in range(2))
    op.args = runtime.TreeAttentionArgs()
    if hasattr(tree, "_check_inputs"):
        op.geometry, op.layout = tree._check_inputs(case, parents, *op.scales), tree._layout(case, parents)
    op.case, op.parents, op.out, op.lse = case, parents, aligned(torch.empty_like(case.q)), None
    op._bind()
    return op


def refused(op, match, case=None, parents=None, **kw):
    fresh, fresh_parents = inputs()
    before, held = bytes(op.args), (op.case, op.parents, op.out, op.lse)
    with pytest.raises(ValueError, match=match):
        op._rebind_same_geometry(case or fresh, fresh_parents if parents is None else parents, **kw)
    assert bytes(op.args) == before and all(a is b for a, b in zip(held, (op.case, op.parents, op.out, op.lse)))


def test_a_good_rebinding(bound):
    case, parents = inputs()
    out, lse = aligned(torch.empty_like(case.q)), torch.empty((TOKENS, HEADS))
    bound._rebind_same_geometry(case, parents, output=out, lse_output=lse)
    assert bound.args.q == case.q.data_ptr() and bound.args.parents == parents.data_ptr()
    assert bound.args.out == out.data_ptr() and bound.args.lse == lse.data_ptr()


@pytest.mark.parametrize("match,make", [
    ("metadata", lambda p: p.long()),                                  # would be read as twice as many words
    ("metadata", lambda p: p.float()),
    ("parents", lambda p: p[:-1]),                                     # would be read past its end
    ("parents", lambda p: p[:, None]),
    ("metadata", lambda p: torch.zeros(2 * TOKENS, dtype=torch.int32)[::2]),
    ("metadata", lambda p: p.to("meta")),                              # of another device
    ("parents", lambda p: p.tolist()),
], ids=["int64", "float", "short", "2d", "strided", "device", "list"])
def test_parents_are_checked(bound, match, make):
    refused(bound, match, parents=make(inputs()[1]))


@pytest.mark.parametrize("field,match,make", [
    ("seq_lens", "metadata", lambda t: t.long()), ("cu_q", "metadata", lambda t: t.float()),
    ("cu_q", "metadata", lambda t: t[:-1]), ("sink", "metadata", lambda t: t[:-1]),
    ("ori_block_table", "block table", lambda t: t.long()), ("ori_block_table", "block table", lambda t: t[:1]),
    ("cmp_block_table", "block table", lambda t: torch.zeros((1, BATCH), dtype=torch.int32).T.expand(BATCH, 2)[:, :1].T),
    ("ori_block_table", "every size", lambda t: torch.zeros((BATCH, 2), dtype=torch.int32)),
    ("ori", "INT8", lambda t: t.float()), ("ori", "every size", lambda t: t[:3]), ("cmp", "INT8", lambda t: None),
    ("q", "every size", lambda t: t[:, :1].contiguous()), ("ori", "16-byte", lambda t: off_by(t, 8)),
    ("cmp", "16-byte", lambda t: off_by(t, 8)), ("window", "every size", lambda w: 64),
    ("window", "window", lambda w: 0), ("softmax_scale", "every size", lambda x: 0.05),
    ("ratio", "every size", lambda r: 1), ("ratio", "ratio 4", lambda r: 4)])
def test_the_case_is_checked(bound, field, match, make):
    case, parents = inputs()
    setattr(case, field, make(getattr(case, field)))
    if field == "q":
        case.sink = case.sink[:1]
    refused(bound, match, case=case, parents=parents)


def test_outputs_are_checked(bound):
    case, parents = inputs()
    refused(bound, "output", case=case, parents=parents, output=torch.empty((TOKENS, HEADS, 512)))
    refused(bound, "overlap", case=case, parents=parents, output=case.q)
    refused(bound, "LSE", case=case, parents=parents, output=aligned(torch.empty_like(case.q)),
            lse_output=torch.empty((TOKENS, HEADS + 1)))
    bound.out = None                                                   # an operator whose caller took its output
    refused(bound, "output", case=case, parents=parents)


@pytest.mark.parametrize("field", ["ori", "cmp", "ori_block_table", "cmp_block_table", "cu_q", "seq_lens", "sink", "q"])
@pytest.mark.parametrize("which", ["output", "lse_output"])
def test_outputs_over_any_input_are_refused(bound, field, which):
    """Also an output that lies between the first and the last byte of pages with room between them."""
    case, parents = inputs()
    good = dict(output=aligned(torch.empty_like(case.q)), lse_output=torch.empty((TOKENS, HEADS)))
    count = {name: x.nbytes for name, x in good.items()}[which]
    held = getattr(case, field)
    # The input at the end of a buffer whose start is the output, a few bytes of it shared.
    room = aligned(torch.zeros(count + held.nbytes, dtype=torch.int8))
    at = count - 16
    moved = room[at:at + held.nbytes].view(held.dtype).view(held.shape).copy_(held)
    setattr(case, field, moved)
    refused(bound, "overlap", case=case, parents=parents,
            **dict(good, **{which: room[:count].view(good[which].dtype).view(good[which].shape)}))


@pytest.mark.parametrize("which", [0, 1])
def test_outputs_over_a_scale_are_refused(bound, which):
    case, parents = inputs()
    lse = bound.scales[which][100:100 + TOKENS * HEADS].view(TOKENS, HEADS)
    refused(bound, "overlap", case=case, parents=parents, output=aligned(torch.empty_like(case.q)), lse_output=lse)


def test_bytes_between_pages_count_as_the_caches():
    from npu_sparse_attn_sharedkv_int8 import pages
    flat = torch.zeros(4 * 100, dtype=torch.int8)
    strided = flat.as_strided((3, 32), (100, 1))
    assert pages._extent(strided) == 232 and pages._extent(flat) == 400 and pages._extent(flat[:0]) == 0
    assert pages._overlap(flat[40:50], strided) and pages._overlap(strided, flat[231:]) and not pages._overlap(strided, flat[232:])
    assert not pages._overlap(flat[:10], flat[10:]) and pages._overlap(flat[:11].view(torch.int8), flat[10:])
