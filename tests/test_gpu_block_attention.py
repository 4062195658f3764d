"""PreparedBlockAttention against attention in 64 bits (block_cases.Attend, whose
expect() derives the bounds)."""
import math
import sys
import zlib

import numpy as np
import pytest

from tests import block_cases as cases
from tests.block_cases import ALL, Attend, BLOCK, DIM

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, file=sys.stderr, flush=True)


def compare(attend, out, lse, expected):
    want, near, want_lse, lse_near = expected
    got = out.float().cpu().numpy().astype(np.float64)
    off = np.abs(got - want) - near
    assert np.isfinite(got).all() and off.max() <= 0, (off.max(), np.unravel_index(off.argmax(), off.shape))
    if lse is not None:
        off = np.abs(lse.cpu().numpy().astype(np.float64) - want_lse) - lse_near
        assert off.max() <= 0, (off.max(), np.unravel_index(off.argmax(), off.shape))


def run(attend, **kw):
    import torch
    from npu_sparse_attn_sharedkv_int8 import PreparedBlockAttention
    case, ori_scale, cmp_scale = attend.device()
    op = PreparedBlockAttention(case, ori_scale, cmp_scale, return_lse=True, **kw)
    op.out.fill_(7)
    op.lse.fill_(7)
    if op.partial is not None:
        op.partial.fill_(math.nan)
        op.units.fill_(12345)
    op.run()
    torch.cuda.synchronize()
    return op


def check(attend):
    op = run(attend)
    compare(attend, op.out, op.lse, attend.expect())
    return op


KINDS = ["int8", "e4m3"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new,lengths", [
    ([1], [1]), ([1], [2]), ([1], [32]), ([1], [33]), ([1], [64]), ([1], [65]), ([1], [1000]), ([1], [5000]),
    ([2], [129]), ([5], [5]), ([9], [300]), ([40], [40]), ([65], [131]), ([130], [700]),
    ([1, 1, 1], [1, 77, 2000]), ([1, 3, 20, 1], [500, 3, 20, 64]), ([0, 4, 0, 1], [9, 90, 0, 33])], ids=str)
def test_lengths(kind, new, lengths):
    check(Attend(zlib.crc32(f"{kind}{new}{lengths}".encode()), new, lengths, kind=kind))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (2, 1), (5, 1), (16, 1), (17, 1), (64, 1), (128, 1), (8, 2), (12, 4), (8, 8), (30, 3)])
def test_heads(kind, heads, kv_heads):
    check(Attend(heads + kv_heads, [1, 3], [200, 333], kind=kind, heads=heads, kv_heads=kv_heads))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("window", [1, 2, 31, 33, 128, 200, 1000])
@pytest.mark.parametrize("ratio", [1, 128])
def test_windows_and_compressed_rows(kind, window, ratio):
    check(Attend(window, [1, 2, 70, 1], [127, 128, 700, 4500], kind=kind, window=window, ratio=ratio))


@pytest.mark.parametrize("kind", KINDS)
def test_strided_pages_with_scales_behind_them(kind):
    check(Attend(3, [2, 1], [300, 900], kind=kind, behind=160, ratio=128, window=128, heads=16, kv_heads=2))


@pytest.mark.parametrize("kind", KINDS)
def test_scales_far_apart(kind):
    # e^+-12: a page's values are up to 10^10 times another's.
    check(Attend(4, [3, 1], [400, 3000], kind=kind, spread=12.0, q_size=1e-4))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("softmax_scale,q_size", [(-1 / 22.0, 1.0), (1 / 22.0, 30.0), (1.0, 1e-3), (1e-9, 1.0), (0.0, 1.0)])
def test_softmax_scales(kind, softmax_scale, q_size):
    check(Attend(5, [2, 20], [300, 200], kind=kind, softmax_scale=softmax_scale, q_size=q_size))


@pytest.mark.parametrize("kind", KINDS)
def test_padding(kind):
    attend = Attend(6, [3, 40], [100, 90], kind=kind, pad_tokens=70, pad_batch=3)
    op = check(attend)
    assert not op.out[43:].any() and not op.lse[43:].any()


@pytest.mark.parametrize("kind", KINDS)
def test_a_request_without_rows_and_one_of_fewer_rows_than_tokens(kind):
    attend = Attend(7, [2, 6, 40], [0, 4, 30], kind=kind)
    op = check(attend)
    assert not op.out[:2].any() and not op.lse[:2].any()
    assert not op.out[2:4].any()                            # tokens below row 0 see nothing


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads", [8, 64])
def test_missing_pages(kind, heads):
    attend = Attend(8, [2, 30], [400, 333], kind=kind, heads=heads)
    attend.ori_table[0, [0, 3, 12]] = [-1, 10 ** 6, -7]
    attend.ori_table[1, :] = -1
    check(attend)
    attend = Attend(9, [1], [500], kind=kind, heads=heads)
    attend.ori_table = np.ascontiguousarray(attend.ori_table[:, :7])      # rows past the table
    check(attend)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads", [8, 32, 64])
def test_what_masked_rows_hold_reaches_nothing(kind, heads):
    """NaN codes and scales behind a request's rows, on pages of no request, and in rows that only later tokens see."""
    new, lengths = [1, 40, 3], [70, 100, 260]
    attend = Attend(10, new, lengths, kind=kind, heads=heads, window=100, ratio=128)
    named = np.unique(attend.ori_table[attend.ori_table >= 0])
    free = np.setdiff1d(np.arange(len(attend.ori.codes)), named)
    expected = attend.expect()
    bad = 127 if kind == "e4m3" else 128
    for b, n in enumerate(lengths):
        attend.ori.codes[attend.ori_table[b, (n - 1) // BLOCK], (n - 1) % BLOCK + 1:] = bad
        entry = attend.cmp_table[b, 0]
        if entry >= 0:
            attend.cmp.codes[entry, n // 128:] = bad
    attend.ori.codes[free], attend.ori.scale[free] = bad, np.nan
    attend.ori_table[0, 3] = free[0]                        # an entry behind the request's rows
    op = run(attend)
    compare(attend, op.out, op.lse, expected)
    # The second request's last row: codes that are no numbers (or a scale that is none) for its last token alone.
    last = attend.ori_table[1, 3]
    if kind == "e4m3":
        attend.ori.codes[last, 3] = 127
    else:
        attend.ori.scale[last] = np.nan                     # rows 96 .. 99: four tokens see one of them
    op = run(attend)
    out, lse = op.out.float().cpu().numpy(), op.lse.cpu().numpy()
    seeing = [40] if kind == "e4m3" else [37, 38, 39, 40]
    rest = [t for t in range(44) if t not in seeing]
    assert np.isnan(out[seeing]).all() and np.isnan(lse[seeing]).all()
    want, near, want_lse, lse_near = expected
    assert (np.abs(out[rest] - want[rest]) <= near[rest]).all() and (np.abs(lse[rest] - want_lse[rest]) <= lse_near[rest]).all()


@pytest.mark.parametrize("kind", KINDS)
def test_queries_that_are_no_numbers(kind):
    attend = Attend(11, [1, 20], [300, 200], kind=kind)
    attend.q[0, 3, 5], attend.q[7, 0, 511], attend.q[9, 1] = np.nan, np.inf, 0
    op = run(attend)
    out = op.out.float().cpu().numpy()
    assert np.isnan(out[0, 3]).all() and np.isnan(out[7, 0]).all()
    clean = attend.q.copy()
    clean[0, 3, 5] = clean[7, 0, 511] = 0
    attend.q = clean
    want, near, *_ = attend.expect()
    rest = np.ones(out.shape[:2], bool)
    rest[0, 3] = rest[7, 0] = False
    assert (np.abs(out - want) <= near)[rest].all()


@pytest.mark.parametrize("kind", KINDS)
def test_sinks_at_their_limits(kind):
    attend = Attend(12, [1, 9], [100, 2000], kind=kind)
    attend.sink[:] = [-math.inf, math.inf, 1e30, -1e30, 60, -60, 0, 5]
    finite = attend.sink.copy()
    op = run(attend)
    attend.sink = np.where(np.isinf(finite), np.sign(finite) * 1e30, finite).astype(np.float32)
    want, near, want_lse, lse_near = attend.expect()
    out, lse = op.out.float().cpu().numpy(), op.lse.cpu().numpy()
    assert (np.abs(out - want) <= near).all()
    assert np.isinf(lse[:, 1]).all() and (np.abs(lse - want_lse) <= lse_near)[:, [0, 2, 3, 4, 5, 6, 7]].all()


@pytest.mark.parametrize("kind", KINDS)
def test_many_requests(kind):
    rng = np.random.default_rng(1)
    new = [int(n) for n in rng.integers(0, 3, 300)]         # more requests than a work-group has threads
    check(Attend(13, new, [n + int(k) for n, k in zip(new, rng.integers(0, 90, 300))], kind=kind, heads=2))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new,heads,length", [(1, 8, 20000), (2, 16, 9000), (1, 64, 9000), (8, 8, 9000)])
def test_split_contexts_give_the_same_twice(kind, new, heads, length):
    import torch
    attend = Attend(14, [new], [length], kind=kind, heads=heads)
    op = check(attend)
    assert op.partial is not None
    first, first_lse = op.out.clone(), op.lse.clone()
    op.partial.fill_(math.nan)
    op.out.zero_()
    op.run()
    assert torch.equal(first, op.out) and torch.equal(first_lse, op.lse)


def test_tables_far_wider_than_the_rows():
    attend = Attend(15, [1, 2], [90, 300])
    wide = np.full((2, 5000), -1, np.int32)
    wide[:, :attend.ori_table.shape[1]] = attend.ori_table
    attend.ori_table = wide
    check(attend)


def test_pages_past_32_bits():
    """A pool of more than 4 GiB: pages at both its ends."""
    import torch
    from npu_sparse_attn_sharedkv_int8 import PreparedBlockAttention
    attend = Attend(16, [2], [120], kind="e4m3")
    expected = attend.expect()
    case, ori_scale, _ = attend.device()
    pages, stride = len(attend.ori.codes), 2 ** 20
    far = 5000
    pool = torch.empty(far * stride, dtype=torch.int8, device="cuda").view(torch.float8_e4m3fn)
    pool = pool.as_strided((far, BLOCK, 1, DIM), (stride, DIM, DIM, 1))
    scales = torch.full((far, 1), math.nan, device="cuda")
    moved = [0, 4999, 4097, 2500, 4500, 4096, 1][:pages]
    for page, to in enumerate(moved):
        pool[to].view(torch.int8).copy_(case.ori[page].view(torch.int8))
        scales[to] = ori_scale[page]
    table = case.ori_block_table
    case.ori_block_table = torch.where(table >= 0, torch.tensor(moved, dtype=torch.int32, device="cuda")[table.clamp(min=0).long()], -1)
    case.ori = pool
    op = PreparedBlockAttention(case, scales, return_lse=True)
    op.run()
    compare(attend, op.out, op.lse, expected)


def test_captured_replayed_with_other_lengths():
    import torch
    from npu_sparse_attn_sharedkv_int8 import PreparedBlockAttention
    attend = Attend(17, [1] * 6, [3000, 40, 700, 64, 65, 5000])
    case, ori_scale, _ = attend.device()
    op = PreparedBlockAttention(case, ori_scale, return_lse=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        op.run()
    for lengths in ([3000, 40, 700, 64, 65, 5000], [1, 40, 2, 64, 65, 30], [0, 0, 700, 0, 1, 4999], [3000, 40, 700, 64, 65, 5000]):
        attend.lengths = lengths
        case.seq_lens.copy_(torch.tensor(lengths, dtype=torch.int32))
        op.out.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        compare(attend, op.out, op.lse, attend.expect())


def test_two_operators_on_two_streams():
    import torch
    from npu_sparse_attn_sharedkv_int8 import PreparedBlockAttention
    first, second = Attend(18, [1, 1], [6000, 900]), Attend(19, [1, 2], [5000, 1900], kind="e4m3")
    ops = []
    for attend in (first, second):
        case, scale, _ = attend.device()
        ops.append(PreparedBlockAttention(case, scale, return_lse=True))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for op, stream in zip(ops, streams):
            with torch.cuda.stream(stream):
                op.run()
    torch.cuda.synchronize()
    for attend, op in zip((first, second), ops):
        compare(attend, op.out, op.lse, attend.expect())


def test_rebinding():
    import torch
    from npu_sparse_attn_sharedkv_int8 import PreparedBlockAttention
    attend, other = Attend(20, [2, 1], [300, 90]), Attend(20, [2, 1], [310, 80])
    other.q += 1
    case, scale, _ = attend.device()
    op = PreparedBlockAttention(case, scale, return_lse=True)
    op.run()
    out = torch.empty_like(op.out)
    lse = torch.empty_like(op.lse)
    theirs, scale, _ = other.device()
    op._rebind_same_geometry(theirs, scale, output=out, lse_output=lse)
    assert op.run() is out
    compare(other, out, lse, other.expect())
    theirs.window = 5
    with pytest.raises(ValueError):
        op._rebind_same_geometry(theirs)
