"""The block-scaled cache as a serving loop uses it: prompts appended in chunks,
tokens one at a time, attention after each, eager and captured; forks and
compactions that move codes and scales together; and the refusals of the
constructors."""
import numpy as np
import pytest

from tests import block_cases as cases
from tests.block_cases import ALL, Attend, BLOCK, DIM
from tests.test_gpu_append import angles
from tests.test_gpu_block_attention import compare

pytestmark = pytest.mark.gpu
KINDS = ["int8", "e4m3"]


class Loop:
    """Requests over one pool of pages with their scales behind them.  `codes` and `scale` are the definition's."""

    def __init__(self, seed, kind, batch, heads=1, pages=40, width=6):
        import torch
        self.rng = np.random.default_rng(seed)
        self.kind, self.heads, self.lengths = kind, heads, [0] * batch
        order = self.rng.permutation(pages)[:batch * width]
        self.table = order.reshape(batch, width).astype(np.int32)
        self.pool = cases.Pool(self.rng, pages, heads, kind, behind=64)
        self.cache, self.scale = self.pool.device()
        self.codes, self.scales = self.pool.codes.copy(), self.pool.scale.copy()
        self.rotation = angles(width * BLOCK, 64)
        self.turn = torch.from_numpy(self.rotation).cuda()
        self.dev_table = torch.from_numpy(self.table).cuda()

    def rows(self, counts):
        """New rows [T, heads, 512] for the requests, and the launch's cu_q and lengths."""
        self.lengths = [n + t for n, t in zip(self.lengths, counts)]
        x = cases.bf16(self.rng.standard_normal((sum(counts), self.heads, DIM)) * np.exp(self.rng.uniform(-1, 1)))
        return x, np.array([0] + list(np.cumsum(counts)), np.int32), np.array(self.lengths, np.int32)

    def define(self, x, cu, lens, counts):
        place = np.concatenate([np.arange(n - t, n) for n, t in zip(lens, counts)])
        x = cases.rotated(x.astype(np.float64), self.rotation, place, True)
        cases.append(self.codes, self.scales, self.kind, x, self.table, cu, lens)

    def attend(self, counts, seed, window=ALL):
        """An Attend over the defined cache."""
        a = Attend(seed, counts, self.lengths, heads=8, kv_heads=self.heads, kind=self.kind, window=window)
        a.ori_table, a.ori.codes, a.ori.scale = self.table, self.codes, self.scales
        return a

    def check_cache(self):
        got = np.ascontiguousarray(self.cache.cpu().view(__import__("torch").int8).numpy().view(np.uint8))
        sign = lambda c: np.where((c & 127) % 127 == 0, c & 127, c) if self.kind == "e4m3" else c  # noqa: E731
        assert (sign(got) == sign(self.codes)).all()
        assert np.array_equal(self.scale.cpu().numpy(), self.scales)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads", [1, 2])
def test_prompts_in_chunks_then_tokens(kind, heads):
    import torch
    from npu_sparse_attn_sharedkv_int8 import PreparedBlockAttention, PreparedCacheAppend, SharedKVCase
    loop = Loop(1, kind, 3, heads)
    put = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda()  # noqa: E731
    for step, counts in enumerate(([40, 7, 32], [25, 1, 33], [1, 1, 1], [1, 0, 1], [1, 1, 1], [3, 1, 40], [1, 1, 1])):
        x, cu, lens = loop.rows(counts)
        cu_dev, lens_dev = put(cu), put(lens)
        PreparedCacheAppend(loop.cache, put(x).to(torch.bfloat16), loop.dev_table, cu_dev, lens_dev, scale=loop.scale,
                            rotation=loop.turn).run()
        a = loop.attend(counts, step, window=50 if step % 2 else ALL)
        loop.define(x, cu, lens, counts)
        case = SharedKVCase(put(a.q).to(torch.bfloat16), loop.cache, loop.dev_table, cu_dev, lens_dev, put(a.sink),
                            window=a.window, softmax_scale=a.softmax_scale)
        op = PreparedBlockAttention(case, loop.scale, return_lse=True)
        op.run()
        loop.check_cache()
        compare(a, op.out, op.lse, a.expect())


@pytest.mark.parametrize("kind", KINDS)
def test_a_captured_step_replayed(kind):
    """A decode step in one graph, replayed over other rows and lengths, with eager work between the replays."""
    import torch
    from npu_sparse_attn_sharedkv_int8 import PreparedBlockAttention, PreparedCacheAppend, SharedKVCase
    loop = Loop(2, kind, 4)
    put = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda()  # noqa: E731
    x, cu, lens = loop.rows([30, 64, 1, 90])
    PreparedCacheAppend(loop.cache, put(x).to(torch.bfloat16), loop.dev_table, put(cu), put(lens), scale=loop.scale,
                        rotation=loop.turn).run()
    loop.define(x, cu, lens, [30, 64, 1, 90])
    ones = [1] * 4
    rows = torch.zeros((4, 1, DIM), dtype=torch.bfloat16, device="cuda")
    q = torch.zeros((4, 8, DIM), dtype=torch.bfloat16, device="cuda")
    places = torch.zeros(4, dtype=torch.int64, device="cuda")
    lens_dev, cu_dev = put(lens), put(np.arange(5, dtype=np.int32))
    sink = torch.zeros(8, device="cuda")
    append = PreparedCacheAppend(loop.cache, rows, loop.dev_table, cu_dev, lens_dev, scale=loop.scale, rotation=loop.turn,
                                 positions=places)
    attend = PreparedBlockAttention(SharedKVCase(q, loop.cache, loop.dev_table, cu_dev, lens_dev, sink, window=ALL), loop.scale,
                                    return_lse=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        append.run()
        attend.run()
    for step in range(6):
        x, cu, lens = loop.rows(ones)
        a = loop.attend(ones, 50 + step)
        rows.copy_(put(x)), q.copy_(put(a.q)), lens_dev.copy_(put(lens)), sink.copy_(put(a.sink))
        places.copy_(put(lens).long() - 1)
        graph.replay()
        torch.cuda.synchronize()
        loop.define(x, cu, lens, ones)
        loop.check_cache()
        compare(a, attend.out, attend.lse, a.expect())
        torch.randn(1000, 1000, device="cuda").sum().item()


@pytest.mark.parametrize("kind", KINDS)
def test_forked_and_compacted_pages_keep_their_scales(kind):
    """Scales behind the codes in one backing move with the pages: two children of a request go on apart."""
    import torch
    from npu_sparse_attn_sharedkv_int8 import (PreparedBlockAttention, PreparedCacheAppend, PreparedPageCompact,
                                               PreparedPageFork, SharedKVCase)
    loop = Loop(3, kind, 1, pages=20)
    put = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda()  # noqa: E731
    x, cu, lens = loop.rows([75])
    PreparedCacheAppend(loop.cache, put(x).to(torch.bfloat16), loop.dev_table, put(cu), put(lens), scale=loop.scale,
                        rotation=loop.turn).run()
    loop.define(x, cu, lens, [75])
    backing = loop.pool.backing.view(20, -1)
    table = put(np.where(np.arange(6) < 3, loop.table, -1).astype(np.int32))
    refs = torch.zeros(20, dtype=torch.int32, device="cuda")
    refs[table[table >= 0].long()] = 1
    fork = PreparedPageFork([backing], table, put(lens), refs, put(np.zeros(2, np.int32)), room=1)
    table, lengths, refs = fork.run()
    # Each child appends a row of its own, far larger in the second.
    x = cases.bf16(loop.rng.standard_normal((2, 1, DIM)) * np.array([1, 50])[:, None, None])
    cu, lens = put(np.arange(3, dtype=np.int32)), lengths + 1
    append = PreparedCacheAppend(loop.cache, put(x).to(torch.bfloat16), table, cu, lens, scale=loop.scale, rotation=loop.turn)
    append.run()
    table, refs, _ = PreparedPageCompact([backing], table, refs).run()
    torch.cuda.synchronize()
    pages = table.cpu().numpy()
    # The definition: both children hold a copy of the parent's last page.
    parent = loop.table[0, :3]
    for child in range(2):
        codes, scales = loop.codes[parent].copy(), loop.scales[parent].copy()
        its = cases.rotated(x[child:child + 1].astype(np.float64), loop.rotation, np.array([75]), True)
        cases.append(codes, scales, kind, its, np.arange(3, dtype=np.int32)[None], [0, 1], [76])
        got = loop.cache.view(torch.int8).cpu().numpy().view(np.uint8)[pages[child, :3]]
        assert np.array_equal(loop.scale.cpu().numpy()[pages[child, :3]], scales)
        assert (np.where(got == 128, 0, got) == np.where(codes == 128, 0, codes))[:2].all()
        assert (np.where(got == 128, 0, got) == np.where(codes == 128, 0, codes))[2, :12].all()
    a = Attend(9, [1, 1], [76, 76], kind=kind)
    a.ori_table = pages
    a.ori.codes = loop.cache.view(torch.int8).cpu().numpy().view(np.uint8)
    a.ori.scale = loop.scale.cpu().numpy()
    op = PreparedBlockAttention(SharedKVCase(put(a.q).to(torch.bfloat16), loop.cache, table, cu, lens, put(a.sink), window=ALL),
                                loop.scale, return_lse=True)
    op.run()
    compare(a, op.out, op.lse, a.expect())


def test_attention_refuses():
    import torch
    from npu_sparse_attn_sharedkv_int8 import PreparedBlockAttention
    from dataclasses import replace
    attend = Attend(1, [2, 1], [100, 300], heads=8, kv_heads=2, ratio=128, window=128)
    case, ori, cmp = attend.device()
    PreparedBlockAttention(case, ori, cmp)
    wide = torch.zeros((3, 8, 2 * DIM), dtype=torch.bfloat16, device="cuda")
    for change in [dict(q=case.q.float()), dict(q=case.q[:, :7].contiguous()), dict(q=wide[..., :DIM]), dict(q=case.q[..., :256]),
                   dict(ratio=4), dict(ratio=64), dict(window=0), dict(window=2 ** 31), dict(cmp_indices=case.cu_q),
                   dict(ori_indices=case.cu_q), dict(ori=case.ori.view(torch.uint8)), dict(ori=case.ori.view(torch.float8_e4m3fn)),
                   dict(ori=case.ori[:, :, :1]), dict(cmp=None), dict(cmp_block_table=None), dict(cu_q=case.cu_q[:2]),
                   dict(cu_q=case.cu_q.long()), dict(seq_lens=case.seq_lens.cpu()), dict(sink=case.sink[:4]),
                   dict(sink=case.sink.double()), dict(ori_block_table=case.ori_block_table[:1]),
                   dict(ori_block_table=case.ori_block_table[:, :0]), dict(ori_block_table=case.ori_block_table.t().contiguous().t())]:
        with pytest.raises(ValueError):
            PreparedBlockAttention(replace(case, **change), ori, cmp)
    for scales in [(None, cmp), (ori, None), (ori[:, :1], cmp), (ori.double(), cmp), (ori.cpu(), cmp), (cmp, ori)]:
        with pytest.raises(ValueError):
            PreparedBlockAttention(case, *scales)
    for outputs in [dict(output=case.q), dict(output=torch.empty_like(case.q).float()), dict(output=torch.empty_like(case.q)[:2]),
                    dict(lse_output=torch.empty(3, 8, device="cuda").half()), dict(lse_output=torch.empty(8, 3, device="cuda").t())]:
        with pytest.raises(ValueError):
            PreparedBlockAttention(case, ori, cmp, **outputs)
    inside = case.ori.view(torch.int8)[0].view(-1)[:3 * 8 * DIM * 2].view(torch.bfloat16).view(3, 8, DIM)
    with pytest.raises(ValueError):
        PreparedBlockAttention(case, ori, cmp, output=inside)
    out = torch.empty_like(case.q)
    with pytest.raises(ValueError):
        PreparedBlockAttention(case, ori, cmp, output=out, lse_output=out.view(-1)[:48].view(torch.float32).view(3, 8))


def test_append_refuses():
    import torch
    from npu_sparse_attn_sharedkv_int8 import PreparedCacheAppend
    from tests.test_gpu_append import Appended
    made = Appended(1, [3, 5], [40, 5], heads=2, behind=64)
    op = made.operator()
    x, table, cu, lens, turn = op.inputs
    cache, scale = made.cache, made.scale
    good = dict(cache=cache, updates=x, block_table=table, cu_q=cu, seq_lens=lens, scale=scale, rotation=turn)
    PreparedCacheAppend(**good)
    spare = torch.zeros((8, 2, DIM + 4), dtype=torch.bfloat16, device="cuda")
    odd = torch.zeros((40, 66), device="cuda")
    one = torch.ones(DIM, device="cuda")
    for change in [dict(scale=None), dict(inverse_scale=one), dict(scale=None, inverse_scale=one), dict(cache=cache.view(torch.uint8)),
                   dict(cache=cache.cpu()), dict(cache=cache[:, :16]), dict(updates=x.float()), dict(updates=x[:, :1]),
                   dict(updates=x[..., :256]), dict(updates=spare[..., :DIM]), dict(updates=x.cpu()), dict(updates=x[:, 0]),
                   dict(block_table=table.long()), dict(block_table=table[:1]), dict(block_table=table[:, :0]), dict(cu_q=cu[:2]),
                   dict(seq_lens=lens.long()), dict(scale=scale[:2]), dict(scale=scale.cpu()), dict(scale=torch.ones(2, len(scale), device="cuda").t()),
                   dict(scale=cache.view(torch.float32)[:, 0, 0, :2]), dict(rotation=turn.half()), dict(rotation=turn[:, :20]),
                   dict(rotation=turn[:, :8]), dict(rotation=odd[:, :64]), dict(rotation=turn[:0]), dict(rotation=turn.cpu()),
                   dict(positions=cu), dict(positions=torch.zeros(8, device="cuda")), dict(rotation=None, positions=torch.zeros(8, dtype=torch.int32, device="cuda")),
                   dict(updates=cache.view(torch.bfloat16)[0, :8, :, :].expand(8, 2, 256)), dict(block_table=None), dict(seq_lens=None)]:
        with pytest.raises(ValueError):
            PreparedCacheAppend(**{**good, **change})
    empty = PreparedCacheAppend(**{**good, "updates": x[:0]})
    before = cache.clone()
    empty.run()
    assert torch.equal(before.view(torch.int8), cache.view(torch.int8))


def test_rebinding_an_append():
    import torch
    from tests.test_gpu_append import Appended
    first, second = Appended(2, [3], [40]), Appended(3, [1, 70], [2, 100], kind="e4m3", heads=2, behind=64)
    op = first.operator()
    op.run()
    first.check(*first.expect())
    other = second.operator()
    x, table, cu, lens, turn = other.inputs
    op._rebind(second.cache, x, table, cu, lens, scale=second.scale, rotation=turn)
    op.run()
    second.check(*second.expect())
    with pytest.raises(ValueError):
        op._rebind(second.cache, x, table, cu[:1], lens, scale=second.scale, rotation=turn)
