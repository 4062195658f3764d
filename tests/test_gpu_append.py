"""PreparedCacheAppend: every code, scale and untouched byte against the
definition in 64 bits (block_cases.append).  Codes and scales are whole numbers
and single roundings: nothing may differ."""
import sys
import zlib

import numpy as np
import pytest

from tests import block_cases as cases

pytestmark = pytest.mark.gpu
DIM, BLOCK = cases.DIM, cases.BLOCK


def say(*a):
    print(*a, file=sys.stderr, flush=True)


def angles(rows, rotary):
    angle = np.arange(rows)[:, None] / 10000.0 ** (np.arange(0, rotary, 2) / rotary)
    return np.concatenate([np.cos(angle), np.sin(angle)], 1).astype(np.float32)


class Appended:
    """One call's inputs on the host, run on the device and checked byte for byte."""

    def __init__(self, seed, new, lengths, *, kind="int8", heads=1, rotary=64, pairs=True, behind=0, pad_tokens=0, pad_batch=0,
                 size=1.0, channel=False, far=False, first=None):
        rng = self.rng = np.random.default_rng(seed)
        self.new, self.lengths, self.kind, self.heads, self.pairs = new, lengths, kind, heads, pairs
        self.cu = np.array([0] + list(np.cumsum(new)) + [sum(new)] * pad_batch, np.int32)
        self.lens = np.array(list(lengths) + [0] * pad_batch, np.int32)
        self.tokens = sum(new) + pad_tokens
        last = [max(0, -(-n // BLOCK)) for n in lengths]
        self.table, pages = cases.table_of(rng, first or [0] * len(new), last, pad_batch)
        self.pool = cases.Pool(rng, pages, heads, kind, behind=behind)
        self.pool.scale *= np.float32(0.25) * size          # most pages that have rows need a larger scale
        self.x = cases.bf16(rng.standard_normal((self.tokens, heads, DIM)) * size)
        self.rotation = angles(700 if far else max(1, max(lengths)), rotary) if rotary else None
        self.positions = None
        if far:
            self.positions = rng.integers(0, 700, self.tokens).astype(np.int64)
        self.inverse = (1 / (0.02 + 0.02 * rng.random(DIM))).astype(np.float32) if channel else None

    def operator(self, strided=False):
        import torch
        from npu_sparse_attn_sharedkv_int8 import PreparedCacheAppend
        self.cache, self.scale = self.pool.device()
        put = lambda x: None if x is None else torch.from_numpy(x).cuda()  # noqa: E731
        x = put(self.x).to(torch.bfloat16)
        if strided:                                         # a part of a projection's output, heads apart too
            wide = torch.full((self.tokens, self.heads + 1, DIM + 64), 9.0, dtype=torch.bfloat16, device="cuda")
            wide[:, 1:, 32:32 + DIM] = x
            x = wide[:, 1:, 32:32 + DIM]
        scales = dict(inverse_scale=put(self.inverse)) if self.inverse is not None else dict(scale=self.scale)
        return PreparedCacheAppend(self.cache, x, put(self.table), put(self.cu), put(self.lens), rotation=put(self.rotation),
                                   positions=put(self.positions), interleaved=self.pairs, **scales)

    def expect(self, skip=()):
        place = self.positions
        if place is None:
            place = np.zeros(self.tokens, np.int64)
            for b, (n, length) in enumerate(zip(self.new, self.lengths)):
                place[self.cu[b]:self.cu[b] + n] = np.arange(length - n, length).clip(min=0)
        if self.rotation is not None:
            place = place.clip(0, len(self.rotation) - 1)
        x = cases.rotated(self.x.astype(np.float64), self.rotation, place, self.pairs)
        codes, scale = self.pool.codes.copy(), self.pool.scale.copy()
        cases.append(codes, scale, self.kind, x, self.table, self.cu, self.lens, inverse=self.inverse, skip=skip)
        return codes, scale

    def one_sign(self, codes):
        """e4m3 has two codes for zero and two that are no number."""
        return np.where((codes & 127) % 127 == 0, codes & 127, codes) if self.kind == "e4m3" else codes

    def check(self, codes, scale):
        import torch
        torch.cuda.synchronize()
        got = np.ascontiguousarray(self.cache.cpu().view(torch.int8).numpy().view(np.uint8))
        got, codes = self.one_sign(got), self.one_sign(codes)
        assert np.array_equal(self.scale.cpu().numpy(), scale)
        wrong = np.argwhere(got != codes)
        assert not len(wrong), wrong[:5]
        if self.pool.behind:                                # the bytes between pages, but for scales in them
            pages, _, heads, _ = codes.shape
            rest = self.pool.backing.view(pages, -1)[:, BLOCK * heads * DIM:].cpu().numpy()
            rest = np.delete(rest, np.s_[8:8 + 4 * heads], 1) if self.pool.behind >= 4 * heads + 16 else rest
            assert (rest == 77).all()


def check(seed, *args, strided=False, **kw):
    case = Appended(seed, *args, **kw)
    op = case.operator(strided)
    assert op.run() is case.cache
    case.check(*case.expect())
    return case, op


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("new,lengths", [
    ([1], [1]), ([1], [32]), ([1], [33]), ([1], [70]), ([31], [31]), ([32], [64]), ([33], [33]), ([2], [33]), ([64], [95]),
    ([1, 1, 1, 1], [5, 32, 64, 97]), ([3, 200, 1, 40], [40, 200, 64, 41]), ([0, 5, 0, 1], [7, 5, 0, 33])], ids=str)
def test_lengths(kind, new, lengths):
    check(zlib.crc32(f"{kind}{new}{lengths}".encode()), new, lengths, kind=kind)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("rotary", [0, 16, 64, 128, 512])
@pytest.mark.parametrize("pairs", [True, False])
def test_rotations(kind, rotary, pairs):
    check(11 + rotary, [40, 1, 7], [90, 33, 7], kind=kind, rotary=rotary, pairs=pairs)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("heads", [1, 2, 3, 8])
def test_heads_strides_and_scales_between_pages(kind, heads):
    check(23 + heads, [5, 1, 34], [50, 32, 34], kind=kind, heads=heads, behind=64, strided=True, far=True)


@pytest.mark.parametrize("rotary,pairs", [(0, True), (64, True), (128, False)])
def test_frozen_channel_scales(rotary, pairs):
    check(5, [40, 1, 7], [90, 33, 7], rotary=rotary, pairs=pairs, channel=True, behind=32)


def test_frozen_codes_are_the_writers():
    import torch
    from npu_sparse_attn_sharedkv_int8 import PreparedCacheWrite
    case = Appended(6, [40, 1, 7], [90, 33, 7], rotary=0, channel=True)
    case.operator().run()
    mine = case.cache.clone()
    case.cache.copy_(torch.from_numpy(case.pool.codes.view(np.int8)))
    slots = [case.table[b, r // BLOCK] * BLOCK + r % BLOCK for b, (n, length) in enumerate(zip(case.new, case.lengths))
             for r in range(length - n, length)]
    PreparedCacheWrite(case.cache, torch.from_numpy(case.x).cuda().to(torch.bfloat16),
                       torch.tensor(slots, dtype=torch.int32, device="cuda"), torch.from_numpy(case.inverse).cuda()).run()
    assert torch.equal(mine, case.cache)


def test_many_requests():
    rng = np.random.default_rng(2)
    new = [int(n) for n in rng.integers(0, 4, 1500)]        # more requests than a work-group has threads
    check(8, new, [n + int(k) for n, k in zip(new, rng.integers(0, 100, 1500))], kind="e4m3")


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_padding_skipped_rows_and_pages(kind):
    case = Appended(9, [6, 3, 5, 4], [38, 3, 0, 2], kind=kind, pad_tokens=9, pad_batch=2, far=True)
    case.positions[[1, 4]] = [-1, 700]                      # outside the rotation
    case.table[1, 0] = len(case.pool.codes)                 # no page of the pool
    # Request 3 has fewer rows than tokens: its first two are below row 0.
    case.operator().run()
    case.check(*case.expect(skip={1, 4}))


def test_rows_past_the_table():
    case = Appended(10, [50], [90])
    case.table = np.ascontiguousarray(case.table[:, :2])
    case.operator().run()
    case.check(*case.expect())


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_values_that_are_no_numbers(kind):
    case = Appended(12, [20, 3, 1], [40, 3, 32], kind=kind, rotary=64)
    case.x[2, 0, [0, 500]] = np.nan
    case.x[5, 0, 9] = np.inf
    case.x[20, 0, 100] = -np.inf
    case.x[21] = 0
    case.x[23] = np.nan                                     # a row without a number
    case.x = cases.bf16(case.x)
    case.operator().run()
    case.check(*case.expect())


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("size", [0.0, 1e-30, 3e-9, 1e30])
def test_sizes_and_growth(kind, size):
    case, op = check(13, [4], [4], kind=kind, size=size or 1e-30)
    if not size:
        case.x[:] = 0
    # Rows one at a time behind them, larger and larger: the scale doubles, codes before are rounded again.
    import torch
    from npu_sparse_attn_sharedkv_int8 import PreparedCacheAppend
    codes, scale = case.expect()
    for length in range(5, 33):
        x = cases.bf16(case.rng.standard_normal((1, 1, DIM)) * max(size, 1e-9) * 1.3 ** (length - 4))
        lens, cu = np.array([length], np.int32), np.array([0, 1], np.int32)
        place = np.array([length % 4])
        PreparedCacheAppend(case.cache, torch.from_numpy(x).cuda().to(torch.bfloat16), torch.from_numpy(case.table).cuda(),
                            torch.from_numpy(cu).cuda(), torch.from_numpy(lens).cuda(), scale=case.scale,
                            rotation=torch.from_numpy(case.rotation).cuda(),
                            positions=torch.from_numpy(place).cuda()).run()
        turned = cases.rotated(x.astype(np.float64), case.rotation, place, True)
        cases.append(codes, scale, kind, turned, case.table, cu, lens)
    case.check(codes, scale)


def test_scale_of_a_page_that_has_none():
    case = Appended(14, [2, 2, 2, 2], [10, 11, 12, 13])
    case.pool.scale[case.table[:4, 0], 0] = [0, np.nan, np.inf, -1]
    case.operator().run()
    case.check(*case.expect())


def test_captured_and_replayed():
    import torch
    case = Appended(15, [1] * 40, [7 + 3 * i for i in range(40)], kind="e4m3", behind=32)
    op = case.operator()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        op.run()
    for _ in range(3):
        case.pool.device()[0]                               # other work between the replays
        case.cache.view(torch.int8).copy_(torch.from_numpy(case.pool.codes.view(np.int8)))
        case.scale.copy_(torch.from_numpy(case.pool.scale))
        graph.replay()
        torch.cuda.synchronize()
    codes, scale = case.expect()
    assert np.array_equal(case.scale.cpu().numpy(), scale)
    got = case.cache.cpu().view(torch.int8).numpy().view(np.uint8)
    assert (case.one_sign(got) == case.one_sign(codes)).all()


def test_on_another_stream():
    import torch
    case = Appended(16, [40, 1], [90, 33])
    op = case.operator()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        op.run()
    torch.cuda.current_stream().wait_stream(stream)
    case.check(*case.expect())
