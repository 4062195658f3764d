"""Host side of the block-scaled caches' operators, without a device: what the C
entries and the constructors refuse, the scratch, and the tests' own codes."""
import ctypes

import numpy as np
import pytest
import torch

import npu_sparse_attn_sharedkv_int8 as package
from npu_sparse_attn_sharedkv_int8 import block_cache, runtime
from tests import block_cases as cases
from tests.test_launch_sizes_host import code
from tests.test_tree_pages_host import INVALID

SLOTS = 512


def good_append(frozen=False):
    """A block whose pointers are never followed: entries that reject it launch nothing."""
    a = runtime.CacheAppendArgs(pageStride=32 * 512, updateStride=512, updateHeadStride=512, scaleStride=1, rotationStride=64,
                                tokens=8, batch=2, heads=1, pages=4, tableWidth=4, rotary=64, rotationRows=100, interleaved=1)
    for name in "cache updates table cuQ seqLens positions rotation".split() + ["inverseScale" if frozen else "scale"]:
        setattr(a, name, 0x1000)
    return a


def good_attention():
    a = runtime.BlockAttentionArgs(oriStride=16384, cmpStride=16384, oriScaleStride=1, cmpScaleStride=1, tokens=8, heads=8,
                                   kvHeads=1, batch=1, oriPages=4, cmpPages=4, oriTableWidth=64, cmpTableWidth=4, ratio=128,
                                   window=2 ** 30, softmaxScale=0.04)
    for name in "q ori cmp oriScale cmpScale oriTable cmpTable cuQ seqLens sinks out partial units".split():
        setattr(a, name, 0x1000)
    return a


def scratch(a):
    sizes = ctypes.c_uint64(), ctypes.c_uint64()
    return runtime.library().sharedkv_block_scratch(ctypes.addressof(a), *map(ctypes.byref, sizes)), *(s.value for s in sizes)


def test_exports():
    for name in ("PreparedCacheAppend", "PreparedBlockAttention"):
        assert name in package.__all__ and getattr(package, name).__name__ == name


@pytest.mark.parametrize("fields", [
    *[{name: 0} for name in "cache updates table cuQ seqLens scale rotation batch heads pages tableWidth rotationRows".split()],
    dict(inverseScale=0x1000), dict(heads=129), dict(codes=2), dict(interleaved=2), dict(int64Positions=2), dict(cache=0x1004),
    dict(updates=0x1008), dict(updateStride=516), dict(updateHeadStride=4), dict(pageStride=16380), dict(pageStride=16384 - 8),
    dict(heads=2, pageStride=16384), dict(scale=0x1002), dict(rotation=0x1008), dict(rotary=8), dict(rotary=528, rotationStride=528),
    dict(rotationStride=60), dict(rotationStride=66), dict(tokens=2 ** 31), dict(batch=2 ** 24), dict(tableWidth=2 ** 26),
    dict(tokens=2 ** 28), dict(tokens=2 ** 24, heads=128, pageStride=2 ** 21), dict(batch=2 ** 22)], ids=str)
def test_append_entry_rejects(fields):
    assert code("launch_sharedkv_append", good_append(), **fields) == INVALID


@pytest.mark.parametrize("fields", [dict(codes=1), dict(heads=2, pageStride=32768), dict(inverseScale=0x1004)], ids=str)
def test_append_entry_rejects_frozen_scales_of(fields):
    assert code("launch_sharedkv_append", good_append(True), **fields) == INVALID


def test_appends_of_nothing_launch_nothing():
    assert code("launch_sharedkv_append", good_append(), tokens=0) == 0
    assert runtime.library().launch_sharedkv_append(None, None) == INVALID


@pytest.mark.parametrize("fields", [
    *[{name: 0} for name in "q ori cmp oriScale cmpScale oriTable cmpTable cuQ seqLens sinks out heads kvHeads batch window ratio "
      "oriPages cmpPages oriTableWidth cmpTableWidth".split()],
    dict(heads=129), dict(heads=8, kvHeads=3), dict(codes=2), dict(ratio=3), dict(ratio=127), dict(q=0x1008), dict(out=0x1004),
    dict(ori=0x1001), dict(cmp=0x1008), dict(oriScale=0x1002), dict(cmpScale=0x1001), dict(oriStride=16000), dict(oriStride=16392),
    dict(cmpStride=16376), dict(kvHeads=2), dict(tokens=1 << 31), dict(batch=1 << 25), dict(oriTableWidth=1 << 27),
    dict(cmpTableWidth=1 << 27)], ids=str)
def test_attention_entry_rejects(fields):
    a = good_attention()
    assert code("launch_sharedkv_block", a, **fields) == INVALID and scratch(a)[0] == INVALID


def test_attention_entry_needs_its_scratch():
    ok, partial, units = scratch(good_attention())
    assert ok == 0 and partial and units
    for name in ("partial", "units"):
        for value in (0, 0x1008):
            assert code("launch_sharedkv_block", good_attention(), **{name: value}) == INVALID
    assert code("launch_sharedkv_block", good_attention(), tokens=0) == 0
    assert runtime.library().launch_sharedkv_block(None, None) == INVALID
    assert runtime.library().sharedkv_block_scratch(ctypes.addressof(good_attention()), None, None) == INVALID


@pytest.mark.parametrize("tokens,heads,kv_heads,batch,width", [
    (1, 1, 1, 1, 64), (8, 8, 1, 4, 256), (320, 8, 1, 32, 16), (4000, 8, 1, 2, 512), (32, 64, 1, 32, 512), (72, 32, 4, 24, 250),
    (256, 8, 8, 256, 100), (9000, 64, 1, 300, 4), (3, 128, 1, 1, 20480)])
def test_scratch_covers_the_plan(tokens, heads, kv_heads, batch, width):
    """Room for SLOTS states at most, of one of the three sizes, and an entry of 32 bytes for every unit that the
    requests can have."""
    a = good_attention()
    a.tokens, a.heads, a.kvHeads, a.batch, a.oriTableWidth, a.ratio = tokens, heads, kv_heads, batch, width, 1
    a.oriStride = 16384 * kv_heads
    ok, partial, units = scratch(a)
    assert ok == 0
    if not partial:
        assert not units
        return
    group = heads // kv_heads
    fits = []
    for rows in (16, 32, 64):
        # The most units of any division of the tokens: all in few requests, or one each.
        even = [tokens // batch + (i < tokens % batch) for i in range(batch)]
        most = [tokens - min(tokens, batch) + 1] + [1] * (min(tokens, batch) - 1)
        needed = max(sum(kv_heads * -(-n * group // rows) for n in division) for division in (even, most))
        fits += [partial % (rows * 514 * 4) == 0 and partial // (rows * 514 * 4) <= SLOTS and units // 32 - 1 >= needed]
    assert any(fits)


def test_contexts_past_the_plans_sums_are_not_split():
    a = good_attention()
    a.tokens, a.heads, a.ratio = 90, 128, 1
    for width, split in ((100_000, True), (1_000_000, False)):
        a.oriTableWidth = width
        ok, partial, _ = scratch(a)
        assert ok == 0 and (partial > 0) == split


def test_divisions_of_the_plan():
    """The kernel's quotients by a group of heads, n * inverse >> bits with the entry's inverse, are exact."""
    rng = np.random.default_rng(0)
    for group in range(1, 129):
        bits = (group - 1).bit_length()
        inverse = ((2 ** 31 << bits) + group - 1) // group
        assert inverse < 2 ** 32
        for n in [0, 1, group - 1, group, 2 ** 31 - 1] + [int(v) for v in rng.integers(0, 2 ** 31, 200)] \
                + [int(v) * group + d for v in rng.integers(1, 2 ** 31 // group, 50) for d in (-1, 0) if v * group < 2 ** 31]:
            assert n * inverse >> 31 + bits == n // group


def test_work_groups_of_a_request_hold_its_pages():
    """An append's request takes cu[b + 1] // 32 + 2 (b + 1) - (cu[b] // 32 + 2 b) work-groups, wherever its rows begin."""
    for first in range(32):
        for rows in range(1, 200):
            groups = (first + rows) // 32 - first // 32 + 2
            assert all((begin + rows - 1) // 32 - begin // 32 + 1 <= groups for begin in range(32))


def test_host_tensors_are_refused():
    cache, table = torch.zeros((3, 32, 1, 512), dtype=torch.int8), torch.zeros((2, 3), dtype=torch.int32)
    ints, cu, scale = torch.zeros(2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), torch.ones(3, 1)
    with pytest.raises(ValueError, match="on a GPU"):
        package.PreparedCacheAppend(cache, torch.zeros((4, 512), dtype=torch.bfloat16), table, cu, ints, scale=scale)
    case = package.SharedKVCase(torch.zeros((2, 8, 512), dtype=torch.bfloat16), cache, table, cu, ints, torch.zeros(8))
    with pytest.raises(ValueError, match="on a GPU"):
        package.PreparedBlockAttention(case, scale)


def test_cache_checks():
    """The shared checks of a cache and its scales, on host tensors."""
    device = torch.device("cpu")

    def check(cache, scale, unit=16):
        block_cache._check_block_cache(cache, scale, device, unit)

    backing = torch.zeros(5 * 17408, dtype=torch.int8)
    cache = backing.as_strided((5, 32, 1, 512), (17408, 512, 512, 1))
    behind = backing.view(torch.float32).as_strided((5, 1), (17408 // 4, 1), 4096)
    check(cache, torch.ones(5, 1))
    check(cache, behind)
    check(cache.view(torch.float8_e4m3fn), behind)
    check(torch.zeros((5, 32, 4, 512), dtype=torch.int8), torch.ones(5, 8)[:, 2:6])
    check(cache[:1], torch.ones(1, 1))
    for bad, scale in [
            (cache.view(torch.uint8), torch.ones(5, 1)), (cache[:, :16], torch.ones(5, 1)), (cache[..., :256], torch.ones(5, 1)),
            (cache, torch.ones(5)), (cache, torch.ones(4, 1)), (cache, torch.ones(5, 2)), (cache, torch.ones(5, 1).double()),
            (cache[:0], torch.ones(0, 1)), (cache, behind.as_strided((5, 1), (17408 // 4, 1), 100)),
            (torch.zeros((5, 32, 2, 512), dtype=torch.int8), torch.ones(2, 5).t()),
            (backing.as_strided((5, 32, 1, 512), (16392, 512, 512, 1)), torch.ones(5, 1)),
            (backing.as_strided((5, 32, 1, 512), (8192, 512, 512, 1)), torch.ones(5, 1)),
            (torch.zeros((5, 32, 2, 1024), dtype=torch.int8)[..., :512], torch.ones(5, 2)),
            (torch.zeros((5, 32, 129, 512), dtype=torch.int8), torch.ones(5, 129))]:
        with pytest.raises(ValueError):
            check(bad, scale)


def test_codes_of_the_tests():
    """The tests' e4m3 codes are torch's, and their roundings."""
    codes = torch.arange(256, dtype=torch.uint8)
    values = codes.view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(values, cases.E4M3, equal_nan=True)
    x = np.random.default_rng(0).standard_normal(20000) * np.exp(np.random.default_rng(1).uniform(-9, 5, 20000))
    x = np.concatenate([x.clip(-448, 448), values[~np.isnan(values)], (values[:126] + values[1:127]) / 2])
    wanted = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(cases.encode(x, "e4m3"), wanted)
    assert np.array_equal(cases.decode(cases.encode(np.arange(-127, 128.0), "int8"), "int8"), np.arange(-127, 128))
