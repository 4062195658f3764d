"""Host side of the tree and page operators, without a device: argument blocks,
what the C entries reject, the bridge's checks, exports, refusals of host
tensors, and the wait state of the LDS DMA."""
import ctypes
import re
from pathlib import Path

import pytest
import torch

import npu_sparse_attn_sharedkv_int8 as package
from npu_sparse_attn_sharedkv_int8 import runtime

CSRC = Path(__file__).resolve().parents[1] / "ascend-int8-attention_amd" / "csrc"
INVALID = 1


def test_exports_and_argument_blocks():
    lib = runtime.library()
    for name in ("PreparedTreeAttention", "PreparedPathCommit", "PreparedPageFork", "PreparedPageCompact"):
        assert name in package.__all__ and getattr(package, name).__name__ == name
    for launch, block, size in runtime.BLOCK_LAUNCHES.values():
        assert hasattr(lib, launch) and getattr(lib, size)() == ctypes.sizeof(block)


def good_tree():
    """A block whose pointers are never followed: entries that reject it launch nothing."""
    a = runtime.TreeAttentionArgs(tokens=8, heads=8, batch=1, oriPages=4, cmpPages=4, oriTableWidth=4, cmpTableWidth=2,
                                  ratio=128, window=128, oriStride=16384, cmpStride=16384, softmaxScale=0.04)
    for name in "q ori cmp oriScale cmpScale oriTable cmpTable cuQ seqLens sinks parents out workspace partial".split():
        setattr(a, name, 0x1000)
    return a


@pytest.mark.parametrize("field,value", [
    ("q", 0), ("ori", 0), ("cmp", 0), ("oriScale", 0), ("cmpScale", 0), ("oriTable", 0), ("cmpTable", 0), ("cuQ", 0),
    ("seqLens", 0), ("sinks", 0), ("parents", 0), ("out", 0), ("heads", 0), ("heads", 129), ("batch", 0), ("window", 0),
    ("ratio", 0), ("oriPages", 0), ("cmpPages", 0), ("oriTableWidth", 0), ("cmpTableWidth", 0), ("oriStride", 16000),
    ("oriStride", 16392), ("cmpStride", 16400 - 24), ("q", 0x1008), ("out", 0x1004), ("ori", 0x1001),
    ("tokens", 1 << 31), ("batch", 1 << 25), ("oriTableWidth", 1 << 27)])
def test_tree_entry_rejects(field, value):
    lib, a = runtime.library(), good_tree()
    setattr(a, field, value)
    assert lib.launch_sharedkv_tree(None, ctypes.addressof(a)) == INVALID
    sizes = ctypes.c_uint64(), ctypes.c_uint64()
    assert lib.sharedkv_tree_scratch(ctypes.addressof(a), *map(ctypes.byref, sizes)) == INVALID


def test_tree_entry_needs_its_scratch():
    lib, a = runtime.library(), good_tree()
    sizes = ctypes.c_uint64(), ctypes.c_uint64()
    assert lib.sharedkv_tree_scratch(ctypes.addressof(a), *map(ctypes.byref, sizes)) == 0
    assert sizes[0].value >= 4 and sizes[1].value > 0
    for name in ("workspace", "partial"):
        b = good_tree()
        setattr(b, name, 0)
        assert lib.launch_sharedkv_tree(None, ctypes.addressof(b)) == INVALID
    assert lib.launch_sharedkv_tree(None, None) == INVALID
    assert lib.sharedkv_tree_scratch(ctypes.addressof(a), None, None) == INVALID
    a.tokens = 0
    assert lib.launch_sharedkv_tree(None, ctypes.addressof(a)) == 0


def test_tree_scratch_covers_the_plan():
    """The states' room follows the units: none where units are not split, at most 768 states of 16 rows or 512 of 32 or
    64 otherwise, and a ticket for every unit."""
    lib = runtime.library()
    for tokens, heads, batch, width in ((1, 1, 1, 2), (8, 8, 1, 4), (320, 8, 32, 16), (244, 16, 4, 1024), (384, 64, 16, 32),
                                        (9000, 64, 300, 4), (3, 128, 1, 2048)):
        a = good_tree()
        a.tokens, a.heads, a.batch, a.oriTableWidth = tokens, heads, batch, width
        sizes = ctypes.c_uint64(), ctypes.c_uint64()
        assert lib.sharedkv_tree_scratch(ctypes.addressof(a), *map(ctypes.byref, sizes)) == 0
        if not sizes[1].value:
            assert not sizes[0].value
            continue
        fits = [rows for rows, items in ((16, 768), (32, 512), (64, 512))
                if sizes[0].value == 4 * (tokens * heads // rows + batch + 1)
                and sizes[1].value % (rows * 514 * 4) == 0 and sizes[1].value // (rows * 514 * 4) <= items]
        assert fits, (tokens, heads, batch, width, sizes[0].value, sizes[1].value)


def test_contexts_past_the_plans_sums_are_not_split():
    """90 tokens of 128 heads over 12.8 M rows have 36 M tiles, more than the work-groups' sums hold."""
    lib, a = runtime.library(), good_tree()
    a.tokens, a.heads, a.ratio, a.window = 90, 128, 1, 2 ** 30
    sizes = ctypes.c_uint64(), ctypes.c_uint64()
    for width, split in ((100_000, True), (400_000, False)):
        a.oriTableWidth = width
        assert lib.sharedkv_tree_scratch(ctypes.addressof(a), *map(ctypes.byref, sizes)) == 0
        assert (sizes[1].value > 0) == split


def test_caches_of_a_pool_are_told_apart():
    from npu_sparse_attn_sharedkv_int8.pages import _all_apart

    def _apart(a, b, dims):
        return _all_apart([a, b], dims)

    flat = torch.zeros(22 * 4096, dtype=torch.int8)
    layers = [flat.as_strided((20, 4, 512), (4096, 512, 1), k * 2048) for k in range(2)]
    halves = [flat.as_strided((20, 8, 256), (4096, 512, 1), k * 256) for k in range(2)]
    odd = [flat.as_strided((19, 8, 256), (4096 - 256, 512, 1), k * 256) for k in range(2)]
    for dims in (1, 2):
        assert _apart(*layers, dims) and _apart(*layers[::-1], dims)
        assert not _apart(layers[0], layers[0], dims)
        assert not _apart(layers[0], flat.as_strided((20, 4, 512), (4096, 512, 1), 1536), dims)
        assert not _apart(layers[0], flat.as_strided((20, 4, 512), (4096, 512, 1), 4096 + 512), dims)
        assert _apart(layers[0], torch.zeros(20, 4, 512, dtype=torch.int8), dims)
        assert _apart(flat[:8192].view(2, 4096), flat[8192:].view(20, 4096), 1)
    assert _apart(*halves, 2) and _apart(*halves[::-1], 2)
    own = torch.zeros(20, 4, 512, dtype=torch.int8)
    assert _all_apart([*layers, own], 2) and not _all_apart([*layers, own, layers[1]], 2)
    many = [flat.as_strided((20, 4, 64), (4096, 64, 1), k * 256) for k in range(16)]
    assert _all_apart(many[::-1], 1) and not _all_apart(many + [flat.as_strided((20, 4, 64), (4096, 64, 1), 128)], 2)
    # Rows that lie side by side in a page, but not from page to page.
    assert not _apart(*odd, 2) and not _apart(*odd[::-1], 2)


def good_commit():
    a = runtime.PathCommitArgs(cacheCount=2, batch=3, depth=4, tokens=30, tableWidth=4, pages=9, pageRows=32, rowBytes=512)
    for name in "caches table cuQ seqLens paths pathLens lengths".split():
        setattr(a, name, 0x1000)
    return a


def good_fork():
    a = runtime.PageForkArgs(cacheCount=1, rows=3, children=4, width=5, pages=9, pageRows=32, room=3, pageBytes=16384)
    for name in "caches table seqLens refs parents newTable newLens newRefs missing workspace".split():
        setattr(a, name, 0x1000)
    return a


def good_compact():
    a = runtime.PageCompactArgs(cacheCount=1, rows=3, width=5, pages=9, pageBytes=16384)
    for name in "caches table refs newTable newRefs moved live workspace".split():
        setattr(a, name, 0x1000)
    return a


@pytest.mark.parametrize("make,launch,cases", [
    (good_commit, "launch_sharedkv_path_commit",
     [(n, 0) for n in "caches table cuQ seqLens paths pathLens lengths cacheCount depth tableWidth pages pageRows rowBytes"
      .split()] + [("rowBytes", 500), ("pages", 1 << 31), ("depth", 1 << 30), ("rowBytes", 0x80000000)]),
    (good_fork, "launch_sharedkv_page_fork",
     [(n, 0) for n in "caches table seqLens refs parents newTable newLens newRefs missing workspace cacheCount rows "
      "children width pages pageRows pageBytes".split()]
     + [("pages", (1 << 22) + 1), ("room", 1 << 30), ("rows", 1 << 20), ("children", 1 << 20), ("width", 1 << 24),
        ("pageBytes", 1 << 46)]),
    (good_compact, "launch_sharedkv_page_compact",
     [(n, 0) for n in "caches table refs newTable newRefs moved live workspace cacheCount pages pageBytes".split()]
     + [("pages", (1 << 22) + 1), ("pageBytes", 1 << 40)])])
def test_page_entries_reject(make, launch, cases):
    lib = runtime.library()
    assert getattr(lib, launch)(None, None) == INVALID
    for field, value in cases:
        a = make()
        setattr(a, field, value)
        assert getattr(lib, launch)(None, ctypes.addressof(a)) == INVALID, (field, value)


def test_workspace_sizes():
    lib = runtime.library()
    for children, width, pages in ((1, 1, 1), (277, 252, 34000), (64, 33, 2049)):
        chunks = -(-pages // 2048)
        assert lib.sharedkv_page_fork_workspace(children, width, pages) == 4 * (
            pages + children * (width + 4) + chunks * 2049)
        assert lib.sharedkv_page_compact_workspace(pages) == 4 * (chunks + 1 + 4 * pages)


def test_bridge_checks():
    bridge = runtime.bridge()
    for name in runtime.BLOCK_LAUNCHES:
        call = getattr(bridge, name)
        with pytest.raises(TypeError):
            call(0x1000)
        with pytest.raises(ValueError):
            call(0, 0)
        with pytest.raises(OverflowError):
            call(-1, 0)
    a = good_tree()
    a.heads = 0
    with pytest.raises(RuntimeError, match="hipError_t 1"):
        bridge.tree_attention(ctypes.addressof(a), 0)


def test_host_tensors_are_refused():
    cache, table = torch.zeros((3, 32, 1, 512), dtype=torch.int8), torch.zeros((2, 3), dtype=torch.int32)
    ints = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU caches"):
        package.PreparedPathCommit(cache, table, torch.zeros(3, dtype=torch.int32), ints, table, ints)
    with pytest.raises(ValueError, match="GPU caches"):
        package.PreparedPageFork(cache, table, ints, torch.zeros(3, dtype=torch.int32), ints)
    with pytest.raises(ValueError, match="GPU caches"):
        package.PreparedPageCompact([cache], table, torch.zeros(3, dtype=torch.int32))
    case = package.SharedKVCase(torch.zeros((2, 8, 512), dtype=torch.bfloat16), cache, table, torch.zeros(3, dtype=torch.int32),
                                ints, torch.zeros(8))
    with pytest.raises(ValueError, match="on a GPU"):
        package.PreparedTreeAttention(case, ints, torch.ones(512))


def test_lds_dma_header_waits_after_its_m0_write():
    """As for the kernels' own inline assembly: a wait state between the scalar write of M0 and the LDS DMA."""
    blocks = re.findall(r'asm volatile\(\s*"([^"]*_load_lds_[^"]*)"', (CSRC / "lds_dma.h").read_text())
    assert len(blocks) == 1
    steps = [step.split()[0] for step in blocks[0].split(r"\n\t")]
    assert steps[0] == "s_mov_b32" and steps[1] == "s_nop" and len(steps) == 3
