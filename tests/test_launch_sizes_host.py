"""Calls whose launches would have more threads than 32 bits count: refused by
the C entries before anything is launched, without a device.  (A call that is
not refused fails here for want of one, with another code.)"""
import ctypes

import pytest

from npu_sparse_attn_sharedkv_int8 import runtime
from tests.test_tree_pages_host import INVALID, good_commit, good_compact, good_fork, good_tree

GROUPS = (2 ** 32 - 1) // 256
KIB64 = 65536


def code(launch, block, **fields):
    for name, value in fields.items():
        setattr(block, name, value)
    return getattr(runtime.library(), launch)(None, ctypes.addressof(block))


@pytest.mark.parametrize("children,slices", [(2 ** 20 - 1, 17), (2 ** 14, 2 ** 10), (GROUPS, 1), (1, GROUPS)])
def test_forks(children, slices):
    assert code("launch_sharedkv_page_fork", good_fork(), children=children, pageBytes=slices * KIB64) == INVALID


def test_commits():
    assert code("launch_sharedkv_path_commit", good_commit(), batch=GROUPS + 1) == INVALID
    assert code("launch_sharedkv_path_commit", good_commit(), batch=2 ** 32 - 1) == INVALID


def test_compactions():
    """Tables of 2^32 - 1 entries and somewhat fewer, of pools that one launch takes with an entry a thread."""
    for rows, width in ((2 ** 16 - 1, 2 ** 16 + 1), (1, 256 * GROUPS - 1)):
        for pages in (9, 2048):
            assert code("launch_sharedkv_page_compact", good_compact(), pages=pages, rows=rows, width=width,
                        newTable=0x2000, newRefs=0x2000) == INVALID
    assert code("launch_sharedkv_page_compact", good_compact(), pages=2 ** 20, rows=2 ** 16, width=2 ** 16) == INVALID


def test_trees():
    sizes = ctypes.c_uint64(), ctypes.c_uint64()
    for fields in (dict(batch=GROUPS), dict(batch=GROUPS - 8, tokens=2 ** 14, heads=8),
                   dict(tokens=2 ** 24 - 2 ** 16, heads=127), dict(tokens=2 ** 23, heads=128, batch=64)):
        a = good_tree()
        assert code("launch_sharedkv_tree", a, **fields) == INVALID, fields
        assert runtime.library().sharedkv_tree_scratch(ctypes.addressof(a), *map(ctypes.byref, sizes)) == INVALID
    # The largest that is taken is: 2^30 query rows but for a few units.
    a = good_tree()
    a.tokens, a.heads = 2 ** 23 - 2 ** 10, 128
    assert runtime.library().sharedkv_tree_scratch(ctypes.addressof(a), *map(ctypes.byref, sizes)) == 0


@pytest.mark.parametrize("field", ["oriTableWidth", "cmpTableWidth"])
def test_tables_whose_rows_and_a_tile_pass_32_bits(field):
    """Tiles of a context are its rows, rounded up to 64, in signed 32 bits."""
    sizes = ctypes.c_uint64(), ctypes.c_uint64()
    limit = (2 ** 31 - 1 - 64) // 32
    for width, expected in ((limit, 0), (limit + 1, INVALID), (2 ** 26 - 1, INVALID)):
        a = good_tree()
        setattr(a, field, width)
        assert runtime.library().sharedkv_tree_scratch(ctypes.addressof(a), *map(ctypes.byref, sizes)) == expected


def test_ordinary_calls_are_not_refused():
    for launch, block in (("launch_sharedkv_page_fork", good_fork()), ("launch_sharedkv_path_commit", good_commit()),
                          ("launch_sharedkv_page_compact", good_compact())):
        import torch
        if not torch.cuda.is_available():                      # with a device this would follow the block's pointers
            assert code(launch, block) not in (0, INVALID)
