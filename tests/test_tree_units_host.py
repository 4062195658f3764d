"""Query rows of a tree launch's units, read off the size of its scratch, without a device.  Few rows take small units
however wide their block tables are (a captured launch's tables are as wide as its longest context): one request of 64 rows
over 65536 keys runs 97 us in units of 16 rows, 220 in units of 32 and 906 in units of 64."""
import ctypes

import pytest

from npu_sparse_attn_sharedkv_int8 import runtime
from tests.test_tree_pages_host import good_tree

WHOLE = 2 ** 30


def rows_of_a_unit(tokens, heads, batch, keys, ratio, window):
    """16, 32 or 64; None where the launch is not split (and needs no scratch)."""
    a = good_tree()
    a.tokens, a.heads, a.batch, a.window, a.ratio = tokens, heads, batch, window, ratio
    a.oriTableWidth, a.cmpTableWidth = keys // 32, max(1, keys // ratio // 32) if ratio > 1 else 0
    sizes = ctypes.c_uint64(), ctypes.c_uint64()
    assert runtime.library().sharedkv_tree_scratch(ctypes.addressof(a), *map(ctypes.byref, sizes)) == 0
    fits = [rows for rows in (16, 32, 64) if sizes[0].value == 4 * (tokens * heads // rows + batch + 1)]
    return fits[0] if sizes[0].value else None


@pytest.mark.parametrize("keys", [4096, 65536, 262144, 2 ** 20])
@pytest.mark.parametrize("tokens,heads", [(1, 8), (4, 8), (8, 8)])
def test_a_lone_request_takes_units_of_16_rows(tokens, heads, keys):
    assert rows_of_a_unit(tokens, heads, 1, keys, 1, WHOLE) == 16


@pytest.mark.parametrize("tokens,heads,batch,keys,ratio,window,rows", [
    (320, 8, 32, 65536, 128, 128, 16), (320, 8, 32, 2 ** 20, 128, 128, 32),       # 19 and 26 us, 39 in units of 64
    (32, 8, 1, 262144, 1, WHOLE, 32), (32, 64, 1, 16384, 1, WHOLE, 32),           # 226 and 112 us
    (32, 64, 1, 65536, 1, WHOLE, 64), (240, 16, 4, 32768, 1, WHOLE, 64)])         # 296 and 243 us
def test_more_rows_and_keys_take_larger_ones(tokens, heads, batch, keys, ratio, window, rows):
    assert rows_of_a_unit(tokens, heads, batch, keys, ratio, window) == rows
