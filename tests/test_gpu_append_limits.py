"""PreparedCacheAppend where FP32 ends: values that vanish beside a page's scale,
infinities in rotated channels; and rows that are skipped.  Byte for byte against
the definition in 64 bits, as test_gpu_append.py."""
import numpy as np
import pytest

from tests import block_cases as cases
from tests.test_gpu_append import Appended, BLOCK, DIM

pytestmark = pytest.mark.gpu
KINDS = ["int8", "e4m3"]


def one_row(case, x, length):
    """Appends the row x [1, 1, 512] behind the first request's, on the device and in the definition; what both then hold."""
    import torch
    from npu_sparse_attn_sharedkv_int8 import PreparedCacheAppend
    codes, scale = case.expect()
    put = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    cu, lens = np.array([0, 1], np.int32), np.array([length], np.int32)
    PreparedCacheAppend(case.cache, put(x).to(torch.bfloat16), put(case.table[:1]), put(cu), put(lens), scale=case.scale,
                        rotation=put(case.rotation)).run()
    turned = cases.rotated(x.astype(np.float64), case.rotation, np.array([length - 1]), case.pairs)
    cases.append(codes, scale, case.kind, turned, case.table[:1], cu, lens)
    return codes, scale


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("peak,tiny", [(1e10, 1e-38), (1e8, 1e-40), (1e30, 1e-12), (3e38, 1.0), (1.0, 1e-39)])
@pytest.mark.parametrize("rotary", [0, 64])
def test_values_that_vanish_beside_the_largest(kind, peak, tiny, rotary):
    case = Appended(40, [20, 3], [50, 3], kind=kind, rotary=rotary)
    case.x *= tiny                                          # both signs, down to denormal ones
    case.x[:, 0, 7] = -tiny
    case.x[::2, 0, 100] = peak                              # 7 channels of a lane's eight beside it
    case.x[3, 0, 470] = -peak
    case.x = cases.bf16(case.x)
    case.operator().run()
    case.check(*case.expect())


@pytest.mark.parametrize("kind", KINDS)
def test_small_rows_on_a_page_that_had_an_infinity(kind):
    case = Appended(41, [3, 2], [3, 60], kind=kind)        # the second for its rotation's length
    case.x[1, 0, 5] = np.inf
    case.operator().run()
    case.check(*case.expect())
    x = cases.bf16(case.rng.standard_normal((1, 1, DIM)) * 1e-10)
    case.check(*one_row(case, x, 4))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("lengths", [[70, 12], [40, 9]], ids=str)
def test_rows_of_zeros(kind, lengths):
    """Fresh pages get the smallest scale, pages that have rows keep theirs."""
    case = Appended(42, [40, 3], lengths, kind=kind)
    case.x[:] = 0
    case.x[1::2] = -0.0
    case.operator().run()
    case.check(*case.expect())


def angled(case, size):
    """The case with its rotation `size` times as long (position 0 too turns by some angle)."""
    angle = np.arange(len(case.rotation))[:, None] * 0.7 + 0.3 + np.arange(case.rotation.shape[1] // 2)
    case.rotation = (np.concatenate([np.cos(angle), np.sin(angle)], 1) * size).astype(np.float32)
    return case


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("pairs", [True, False])
@pytest.mark.parametrize("channels", [[448], [449], [511], [480, 481], [479, 450], [460, 12]], ids=str)
def test_infinities_in_rotated_channels(kind, pairs, channels):
    case = angled(Appended(43, [40, 3, 1], [70, 9, 33], kind=kind, pairs=pairs), 1.0)
    for i, channel in enumerate(channels):
        case.x[7 + 30 * (i % 2), 0, channel] = np.inf if i % 2 else -np.inf
    case.x[41, 0, channels[0]] = np.inf                     # of a page that has rows
    case.x[42, 0, 449] = np.nan                             # beside numbers: none of the page's scale
    case.operator().run()
    case.check(*case.expect())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("channel", [448, 449, 479, 480, 510, 511])
def test_an_infinity_on_its_own(kind, channel):
    case = angled(Appended(44, [2, 1], [2, 20], kind=kind), 1.0)
    case.x[0, 0, channel] = case.x[2, 0, channel] = np.inf
    case.operator().run()
    case.check(*case.expect())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("pairs", [True, False])
def test_products_past_the_largest_number(kind, pairs):
    """A rotation longer than 1: finite values whose products pass FP32, and some that come back below it."""
    case = angled(Appended(45, [40, 3], [70, 9], kind=kind, pairs=pairs), 4.0)
    case.x[2, 0, 448:] *= 1e38
    case.x[41, 0, 449::2] *= 1e38
    case.x = cases.bf16(case.x)
    case.operator().run()
    case.check(*case.expect())


def again(case, new, length, written, size):
    """The first request's last `new` rows given again, all but `written` with positions outside the rotation; the rows."""
    import torch
    from npu_sparse_attn_sharedkv_int8 import PreparedCacheAppend
    put = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    x = cases.bf16(case.rng.standard_normal((new, 1, DIM)) * size)
    places = np.where(np.arange(new) % 2, -1, len(case.rotation)).astype(np.int32)
    for row in written:
        places[row - (length - new)] = row
    PreparedCacheAppend(case.cache, put(x).to(torch.bfloat16), put(case.table[:1]), put(np.array([0, new], np.int32)),
                        put(np.array([length], np.int32)), scale=case.scale, rotation=put(case.rotation),
                        positions=put(places)).run()
    return x


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("length", [33, 40])
def test_pages_of_skipped_rows_keep_their_scales(kind, length):
    """Rows that are in the cache already, given again with positions outside the rotation: nothing changes."""
    case = Appended(46, [length, 5], [length, 5], kind=kind)
    case.operator().run()
    codes, scale = case.expect()
    case.check(codes, scale)
    again(case, length - BLOCK, length, [], 50.0)           # the second page's rows, all of them
    case.check(codes, scale)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size", [0.1, 40.0])
def test_rows_behind_skipped_ones(kind, size):
    """A prompt of which 40 rows are in the cache, given whole: the rest goes behind them, as if given alone."""
    case = Appended(48, [40, 1], [40, 60], kind=kind)
    case.operator().run()
    codes, scale = case.expect()
    x = again(case, 45, 45, range(40, 45), size)
    turned = cases.rotated(x[40:].astype(np.float64), case.rotation, np.arange(40, 45), True)
    cases.append(codes, scale, kind, turned, case.table[:1], [0, 5], [45])
    case.check(codes, scale)


@pytest.mark.parametrize("kind", KINDS)
def test_a_row_between_skipped_ones(kind):
    """It is replaced, and all others of the page go over to the scale that it takes."""
    case = Appended(49, [45, 1], [45, 60], kind=kind)
    case.operator().run()
    codes, scale = case.expect()
    x = again(case, 13, 45, [38], 40.0)
    page, old = case.table[0, 1], scale.copy()
    turned = cases.rotated(x[6:7].astype(np.float64), case.rotation, np.array([38]), True)
    cases.append(codes, scale, kind, turned, case.table[:1], [0, 1], [39])
    grown = scale[page, 0] / old[page, 0]
    assert grown > 1
    codes[page, 7:13] = cases.encode(cases.decode(codes[page, 7:13], kind) / grown, kind)
    case.check(codes, scale)
