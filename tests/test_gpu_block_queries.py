"""PreparedBlockAttention with queries of which a few channels are far larger than
the others, against 64 bits, with bounds by the row's mean and not by its largest
value; every unit size (16, 32 and 64 query rows), split contexts among them."""
import math

import numpy as np
import pytest

from tests.block_cases import Attend, bf16, BLOCK, DIM
from tests.test_gpu_block_attention import run

pytestmark = pytest.mark.gpu
KINDS = ["int8", "e4m3"]
# Table pages by which 512 query rows over whole contexts take units of 16, 32 or 64 rows.
WIDTH = {1: 100, 2: 400, 4: 12500}


def attend_of(rt, seed, kind, **kw):
    """8 tokens of 64 heads (512 query rows) over 300 and 700 rows."""
    a = Attend(seed, [3, 5], [300, 700], heads=64, kind=kind, **kw)
    wide = np.full((2, WIDTH[rt]), -1, np.int32)
    wide[:, :a.ori_table.shape[1]] = a.ori_table
    a.ori_table = wide
    return a


def launch(a, rt):
    op = run(a)
    assert op.partial.numel() % (16 * rt * (DIM + 2)) == 0
    rows = 8 * 64
    tiles = (WIDTH[rt] + 1) // 2
    most = min(rows // (16 * rt) + 2, 8 * -(-64 // (16 * rt))) + 1       # units that the launch makes room for
    assert op.partial.numel() == min(512, -(-most * tiles // 8) * 8) * 16 * rt * (DIM + 2)
    return op


def compare(a, op, rows=None):
    """Out and log-sum-exp of the rows [token, head] that are True (all).

    Bounds.  INT8 holds a row of Q in whole numbers of one unit, a power of two
    of which the smaller of the row's largest |q| and 8 times its mean |q| takes
    more than 16256: off by half a unit, min / 32512, at most.  e4m3 takes Q as it
    is.  The rest is as in block_cases.Attend.expect: sums 2^-20 sum_c |q code|,
    score and lift 2^-21 (1.5 max|s| + max|lift| + 24), a weight twice all that, 2^-11 (FP16)
    and 2^-17; the output's rounding 2^-8, weights that fall below FP16's numbers 2^-33."""
    q = bf16(a.q).astype(np.float64)
    got, got_lse = op.out.float().cpu().numpy().astype(np.float64), op.lse.cpu().numpy().astype(np.float64)
    rows = np.ones(q.shape[:2], bool) if rows is None else rows
    scale_of = abs(a.softmax_scale)
    for b, (n, length) in enumerate(zip(a.new, a.lengths)):
        for i in range(n):
            t, place = a.cu[b] + i, length - n + i
            code, scale = a.rows(a.ori, a.ori_table, b, np.arange(place + 1), 0)
            sink = a.sink.astype(np.float64)
            with np.errstate(invalid="ignore"):
                s = q[t] @ code.T * scale * a.softmax_scale
                top = np.maximum(s.max(1), sink)
                e = np.exp(s - top[:, None])
                total = e.sum(1) + np.exp(sink - top)
                p = e / total[:, None]
                size = np.abs(q[t])
                half = np.zeros(len(size)) if a.kind == "e4m3" else np.minimum(size.max(1), 8 * size.mean(1) * (1 + 2 ** -20)) / 32512
                d = scale_of * half * (np.abs(code).sum(1) * scale).max()
                d += scale_of * 2.0 ** -20 * (size @ np.abs(code).T * scale).max(1)
                d += 2.0 ** -21 * (1.5 * np.abs(s).max(1) + np.abs(np.log2(scale)).max() + 24)
                want, value = p @ (code * scale[:, None]), np.abs(code) * scale[:, None]
                near = 2.0 ** -8 * np.abs(want) + (2 * d + 2.0 ** -11 + 2.0 ** -17)[:, None] * (p @ value) \
                    + 2.0 ** -33 * (p * scale).max(1)[:, None] * np.abs(code).sum(0)
                lse = top + np.log(total)
                lse_near = d + 2.0 ** -21 * np.abs(lse) + 2.0 ** -19
            its = rows[t]
            assert (np.abs(got[t] - want) <= near)[its].all(), (t, np.abs(got[t] - want)[its].max())
            off = np.abs(got_lse[t] - lse) - lse_near
            assert (off <= 0)[its].all(), (t, off[its].max())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rt", [1, 2, 4])
@pytest.mark.parametrize("size,softmax_scale", [(30, 1 / 22.6), (100, 1 / 22.6), (300, 1 / 22.6), (3000, -1 / 500)])
def test_a_channel_far_larger(kind, rt, size, softmax_scale):
    a = attend_of(rt, 60, kind, softmax_scale=softmax_scale)
    a.q[:, :, 77] = size
    a.q[:, 1::2, 400] = -size / 3
    a.q[:, 5] = a.rng.standard_normal(DIM)                  # rows without, beside rows with
    compare(a, launch(a, rt))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rt", [1, 2, 4])
def test_rows_of_every_spread(kind, rt):
    """Heavy tails, single channels, zeros; and rows that are no numbers beside them."""
    a = attend_of(rt, 61, kind, softmax_scale=1 / 300)
    a.q *= np.exp(2.5 * a.rng.standard_normal(a.q.shape))   # log-normal: largest some 100 times the mean
    a.q[:, 2] = 0
    a.q[:, 3] = 0
    a.q[:, 3, 511] = 7.0                                    # the largest is 512 times the mean
    a.q[:, 4] = 0
    a.q[:, 4, [0, 64]] = [-1e-3, 1e3]
    a.q[:, 5] = 1.0                                         # all alike
    a.q[:, 6] *= 1e-30
    compare(a, launch(a, rt))
    a.q[1, 7, 9], a.q[6, 33, 300] = np.nan, np.inf
    op = launch(a, rt)
    rows = np.ones((8, 64), bool)
    rows[1, 7] = rows[6, 33] = False
    compare(a, op, rows)
    out = op.out.float().cpu().numpy()
    assert np.isnan(out[1, 7]).all() and np.isnan(out[6, 33]).all()


@pytest.mark.parametrize("kind", KINDS)
def test_one_token_over_a_long_context(kind):
    """Units of 16 rows, split; two thousand keys decide the log-sum-exp."""
    a = Attend(62, [1], [6000], heads=8, kind=kind)
    a.q[:, :, 3], a.q[:, 4:, 200] = 100, -300
    op = run(a)
    assert op.partial is not None
    compare(a, op)
