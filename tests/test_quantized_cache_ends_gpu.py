"""The 8-bit cache's attention at the ends of its range: values that are no numbers beside weights that are summed, queries of any size."""
import numpy as np
import pytest

from tests import quantized_cache_plain as Q
from tests import state_space_plain as P
from tests.quantized_cache_gpu import Served

pytestmark = pytest.mark.gpu

ALL = 0xFFFFFFFF


@pytest.mark.parametrize("dt,apart", [(P.BF16, False), (P.F32, False), (P.F16, False), (P.BF16, True), (P.F32, True)])      # (values of 2^40 are no f16 numbers)
@pytest.mark.parametrize("lengths,rows", [([100, 40], [1, 1]), ([100, 40], [20, 30]), ([100, 40], [90, 70]), ([400, 260], [90, 70])])
def test_weights_beside_values_that_are_no_numbers(ctx, dt, apart, lengths, rows):
    """a value block without a number makes the rows NaN that see it; their weights are of scores, which are numbers"""
    s = Served(ctx, Q.I8, 16, 2, 64, lengths, room=500)
    s.append(rows, P.F32)
    if apart:
        for i in range(2):
            for k in range(len(s.table[0])):
                s.plain.scales[1][s.table[i, k]] = 2.0 ** [-60, 40, -5, -30, 20][(k + i) % 5]
    for which in ([(0, 2, 1), (1, 3, 0)], [(0, 0, 1), (1, 1, 0), (1, 2, 0)]):
        for i, k, h in which:
            s.plain.scales[1][s.table[i, k], h] = np.nan
        s.scales = [ctx.upload(x.astype(np.float32)) for x in s.plain.scales]
        got = s.attend(rows, 4, dt, weight_rows=ALL)
        assert np.isnan(got).any() and not np.isnan(got).all()
        s.attend(rows, 4, dt, window=30, weight_rows=ALL)
        s.attend(rows, 4, dt, window=50, first=8, cap=20.0, sinks=[0.5, -1.0, 0.0, 3.0], weight_rows=5)


@pytest.mark.parametrize("dt,power", [(P.F32, 123), (P.BF16, 123), (P.F32, 116), (P.BF16, 116), (P.F32, -121), (P.BF16, -121), (P.F32, -100), (P.BF16, -100)])
@pytest.mark.parametrize("rows", [[3], [40]])
@pytest.mark.parametrize("cap", [0.0, 20.0])
def test_queries_of_any_size(ctx, dt, power, rows, cap):
    """finite queries from one end of the type to the other, with a scale that makes scores of them"""
    s = Served(ctx, Q.I8, 32, 1, 64, [70], room=200)
    s.append(rows, P.F32)
    x = np.clip(s.rng.standard_normal((rows[0] + 2, 4 * 64)), -7, 7) * 2.0 ** power
    s.attend(rows, 4, dt, query=x, scale=2.0 ** -(power + 3), cap=cap, weight_rows=2)
