"""The 8-bit cache's attention at the ends of its range: values that are no numbers beside weights that are summed, queries and caps of any size, one scratch for calls of many sizes, sequences longer than was said."""
import ctypes as C

import numpy as np
import pytest

from tests import quantized_cache_plain as Q
from tests import state_space_plain as P
from tests.quantized_cache_gpu import Served
from uzu_b200 import binding as B

pytestmark = pytest.mark.gpu

ALL = 0xFFFFFFFF
TYPES = [P.BF16, P.F32, P.F16]


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


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("dim,heads", [(64, 8), (128, 8), (64, 2), (256, 4)])
def test_one_scratch_for_many_calls(ctx, dt, dim, heads):
    """what is asked for before there are pointers, for the largest pass, is enough for every smaller one, wherever its rows are"""
    s = Served(ctx, Q.I8, 32, 2, dim, [300, 280, 5], room=420)
    most = [70, 9, 70]
    s.append(most, P.F32)
    a = B.QuantizedCacheAttentionArgs(cache=s.cache(), sequences=s.sequences(most, sum(most) + 2), heads=heads, query_row_stride=heads * dim, query_head_stride=dim, out_stride=heads * dim, weight_rows=ALL,
                                      scale=0.125, data_type=dt)
    size = ctx.lib.uzu_quantized_cache_attention_scratch_bytes(ctx.h, C.byref(a))
    scratch = ctx.upload(np.zeros(size, np.uint8))
    before = s.device_weights()
    for rows, kw in (([70, 9, 70], dict()), ([70, 9, 70], dict(shift=1, stride=heads * dim + 3)), ([17, 9, 3], dict(shift=1)), ([17, 9, 3], dict()), ([9, 8, 9], dict(scale=-0.125)), ([1, 1, 1], dict(window=40, first=3)),
                     ([5, 4, 5], dict(weight_rows=0)), ([33, 0, 0], dict(max_length=333)), ([0, 5, 1], dict(cap=30.0))):
        kw = dict(dict(weight_rows=ALL), **kw)
        query = s.rng.standard_normal((sum(rows) + 2, heads * dim))
        want, _ = s.attend(rows, heads, dt, query=query, check=False, **kw)
        b, out = B.QuantizedCacheAttentionArgs.from_buffer_copy(s.last), s.kept[-3]
        assert out.ptr == b.out and b.scratch_bytes <= size, (rows, kw, b.scratch_bytes, size)
        # the same call once more in the large scratch: the same bits
        b.scratch, b.scratch_bytes = scratch.ptr, size
        s.run("attention", ("uzu_quantized_cache_attention_encode", b))
        assert np.array_equal(out.get()[0], want)
    assert np.isfinite(before).all()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("cap", [1e-38, 1e-12, 1e-3, 60.0, 1e3, 1e5, 1e9, 3e38])
@pytest.mark.parametrize("rows,heads", [([3, 1], 4), ([40, 50], 4), ([90, 20], 8)])
def test_caps_of_any_size(ctx, dt, cap, rows, heads):
    """a cap far above the scores leaves them as they are, one far below makes them alike"""
    s = Served(ctx, Q.I8, 32, 2, 64, [70, 130], room=260)
    s.append(rows, P.F32)
    cap = float(np.float32(cap))
    query = s.rng.standard_normal((sum(rows) + 2, heads * 64))
    before = s.device_weights()
    got, grown = s.attend(rows, heads, dt, query=query, cap=cap, weight_rows=ALL, check=False)
    assert np.isfinite(got).all()
    at, want_weights = 0, before.copy()
    slack = np.zeros_like(before)
    for i, n in enumerate(rows):
        mine = P.of_kept(P.to_kept(query[at:at + n], dt), dt).reshape(n, heads, 64)
        tensor = dt == P.BF16 and n > 8 and n * heads // 2 > 64
        ref, bound, grow, grow_bound = s.plain.attend(s.table[i], s.lengths[i], mine, s.capacity(), float(np.float32(0.125)), cap=cap, weight_rows=ALL, q_error=2.0 ** -22 if dt == P.F32 else 0.0, tensor=tensor)
        # Capped scores of 16-bit rows may be off by 2^-21 of caps of up to 64, with larger ones by two units in the last place of themselves, as f32 rows' are: each weight by twice that, scores' and the largest's
        off = 2 * (2.0 ** -21 * cap if dt != P.F32 and cap <= 64 else 2.0 ** -21 * min(cap, 40.0))
        bound += off * 2 * np.abs(s.plain.numbers(1, s.table[i], np.arange(s.lengths[i] + n))[0]).max()
        grow_bound += off * 2 * grow
        assert np.abs(ref).max() > 0.01
        tol = P.HALF_STEP[dt] * (np.abs(ref) + bound) + P.TINY[dt] + bound
        worst = np.abs(got[at:at + n].reshape(ref.shape) - ref) / tol
        assert worst.max() <= 1, (i, float(worst.max()))
        tokens = np.arange(len(grow))
        b = s.table[i][tokens // 32]
        want_weights[b, :, tokens % 32] += grow
        slack[b, :, tokens % 32] += grow_bound
        at += n
    after = s.device_weights()
    assert (np.abs(after - want_weights) <= slack + 2.0 ** -24 * (1 + max(rows) * heads / 16) * np.abs(want_weights) + 1e-30).all()


def _held(s, rows, heads, dt, max_length, window, first):
    """attention with weights against the definition"""
    query = s.rng.standard_normal((sum(rows) + 2, heads * 64))
    before = s.device_weights()
    got, _ = s.attend(rows, heads, dt, query=query, max_length=max_length, window=window, first=first, weight_rows=ALL, check=False)
    want, slack, at = before.copy(), np.zeros_like(before), 0
    for i, n in enumerate(rows):
        mine = P.of_kept(P.to_kept(query[at:at + n], dt), dt).reshape(n, heads, 64)
        given = (s.table[i], s.lengths[i], mine, s.capacity(max_length), float(np.float32(0.125)), window, first, 0.0, None, ALL, 2.0 ** -22 if dt == P.F32 else 0.0)
        ref, bound, grow, grow_bound = s.plain.attend(*given)
        if dt == P.BF16 and n > 8 and n * heads // 2 > 64:
            # Weights are one f16 number there. F16 numbers are 2^-10 apart from 1 to 2: a rounding is off by up to 2^-11 of the value, which is twice what the form's bound takes for it
            bound = bound + 2 * (s.plain.attend(*given, tensor=True)[1] - bound)
        mine_got = got[at:at + n].reshape(ref.shape)
        tol = P.HALF_STEP[dt] * (np.abs(ref) + bound) + P.TINY[dt] + bound
        assert (np.abs(mine_got - ref) <= tol).all(), (i, float((np.abs(mine_got - ref) / tol).max()))
        tokens = np.arange(len(grow))
        b = s.table[i][tokens // s.plain.block]
        want[b, :, tokens % s.plain.block] += grow
        slack[b, :, tokens % s.plain.block] += grow_bound
        at += n
    # (an addition for each tile of 16 pairs)
    assert (np.abs(s.device_weights() - want) <= slack + 2.0 ** -24 * (1 + max(rows) * heads / 16) * np.abs(want) + 1e-30).all()
    s.plain.weights = s.device_weights()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rows", [[1, 1, 1], [3, 20, 9], [70, 40, 50]])
@pytest.mark.parametrize("window,first", [(0, 0), (7, 0), (40, 5), (100, 20)])
def test_sequences_behind_max_length(ctx, dt, rows, window, first):
    """keys behind max_length are left out, and rows stay the tokens that they are: windows that begin behind it are empty"""
    s = Served(ctx, Q.I8, 16, 2, 64, [60, 20, 150], room=240)
    s.append(rows, P.F32)
    for max_length in (50, 64, 23):
        _held(s, rows, 8, dt, max_length, window, first)
