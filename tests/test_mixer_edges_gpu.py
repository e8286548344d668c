"""The state space mixer's entries at the ends of their ranges, against their definitions in float64."""
import ctypes as C

import numpy as np
import pytest

from tests import state_space_plain as P
from tests.test_state_space_gpu import _np, _Rows, _table
from uzu_b200 import binding as B

pytestmark = pytest.mark.gpu

FAR = [-41.0, -42.0, -50.0, -60.0, -87.0, -88.0, -100.0, -104.0, -1e4, -1e18, -2.0 ** 62, -1e20, -1e30, 0.0, 1e-30, 0.5, 20.0, 1e20, float("inf"), float("-inf"), float("nan"), -0.25, 3.0, -1e-30]


def _run_conv(ctx, u, w, seqs, dt, slots, shift=0, act=B.ACT_SILU, state=None):
    """(rows of output, state): float64 values of what the device holds"""
    rows, channels = u.shape
    taps = w.shape[1]
    x, out = _Rows(ctx, u, dt, shift=shift), _Rows(ctx, np.zeros((rows, channels)), dt, shift=shift)
    st = np.zeros((slots, max(taps - 1, 1), channels)) if state is None else state
    sb, wb, t = ctx.upload(P.to_kept(st, dt)), ctx.upload(w.astype(np.float32)), _table(seqs)
    a = B.CausalConvArgs(input=x.ptr, output=out.ptr, weights=wb.ptr, bias=0, state=sb.ptr if taps > 1 else 0, sequences=C.addressof(t), sequence_count=len(seqs), rows=rows, slots=slots,
                         channels=channels, taps=taps, input_stride=x.stride, output_stride=out.stride, activation=act, data_type=dt)
    with ctx.command_buffer("conv") as cmd:
        cmd.encode("uzu_causal_conv_encode", C.byref(a))
    return out.get()[0], P.of_kept(sb.numpy(_np(dt), st.shape), dt)


@pytest.mark.parametrize("dt", [P.BF16, P.F32, P.F16])
@pytest.mark.parametrize("shift", [0, 1])
def test_conv_gate_far_from_zero(ctx, dt, shift):
    """silu of sums far below zero, infinite, tiny or no number, each beside each in one row's neighbouring channels: every row is a sequence of one tap with weight 1"""
    v = np.array(FAR)
    u = np.empty((len(v), 2 * len(v)))
    u[:, 0::2], u[:, 1::2] = v[:, None], v[None, :]
    got, _ = _run_conv(ctx, u, np.ones((u.shape[1], 1)), [(i, 1, i, 1) for i in range(len(v))], dt, len(v), shift)
    x = P.of_kept(P.to_kept(u, dt), dt)
    with np.errstate(invalid="ignore"):
        ref = P.silu(x)
    finite = np.isfinite(ref)
    assert finite.any() and np.array_equal(np.isnan(got), np.isnan(ref)) and np.array_equal(got[np.isinf(ref)], ref[np.isinf(ref)])
    x, ref, got = x[finite], ref[finite], got[finite]
    # an exponential of x log2 e (its own error, the exponent's rounding), at most six more roundings; below 2^-126 the exponential's last place is 2^-149
    bound = (2.0 ** -21 + 2.0 ** -22 * np.minimum(np.abs(x), 200.0)) * np.abs(ref) + np.minimum(np.abs(x), 2.0 ** 100) * 2.0 ** -149
    assert (np.abs(got - ref) <= P.HALF_STEP[dt] * (np.abs(ref) + bound) + P.TINY[dt] + bound).all(), [(a, b, c) for a, b, c, m in zip(x, got, ref, np.abs(got - ref) > bound + P.HALF_STEP[dt] * np.abs(ref) + P.TINY[dt]) if m][:8]


@pytest.mark.parametrize("dt", [P.BF16, P.F32])
@pytest.mark.parametrize("channels,taps", [(40, 4), (33, 2), (64, 8)])
def test_conv_gate_of_large_sums(ctx, dt, channels, taps):
    """many sums far below zero, in the first strip behind a slot's inputs and in later ones; the slots take their new inputs all the same"""
    rng = np.random.default_rng(channels)
    seqs, rows = [(0, 150, 1, 0), (150, 3, 0, 0), (153, 90, 2, 1)], 243
    u, w, st = 30 * rng.standard_normal((rows, channels)), rng.standard_normal((channels, taps)).astype(np.float32), 30 * rng.standard_normal((3, taps - 1, channels))
    got, state = _run_conv(ctx, u, w, seqs, dt, 3, state=st)
    k = lambda v: P.of_kept(P.to_kept(v, dt), dt)
    ref, after, mag = P.conv(k(u), w.astype(np.float64), np.zeros(channels), k(st), seqs)
    # the bound of the convolution's other tests: taps + 1 additions in 32 bits, an exponential of a value of up to `mag`
    bound = 1.1 * (taps + 2) * 2.0 ** -24 * mag + (2.0 ** -21 + 2.0 ** -22 * mag) * np.abs(ref)
    far = ref[(ref > -1e-15) & (ref < 0)]
    assert far.size > rows
    assert (np.abs(got - ref) <= P.HALF_STEP[dt] * (np.abs(ref) + bound) + P.TINY[dt] + bound).all() and np.array_equal(state, after)
    # the sums' own errors move such a value by a part of itself only
    small = (ref > -1e-15) & (ref < 0)
    part = (taps + 4) * 2.0 ** -23 * mag + 2.0 ** -20 + P.HALF_STEP[dt]
    assert (np.abs(got - ref) <= part * np.abs(ref) * 1.1 + P.TINY[dt] + np.minimum(mag, 1000) * 2.0 ** -149)[small].all()


@pytest.mark.parametrize("dt", [P.BF16, P.F32])
@pytest.mark.parametrize("taps", [1, 2, 3, 4, 5, 6, 7, 8])
@pytest.mark.parametrize("act", [B.ACT_SILU, B.ACT_IDENTITY])
def test_conv_infinite_inputs_reach_their_window_only(ctx, dt, taps, act):
    """an input that is infinite or no number shows in the taps rows that read it, in its channel, and nowhere else"""
    rng = np.random.default_rng(taps)
    rows, channels, seqs = 60, 24, [(0, 45, 1, 0), (45, 15, 0, 1)]
    u, w, st = rng.standard_normal((rows, channels)), rng.standard_normal((channels, taps)), rng.standard_normal((2, max(taps - 1, 1), channels))
    clean, _ = _run_conv(ctx, u, w, seqs, dt, 2, act=act, state=st)
    hit = np.zeros((rows, channels), bool)
    for row, channel, value in [(3, 2, np.inf), (20, 9, np.nan), (31, 23, -np.inf), (44, 5, np.inf), (46, 0, np.nan)]:
        u[row, channel] = value
        hit[row:min(row + taps, 45 if row < 45 else rows), channel] = True
    got, _ = _run_conv(ctx, u, w, seqs, dt, 2, act=act, state=st)
    assert not np.isfinite(got[hit]).any()
    beside = ~hit & hit.reshape(rows, channels // 2, 2)[:, :, ::-1].reshape(rows, channels)      # the gate takes one reciprocal for two channels: 2^-21 of the value each time, and its rounding
    assert np.array_equal(got[~hit & ~beside], clean[~hit & ~beside])
    assert (np.abs(got - clean)[beside] <= (2.0 ** -20 + 2 * P.HALF_STEP[dt]) * np.abs(clean[beside])).all()
