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
    with np.errstate(over="ignore", invalid="ignore"):
        got, _ = _run_conv(ctx, u, np.ones((u.shape[1], 1)), [(i, 1, i, 1) for i in range(len(v))], dt, len(v), shift)
        x = P.of_kept(P.to_kept(u, dt), dt)
        ref = P.silu(x)
    finite = np.isfinite(ref)
    assert finite.any() and np.array_equal(np.isnan(got), np.isnan(ref)) and np.array_equal(got[np.isinf(ref)], ref[np.isinf(ref)])
    x, ref, got = x[finite], ref[finite], got[finite]
    # an exponential of x log2 e (its own error, the exponent's rounding), at most six more roundings. Below -87.3 the reciprocal of 1 + e^-x is no normal number any more and taken as 0:
    # off by the value, which is less than 88 * 2^-126 there, and 0 where e^-x is infinite in 32 bits
    bound = (2.0 ** -21 + 2.0 ** -22 * np.minimum(np.abs(x), 200.0)) * np.abs(ref) + np.where(x < -87.3, np.abs(ref), 0.0)
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
    none = np.where(np.abs(ref) < 2.0 ** -119, np.abs(ref), 0.0)      # (0 below -87.3)
    assert (np.abs(got - ref) <= part * np.abs(ref) * 1.1 + P.TINY[dt] + none)[small].all()


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
    assert np.array_equal(got[~hit], clean[~hit])


def _run_scan(ctx, v, heads, groups, dim, n, seqs, slots, dt=P.BF16, state=None, scratch=True):
    """v: x, z, b, c, dt rows, a, d, dt_bias. (out, state) in float64"""
    rows = v["x"].shape[0]
    X, Z, Bm, Cm, D = (_Rows(ctx, v[k], dt) for k in ("x", "z", "b", "c", "dt"))
    out = _Rows(ctx, np.zeros((rows, heads * dim)), dt)
    st = np.zeros((slots, heads, dim, n), np.float32) if state is None else state
    f32 = [ctx.upload(np.asarray(w, np.float32)) for w in (v["a"], v["d"], v["dt_bias"], st)]
    t = _table(seqs)
    a = B.StateSpaceScanArgs(x=X.ptr, dt=D.ptr, b=Bm.ptr, c=Cm.ptr, z=Z.ptr, a=f32[0].ptr, d=f32[1].ptr, dt_bias=f32[2].ptr, state=f32[3].ptr, out=out.ptr, sequences=C.addressof(t),
                             sequence_count=len(seqs), rows=rows, slots=slots, heads=heads, groups=groups, head_dim=dim, state_size=n, x_stride=X.stride, dt_stride=D.stride, b_stride=Bm.stride,
                             c_stride=Cm.stride, z_stride=Z.stride, out_stride=out.stride, dt_min=0.0, dt_max=float("inf"), dt_softplus=1, data_type=dt)
    if scratch:
        a.scratch_bytes = ctx.lib.uzu_state_space_scan_scratch_bytes(ctx.h, C.byref(a))
        sc = ctx.buffer(max(16, a.scratch_bytes), B.BUFFER_DEVICE)
        a.scratch = sc.ptr
    with ctx.command_buffer("scan") as cmd:
        cmd.encode("uzu_state_space_scan_encode", C.byref(a))
    return out.get()[0], f32[3].numpy(np.float32, st.shape).astype(np.float64), a.scratch_bytes


def _scan_rows(rng, rows, heads, groups, dim, n):
    v = {k: rng.standard_normal((rows, w)) for k, w in (("x", heads * dim), ("z", heads * dim), ("b", groups * n), ("c", groups * n), ("dt", heads))}
    v["a"], v["d"], v["dt_bias"] = -(1 + 15 * rng.random(heads)), rng.standard_normal(heads), np.zeros(heads)
    return v


@pytest.mark.parametrize("dim,n", [(64, 128), (128, 64)])
@pytest.mark.parametrize("loud", [32, 64, 96])
def test_quiet_tokens_behind_loud_ones(ctx, dim, n, loud):
    """Tokens of large steps and no input wipe the state out and add nothing: what follows in their chunk is as without them, to the bit (blocks of 32 tokens have sums of their own; a
    difference of sums over the loud tokens too would lose the quiet ones' digits)."""
    heads, groups = 32, 2
    v = _scan_rows(np.random.default_rng(loud), 128, heads, groups, dim, n)
    v["dt"] -= 4.0                       # steps of about 0.02
    v["dt"][:loud], v["x"][:loud] = 40.0, 0.0
    behind = {k: w[loud:] if w.shape[0] == 128 else w for k, w in v.items()}
    out, state, _ = _run_scan(ctx, v, heads, groups, dim, n, [(0, 128, 0, 1)], 1)
    ref, after, _ = _run_scan(ctx, behind, heads, groups, dim, n, [(0, 128 - loud, 0, 1)], 1)
    assert np.isfinite(out).all() and not out[:loud].any() and ref.any()
    assert np.array_equal(out[loud:], ref) and np.array_equal(state, after)


@pytest.mark.parametrize("dim,n", [(64, 128), (128, 64)])
def test_loud_and_quiet_tokens(ctx, dim, n):
    """steps of 1e-3 and of 40 side by side, against the recurrence in 64 bits, whose errors are carried along token by token"""
    heads, groups, rows = 4, 2, 300
    rng = np.random.default_rng(dim)
    v = _scan_rows(rng, rows, heads, groups, dim, n)
    v["dt"] = np.where(rng.random((rows, heads)) < 0.3, 40.0, rng.standard_normal((rows, heads)) - 5)
    v["dt"][40:90] -= 45.0 * (v["dt"][40:90] > 20)       # a quiet stretch
    st = rng.standard_normal((1, heads, dim, n)).astype(np.float32)
    out, state, _ = _run_scan(ctx, v, heads, groups, dim, n, [(0, rows, 0, 0)], 1, state=st)
    k = lambda w, *s: P.of_kept(P.to_kept(w, P.BF16), P.BF16).reshape(rows, *s)
    x, z, b, c = k(v["x"], heads, dim), k(v["z"], heads, dim), k(v["b"], groups, n), k(v["c"], groups, n)
    a, d = v["a"].astype(np.float32).astype(np.float64), v["d"].astype(np.float32).astype(np.float64)
    step = P.steps(k(v["dt"], heads), 0.0)
    ref, rstate, mag, smag = P.scan(x, step, b, c, z, a, d, st.astype(np.float64), [(0, rows, 0, 0)])
    # Of a decay over several tokens: each token's own part |step a| of it with three roundings, and a block's sum (at most 32 of 150) with six where it is a difference of two.
    # e, m: errors and magnitudes of the state in the recurrence over absolute values
    bb = np.repeat(np.abs(b), heads // groups, 1)
    m = np.abs(st[0]).astype(np.float64)
    e = np.zeros_like(m)
    bound = np.zeros_like(ref)
    cc = np.repeat(np.abs(c), heads // groups, 1)
    for t in range(rows):
        l = np.minimum(np.abs(step[t] * a), 104.0)
        f = np.exp(-np.abs(step[t] * a))[:, None, None]
        add = (step[t][:, None] * np.abs(x[t]))[:, :, None] * bb[t][:, None, :]
        e = f * (e + 2.0 ** -24 * (4 + 8 * l)[:, None, None] * m) + 2.0 ** -24 * 6 * add
        m = f * m + add
        bound[t] = (e * cc[t][:, None, :]).sum(-1)
    # the state's sum: inputs as two bf16 parts
    assert (np.abs(state[0] - rstate[0]) <= e + 2.0 ** -16 * m + 2.0 ** -24 * np.abs(rstate[0]) + 2.0 ** -140).all()
    gate = np.abs(P.silu(z))
    bound = bound + (2.0 ** -8 + np.log(2) * 6 * 2.0 ** -24 * 32 * 150 + 2.0 ** -24 * (n + 8)) * mag
    bound = bound * gate + (2.0 ** -21 + 2.0 ** -22 * np.abs(z)) * np.abs(ref)
    got = out.reshape(rows, heads, dim)
    assert np.isfinite(got).all()
    assert (np.abs(got - ref) <= P.HALF_STEP[P.BF16] * (np.abs(ref) + bound) + P.TINY[P.BF16] + bound).all()


@pytest.mark.parametrize("dt,dim,n", [(P.BF16, 64, 128), (P.BF16, 128, 64), (P.F32, 20, 12)])
def test_a_step_that_is_no_number(ctx, dt, dim, n):
    """makes its head's outputs from its token on and its head's state no number; nothing before it, no other head"""
    heads, groups, rows = 4, 2, 300
    v = _scan_rows(np.random.default_rng(7), rows, heads, groups, dim, n)
    v["dt"] -= 3.0
    clean, cstate, _ = _run_scan(ctx, v, heads, groups, dim, n, [(0, rows, 0, 1)], 1, dt=dt)
    for row in (0, 45, 127, 128, 201, 299):
        w = dict(v, dt=v["dt"].copy())
        w["dt"][row, 1] = np.nan
        out, state, _ = _run_scan(ctx, w, heads, groups, dim, n, [(0, rows, 0, 1)], 1, dt=dt)
        hit = np.zeros((rows, heads, dim), bool)
        hit[row:, 1] = True
        out, ref = out.reshape(hit.shape), clean.reshape(hit.shape)
        assert np.isnan(out[hit]).all() and np.array_equal(out[~hit], ref[~hit])
        others = [0, 2, 3]
        assert np.isnan(state[0, 1]).all() and np.array_equal(state[0, others], cstate[0, others])


@pytest.mark.parametrize("shift", [-4.0, -8.0])
@pytest.mark.parametrize("cut", [(2, 1, 64, 128, [(0, 2500, 1, 0)]), (4, 4, 64, 64, [(0, 1500, 0, 0), (1500, 40, 1, 1)]), (2, 2, 128, 64, [(3, 1290, 0, 1)])])
def test_parts_and_whole_agree(ctx, cut, shift):
    """the same rows in parts (with a scratch), whole, and whole again: the whole ones to the bit, the parts within both sides' roundings of the recurrence"""
    heads, groups, dim, n, seqs = cut
    rows = max(f + m for f, m, _, _ in seqs)
    rng = np.random.default_rng(rows)
    v = _scan_rows(rng, rows, heads, groups, dim, n)
    v["dt"] += shift
    st = rng.standard_normal((2, heads, dim, n)).astype(np.float32)
    parts, pstate, scratch = _run_scan(ctx, v, heads, groups, dim, n, seqs, 2, state=st)
    whole, wstate, _ = _run_scan(ctx, v, heads, groups, dim, n, seqs, 2, state=st, scratch=False)
    again, astate, _ = _run_scan(ctx, v, heads, groups, dim, n, seqs, 2, state=st, scratch=False)
    assert scratch > 0 and np.array_equal(whole, again) and np.array_equal(wstate, astate)
    k = lambda w, *s: P.of_kept(P.to_kept(w, P.BF16), P.BF16).reshape(rows, *s)
    a = v["a"].astype(np.float32).astype(np.float64)
    step = P.steps(k(v["dt"], heads), 0.0)
    z = k(v["z"], heads, dim)
    ref, state, mag, smag = P.scan(k(v["x"], heads, dim), step, k(v["b"], groups, n), k(v["c"], groups, n), z, a, v["d"].astype(np.float32).astype(np.float64), st.astype(np.float64), seqs)
    # a token's decay is off by three roundings and |step a| of four, its state by two; over the longest sequence, for the head of the largest sum
    unit = 2.0 ** -24 * (max(5 * m + 4 * float(np.abs(step * a)[f:f + m].sum(0).max()) for f, m, _, _ in seqs) + n + 8)
    assert (np.abs(pstate - wstate) <= 2 * ((unit + 2.0 ** -16) * smag + 2.0 ** -24 * np.abs(state))).all()
    cov = np.zeros(rows, bool)
    for f, m, _, _ in seqs:
        cov[f:f + m] = True
    bound = ((unit + 2.0 ** -8) * mag * np.abs(P.silu(z)) + (2.0 ** -21 + 2.0 ** -22 * np.abs(z) + P.HALF_STEP[P.BF16]) * np.abs(ref))[cov]
    assert (np.abs(parts - whole).reshape(ref.shape)[cov] <= 2 * 1.01 * bound + P.TINY[P.BF16]).all()


@pytest.mark.parametrize("dt", [P.BF16, P.F32, P.F16])
@pytest.mark.parametrize("heads,groups,dim,n", [(4, 2, 64, 128), (6, 3, 33, 20)])
def test_step_without_a_list_of_slots(ctx, dt, heads, groups, dim, n):
    """row r is slot r: three calls as with the list 0, 1, ..., to the bit, and the slots behind the rows stay"""
    rng = np.random.default_rng(heads)
    rows, slots, taps, inner = 3, 5, 4, heads * dim
    ch = inner + 2 * groups * n
    w, cbias = rng.standard_normal((ch, taps)).astype(np.float32), rng.standard_normal(ch).astype(np.float32)
    conv0, st0 = P.to_kept(rng.standard_normal((slots, taps - 1, ch)), dt), rng.standard_normal((slots, heads, dim, n)).astype(np.float32)
    f32 = [ctx.upload(u) for u in (w, cbias, -(1 + 15 * rng.random(heads)).astype(np.float32), rng.standard_normal(heads).astype(np.float32), (rng.standard_normal(heads) - 3).astype(np.float32))]
    listed = ctx.upload(np.arange(rows, dtype=np.uint32))
    tokens = [[_Rows(ctx, rng.standard_normal((rows, u)), dt) for u in (ch, inner, heads)] for _ in range(3)]
    results = []
    for names in (listed.ptr, 0):
        conv_b, st_b, tick = ctx.upload(conv0), ctx.upload(st0), ctx.upload(np.zeros(rows * groups, np.uint32))
        outs = []
        for X, Z, D in tokens:
            out = _Rows(ctx, np.zeros((rows, inner)), dt)
            a = B.StateSpaceStepArgs(xbc=X.ptr, dt=D.ptr, z=Z.ptr, conv_weights=f32[0].ptr, conv_bias=f32[1].ptr, conv_state=conv_b.ptr, a=f32[2].ptr, d=f32[3].ptr, dt_bias=f32[4].ptr,
                                     state=st_b.ptr, out=out.ptr, slots=names, tickets=tick.ptr, rows=rows, slot_count=slots, heads=heads, groups=groups, head_dim=dim, state_size=n, taps=taps,
                                     xbc_stride=X.stride, dt_stride=D.stride, z_stride=Z.stride, out_stride=out.stride, dt_min=0.0, dt_max=float("inf"), dt_softplus=1, activation=B.ACT_SILU,
                                     data_type=dt)
            with ctx.command_buffer("step") as cmd:
                cmd.encode("uzu_state_space_step_encode", C.byref(a))
            outs.append(out.get()[0])
            assert not tick.numpy(np.uint32, (rows * groups,)).any()
        results.append((np.stack(outs), conv_b.numpy(_np(dt), conv0.shape), st_b.numpy(np.float32, st0.shape)))
    for with_list, without in zip(*results):
        assert np.array_equal(with_list, without)
    assert np.array_equal(results[1][1][rows:], conv0[rows:]) and np.array_equal(results[1][2][rows:], st0[rows:]) and not np.array_equal(results[1][2][:rows], st0[:rows])
