"""The state space mixer's entries against their definitions in float64: packed prompts, single tokens, a run of them together."""
import ctypes as C

import numpy as np
import pytest

from tests import state_space_plain as P
from uzu_b200 import binding as B

pytestmark = pytest.mark.gpu

SENTINEL = 0x5A      # bytes of what a call leaves alone


def _np(dt):
    return {P.BF16: np.uint16, P.F32: np.float32, P.F16: np.float16}[dt]


class _Rows:
    """rows of `width` elements, `stride` apart, `shift` elements into a buffer of their own"""

    def __init__(self, ctx, values, dt, stride=0, shift=0):
        rows, width = values.shape
        self.stride, self.shift, self.width, self.rows, self.dt = stride or width, shift, width, rows, dt
        flat = np.frombuffer(bytes([SENTINEL]) * ((rows * self.stride + shift + 8) * np.dtype(_np(dt)).itemsize), _np(dt)).copy()
        self.view(flat)[:, :width] = P.to_kept(values, dt)
        self.buf = ctx.upload(flat)
        self.ptr = self.buf.ptr + shift * flat.itemsize
        self.n = flat.size

    def view(self, flat):
        return flat[self.shift:self.shift + self.rows * self.stride].reshape(self.rows, self.stride)

    def raw(self):
        return self.view(self.buf.numpy(_np(self.dt), (self.n,)))

    def get(self):
        """float64 values, and whether everything beside the rows is as it was"""
        raw = self.raw()
        return P.of_kept(raw[:, :self.width], self.dt), raw


def _kept(values, dt):
    return P.of_kept(P.to_kept(values, dt), dt)


def _table(seqs):
    return (B.RowSequence * max(1, len(seqs)))(*[B.RowSequence(*s) for s in seqs])


def _check(got, ref, bound, dt, what):
    """within a rounding of the reference and `bound`"""
    assert np.isfinite(got).all(), what
    tol = P.HALF_STEP[dt] * (np.abs(ref) + bound) + P.TINY[dt] + bound
    worst = (np.abs(got - ref) / tol).max(initial=0)
    assert worst <= 1, (what, float(worst))


# ---- convolution ----------------------------------------------------------------------------------------------------------------------------------
def _conv(ctx, dt, channels, taps, seqs, rows, slots, act=True, stride=0, shift=0, bias=True, seed=0):
    rng = np.random.default_rng(seed)
    u, w = rng.standard_normal((rows, channels)), rng.standard_normal((channels, taps)).astype(np.float32)
    b = rng.standard_normal(channels).astype(np.float32) if bias else np.zeros(channels, np.float32)
    st = rng.standard_normal((slots, max(taps - 1, 1), channels))
    covered = np.zeros(rows, bool)
    for f, n, _, _ in seqs:
        covered[f:f + n] = True
    u[~covered] = np.nan                     # rows of no sequence are not read into any
    x = _Rows(ctx, u, dt, stride, shift)
    out = _Rows(ctx, np.zeros((rows, channels)), dt, stride, shift)
    before = out.raw().copy()
    sb = ctx.upload(P.to_kept(st, dt))
    wb, bb = ctx.upload(w), ctx.upload(b)
    t = _table(seqs)
    a = B.CausalConvArgs(input=x.ptr, output=out.ptr, weights=wb.ptr, bias=bb.ptr if bias else 0, state=sb.ptr if taps > 1 else 0, sequences=C.addressof(t), sequence_count=len(seqs), rows=rows,
                         slots=slots, channels=channels, taps=taps, input_stride=x.stride, output_stride=out.stride, activation=B.ACT_SILU if act else B.ACT_IDENTITY, data_type=dt)
    with ctx.command_buffer("conv") as cmd:
        cmd.encode("uzu_causal_conv_encode", C.byref(a))
    ref, state, mag = P.conv(_kept(u, dt), w.astype(np.float64), b.astype(np.float64), _kept(st, dt)[:, :taps - 1], seqs, act)
    got, raw = out.get()
    # taps + 1 additions in 32 bits; the gate: an exponential of a value of up to `mag` and a division, its slope below 1.1
    bound = 1.1 * (taps + 2) * 2.0 ** -24 * mag + (2.0 ** -21 + 2.0 ** -22 * mag) * np.abs(np.nan_to_num(ref))
    _check(got[covered], ref[covered], bound[covered], dt, "out")
    assert np.array_equal(raw[~covered], before[~covered]) and np.array_equal(raw[:, channels:], before[:, channels:])
    if taps > 1:
        assert np.array_equal(sb.numpy(_np(dt), (slots, taps - 1, channels)), P.to_kept(state, dt))


RAGGED = [(0, 9, 3, 0), (9, 1, 0, 1), (10, 0, 1, 0), (10, 130, 4, 0), (140, 2, 2, 0), (142, 3, 5, 1), (146, 70, 6, 0), (220, 0, 7, 1)]


@pytest.mark.parametrize("dt", [P.BF16, P.F32, P.F16])
@pytest.mark.parametrize("taps", [1, 2, 3, 4, 5, 8])
def test_conv_ragged(ctx, dt, taps):
    _conv(ctx, dt, 72, taps, RAGGED, 223, 9)


@pytest.mark.parametrize("channels,stride,shift", [(8, 0, 0), (1, 0, 0), (63, 0, 0), (64, 72, 8), (64, 65, 0), (64, 0, 1), (1032, 0, 0)])
@pytest.mark.parametrize("act", [True, False])
def test_conv_layouts(ctx, channels, stride, shift, act):
    _conv(ctx, P.BF16, channels, 4, [(0, 40, 1, 0), (40, 7, 0, 1)], 48, 2, act, stride, shift, bias=act)


def test_conv_many_sequences(ctx):
    """more than one launch takes"""
    seqs = [(3 * i, 1 + i % 3, i, i % 2) for i in range(300)]
    _conv(ctx, P.BF16, 16, 4, seqs, 900, 300)


def test_conv_empty(ctx):
    _conv(ctx, P.BF16, 16, 4, [], 5, 1)


def test_conv_long(ctx):
    _conv(ctx, P.BF16, 2048, 4, [(0, 3001, 0, 0), (3001, 1096, 1, 0)], 4097, 2)


# ---- scan ------------------------------------------------------------------------------------------------------------------------------------------
def _scan_inputs(rng, rows, heads, groups, dim, n, dt):
    x, z = rng.standard_normal((rows, heads * dim)), rng.standard_normal((rows, heads * dim))
    b, c = rng.standard_normal((rows, groups * n)), rng.standard_normal((rows, groups * n))
    d = rng.standard_normal((rows, heads))
    a = -(1 + 15 * rng.random(heads)).astype(np.float32)
    skip = (1 + 0.2 * rng.standard_normal(heads)).astype(np.float32)
    size = np.exp(np.log(1e-3) + rng.random(heads) * np.log(100.0))
    bias = (size + np.log(-np.expm1(-size))).astype(np.float32)
    return x, z, b, c, d, a, skip, bias


def _scan(ctx, dt, heads, groups, dim, n, seqs, rows, slots, gate=True, pad=0, seed=0, softplus=True, lo=0.0, hi=float("inf"), scratch=True, chunks=False, skip_d=True, scale_dt=1.0):
    rng = np.random.default_rng(seed)
    x, z, b, c, d, a, skip, bias = _scan_inputs(rng, rows, heads, groups, dim, n, dt)
    d = d * scale_dt
    if not softplus:
        d, bias = np.abs(d) * 0.05, np.zeros_like(bias)
    covered = np.zeros(rows, bool)
    for f, m, _, _ in seqs:
        covered[f:f + m] = True
    for v in (x, z, b, c, d):
        v[~covered] = np.nan
    st = rng.standard_normal((slots, heads, dim, n)).astype(np.float32)
    bufs = [_Rows(ctx, v, dt, v.shape[1] + pad if pad else 0) for v in (x, z, b, c, d)]
    xb, zb, bb, cb, db = bufs
    out = _Rows(ctx, np.zeros((rows, heads * dim)), dt, heads * dim + pad if pad else 0)
    before = out.raw().copy()
    f32 = [ctx.upload(v) for v in (a, skip, bias, st)]
    t = _table(seqs)
    args = B.StateSpaceScanArgs(x=xb.ptr, dt=db.ptr, b=bb.ptr, c=cb.ptr, z=zb.ptr if gate else 0, a=f32[0].ptr, d=f32[1].ptr if skip_d else 0, dt_bias=f32[2].ptr if softplus else 0,
                                state=f32[3].ptr, out=out.ptr, sequences=C.addressof(t), sequence_count=len(seqs), rows=rows, slots=slots, heads=heads, groups=groups, head_dim=dim, state_size=n,
                                x_stride=xb.stride, dt_stride=db.stride, b_stride=bb.stride, c_stride=cb.stride, z_stride=zb.stride, out_stride=out.stride, dt_min=lo, dt_max=hi,
                                dt_softplus=int(softplus), data_type=dt)
    if scratch:
        args.scratch_bytes = ctx.lib.uzu_state_space_scan_scratch_bytes(ctx.h, C.byref(args))
        sc = ctx.buffer(max(16, args.scratch_bytes), B.BUFFER_DEVICE)
        args.scratch = sc.ptr
    with ctx.command_buffer("scan") as cmd:
        cmd.encode("uzu_state_space_scan_encode", C.byref(args))
    k = lambda v, *s: np.nan_to_num(_kept(v, dt)).reshape(rows, *s)
    a64, s64 = a.astype(np.float64), (skip if skip_d else 0 * skip).astype(np.float64)
    step = P.steps(k(d, heads), bias.astype(np.float64), softplus, lo, hi)
    ref, state, mag, smag = P.scan(k(x, heads, dim), step, k(b, groups, n), k(c, groups, n), k(z, heads, dim) if gate else None, a64, s64, st.astype(np.float64), seqs)
    got, raw = out.get()
    longest = max([m for _, m, _, _ in seqs], default=0)
    # in 32 bits: two roundings a token of the state, a decay that is off by 3 steps of its own and |step a| of the step's four, n + 2 of a read-out
    unit = 2.0 ** -24 * (longest * (5 + 4 * float(np.abs(step * a64).max(initial=0))) + n + 8)
    # in chunks: scores and the state that is read out rounded to bf16, decayed inputs to two of them
    y_unit, s_unit = (unit + 2.0 ** -8, unit + 2.0 ** -16) if chunks else (unit, unit)
    bound = y_unit * mag
    if gate:
        zz = k(z, heads, dim)
        bound = bound * np.abs(P.silu(zz)) + (2.0 ** -21 + 2.0 ** -22 * np.abs(zz)) * np.abs(np.nan_to_num(ref))
    cov = covered
    _check(got.reshape(rows, heads, dim)[cov], ref[cov], bound[cov], dt, "out")
    assert np.array_equal(raw[~cov], before[~cov]) and np.array_equal(raw[:, heads * dim:], before[:, heads * dim:])
    _check(f32[3].numpy(np.float32, st.shape).astype(np.float64), state, s_unit * smag, P.F32, "state")
    named = {s for _, _, s, _ in seqs}
    for s in range(slots):
        if s not in named:
            assert np.array_equal(f32[3].numpy(np.float32, st.shape)[s], st[s])


@pytest.mark.parametrize("dt", [P.BF16, P.F32, P.F16])
@pytest.mark.parametrize("heads,groups,dim,n", [(4, 2, 16, 16), (2, 1, 33, 7), (3, 3, 1, 1), (2, 1, 40, 65), (2, 2, 70, 130), (1, 1, 256, 256)])
def test_scan_shapes(ctx, dt, heads, groups, dim, n):
    _scan(ctx, dt, heads, groups, dim, n, RAGGED, 223, 9)


@pytest.mark.parametrize("over", [dict(gate=False), dict(pad=3), dict(softplus=False), dict(lo=0.01, hi=0.02), dict(skip_d=False), dict(scratch=False), dict(scale_dt=30.0)])
def test_scan_forms(ctx, over):
    _scan(ctx, P.F32, 4, 1, 32, 32, RAGGED, 223, 9, **over)


@pytest.mark.parametrize("dt", [P.BF16, P.F32])
@pytest.mark.parametrize("rows,seqs", [(700, [(0, 700, 1, 0)]), (601, [(0, 300, 0, 1), (300, 301, 1, 0)]), (150, [(3, 140, 0, 0)])])
def test_scan_token_by_token_in_parts(ctx, rows, seqs, dt):
    _scan(ctx, dt, 2, 1, 40, 24, seqs, rows, 2)


def test_scan_many_sequences(ctx):
    _scan(ctx, P.F32, 2, 1, 8, 8, [(3 * i, 1 + i % 3, i, i % 2) for i in range(300)], 900, 300)


def test_scan_empty(ctx):
    _scan(ctx, P.F32, 2, 1, 8, 8, [], 4, 1)


# heads of whole chunks' shapes in bf16: on the tensor cores
CHUNKED = [(0, 1, 3, 0), (1, 127, 0, 1), (128, 128, 1, 0), (256, 129, 4, 0), (390, 300, 2, 0), (690, 0, 5, 1), (690, 0, 6, 0), (700, 64, 7, 1)]


@pytest.mark.parametrize("heads,groups,dim,n", [(2, 1, 64, 128), (2, 2, 64, 64), (2, 1, 128, 64), (2, 1, 128, 128), (1, 1, 192, 128)])
@pytest.mark.parametrize("over", [dict(), dict(gate=False, pad=8), dict(scale_dt=30.0), dict(skip_d=False, lo=0.5, hi=20.0)])
def test_scan_chunks(ctx, heads, groups, dim, n, over):
    _scan(ctx, P.BF16, heads, groups, dim, n, CHUNKED, 770, 9, chunks=True, **over)


@pytest.mark.parametrize("scratch", [True, False])
@pytest.mark.parametrize("rows,seqs", [(2500, [(0, 2500, 1, 0)]), (2049, [(0, 1025, 0, 1), (1025, 1024, 1, 0)]), (1100, [(3, 1090, 0, 0)])])
def test_scan_in_parts(ctx, rows, seqs, scratch):
    """few heads: long sequences are cut, with a scratch"""
    _scan(ctx, P.BF16, 2, 1, 64, 128, seqs, rows, 2, chunks=True, scratch=scratch)


def test_scan_parts_and_whole_agree(ctx):
    """parts start from the sums of the parts before them: the state differs by roundings only (checked against float64 above); whole sequences give the same bits twice"""
    _scan(ctx, P.BF16, 4, 4, 64, 64, [(0, 1500, 0, 0), (1500, 40, 1, 1)], 1540, 3, chunks=True)


def test_scan_many_sequences_in_chunks(ctx):
    _scan(ctx, P.BF16, 1, 1, 64, 64, [(3 * i, 1 + i % 3, i, i % 2) for i in range(300)], 900, 300, chunks=True)


def test_scan_of_a_full_chip_repeats_itself(ctx):
    """every SM at work, memory busy: the same call gives the same bits (a stage that is given away too early shows here, as rows of another chunk)"""
    import torch
    g = torch.Generator(device="cuda").manual_seed(1)
    heads, dim, n, rows = 128, 64, 128, 4096
    inner, ch = heads * dim, heads * dim + 2 * n
    xbc = torch.randn(rows, ch, device="cuda", generator=g).to(torch.bfloat16)
    proj = torch.randn(rows, inner + heads, device="cuda", generator=g).to(torch.bfloat16)
    a, state0 = -1 - 15 * torch.rand(heads, device="cuda", generator=g), torch.randn(1, heads, dim, n, device="cuda", generator=g)
    bias, state, out = torch.full((heads,), -4.0, device="cuda"), torch.empty_like(state0), torch.empty(rows, inner, device="cuda", dtype=torch.bfloat16)
    t = _table([(0, rows, 0, 0)])
    e = 2
    args = B.StateSpaceScanArgs(x=xbc.data_ptr(), b=xbc.data_ptr() + e * inner, c=xbc.data_ptr() + e * (inner + n), z=proj.data_ptr(), dt=proj.data_ptr() + e * inner, a=a.data_ptr(),
                                d=bias.data_ptr(), dt_bias=bias.data_ptr(), state=state.data_ptr(), out=out.data_ptr(), sequences=C.addressof(t), sequence_count=1, rows=rows, slots=1, heads=heads,
                                groups=1, head_dim=dim, state_size=n, x_stride=ch, b_stride=ch, c_stride=ch, dt_stride=inner + heads, z_stride=inner + heads, out_stride=inner, dt_min=0.0, dt_max=1.0,
                                dt_softplus=1, data_type=P.BF16)
    first = None
    for _ in range(30):
        state.copy_(state0)
        torch.cuda.synchronize()
        with ctx.command_buffer("scan") as cmd:
            cmd.encode("uzu_state_space_scan_encode", C.byref(args))
        now = (out.clone(), state.clone())
        first = first or now
        assert torch.equal(first[0].view(torch.int16), now[0].view(torch.int16)) and torch.equal(first[1], now[1])


# ---- one token ------------------------------------------------------------------------------------------------------------------------------------
def _step_case(ctx, dt, heads, groups, dim, n, taps, slots, slot_count, gate=True, act=True, seed=0, calls=1, pad=0, graph=False):
    rng = np.random.default_rng(seed)
    rows, inner, ch = len(slots), heads * dim, heads * dim + 2 * groups * n
    order = list(range(rows)) if slots is None else slots
    w, cbias = rng.standard_normal((ch, taps)).astype(np.float32), rng.standard_normal(ch).astype(np.float32)
    conv0, st0 = rng.standard_normal((slot_count, max(1, taps - 1), ch)), rng.standard_normal((slot_count, heads, dim, n)).astype(np.float32)
    a = -(1 + 15 * rng.random(heads)).astype(np.float32)
    skip, bias = rng.standard_normal(heads).astype(np.float32), (rng.standard_normal(heads) - 3).astype(np.float32)
    conv_b, st_b, tick = ctx.upload(P.to_kept(conv0, dt)), ctx.upload(st0), ctx.upload(np.zeros(rows * groups, np.uint32))
    f32 = [ctx.upload(v) for v in (w, cbias, a, skip, bias)]
    sl = ctx.upload(np.array(slots, np.uint32))
    conv, st = _kept(conv0, dt)[:, :taps - 1], st0.astype(np.float64)
    seen, live = set(), []
    for r, s in enumerate(slots):
        if s < slot_count and s not in seen:
            seen.add(s)
            live.append(r)
    smag = np.abs(st)
    for call in range(calls):
        xbc, z, d = rng.standard_normal((rows, ch)), rng.standard_normal((rows, inner)), rng.standard_normal((rows, heads))
        X, Z, Dt = (_Rows(ctx, v, dt, v.shape[1] + pad if pad else 0) for v in (xbc, z, d))
        out = _Rows(ctx, np.zeros((rows, inner)), dt, inner + pad if pad else 0)
        before = out.raw().copy()
        args = B.StateSpaceStepArgs(xbc=X.ptr, dt=Dt.ptr, z=Z.ptr if gate else 0, conv_weights=f32[0].ptr, conv_bias=f32[1].ptr, conv_state=conv_b.ptr if taps > 1 else 0, a=f32[2].ptr, d=f32[3].ptr,
                                    dt_bias=f32[4].ptr, state=st_b.ptr, out=out.ptr, slots=sl.ptr, tickets=tick.ptr, rows=rows, slot_count=slot_count, heads=heads, groups=groups, head_dim=dim,
                                    state_size=n, taps=taps, xbc_stride=X.stride, dt_stride=Dt.stride, z_stride=Z.stride, out_stride=out.stride, dt_min=0.0, dt_max=float("inf"), dt_softplus=1,
                                    activation=B.ACT_SILU if act else B.ACT_IDENTITY, data_type=dt)
        with ctx.command_buffer("step") as cmd:
            cmd.encode("uzu_state_space_step_encode", C.byref(args))
        assert cmd.launches == 1
        got, raw = out.get()
        xk, zk, dk = (_kept(v, dt) for v in (xbc, z, d))
        for r in live:
            s = slots[r]
            seq = [(0, 1, 0, 0)]
            v, cs, mag = P.conv(xk[r:r + 1], w.astype(np.float64), cbias.astype(np.float64), conv[s:s + 1], seq, act)
            conv[s] = cs[0]
            off = 1.1 * (taps + 2) * 2.0 ** -24 * mag[0] + (2.0 ** -21 + 2.0 ** -22 * mag[0]) * np.abs(v[0])      # of the convolution
            x, b, c = v[0, :inner].reshape(1, heads, dim), v[0, inner:inner + groups * n].reshape(1, groups, n), v[0, inner + groups * n:].reshape(1, groups, n)
            step = P.steps(dk[r:r + 1], bias.astype(np.float64))
            prev = smag[s].copy()
            y, s1, ymag, _ = P.scan(x, step, b, c, zk[r:r + 1].reshape(1, heads, dim) if gate else None, a.astype(np.float64), skip.astype(np.float64), st[s:s + 1], seq)
            ox, ob, oc = off[:inner].reshape(heads, dim), np.repeat(off[inner:inner + groups * n].reshape(groups, n), heads // groups, 0), np.repeat(off[inner + groups * n:].reshape(groups, n), heads // groups, 0)
            bb, cc = np.repeat(np.abs(b[0]), heads // groups, 0), np.repeat(np.abs(c[0]), heads // groups, 0)
            add = step[0][:, None, None] * (ox[:, :, None] * (bb + ob)[:, None, :] + np.abs(x[0])[:, :, None] * ob[:, None, :])
            unit = 2.0 ** -24 * (8 + 8 * float(np.abs(step * a).max()))
            f = np.exp(step[0] * a)[:, None, None]
            mags = f * prev + np.abs(step[0][:, None, None] * x[0][:, :, None] * bb[:, None, :])
            s_bound = (unit * (call + 1) * mags + add * 1.01) + (call > 0) * 0.0
            err = np.abs(st_b.numpy(np.float32, st0.shape)[s].astype(np.float64) - s1[0])
            assert (err <= s_bound + (0 if call == 0 else carried[s] * f) + 2.0 ** -24 * np.abs(s1[0])).all(), ("state", r, call)
            carried = {} if call == 0 and r == live[0] else carried
            carried[s] = s_bound + (0 if call == 0 else carried[s] * f) + 2.0 ** -24 * np.abs(s1[0])
            y_bound = (carried[s] * cc[:, None, :] + (np.abs(s1[0]) + carried[s]) * oc[:, None, :]).sum(-1) + (n + 4) * 2.0 ** -24 * (ymag[0] + 1e-30) + np.abs(skip)[:, None] * ox
            ref = y[0]
            if gate:
                zz = zk[r].reshape(heads, dim)
                y_bound = y_bound * np.abs(P.silu(zz)) + (2.0 ** -21 + 2.0 ** -22 * np.abs(zz)) * np.abs(ref)
            _check(got[r].reshape(heads, dim), ref, y_bound, dt, ("out", r, call))
            st[s], smag[s] = s1[0], mags
        left = [r for r in range(rows) if r not in live]
        assert np.array_equal(raw[left], before[left]) and np.array_equal(raw[:, inner:], before[:, inner:])
        if taps > 1:
            assert np.array_equal(conv_b.numpy(_np(dt), (slot_count, taps - 1, ch)), P.to_kept(conv, dt))
        assert not tick.numpy(np.uint32, (rows * groups,)).any()
        for s in range(slot_count):
            if s not in seen:
                assert np.array_equal(st_b.numpy(np.float32, st0.shape)[s], st0[s])


@pytest.mark.parametrize("dt", [P.BF16, P.F32, P.F16])
@pytest.mark.parametrize("heads,groups,dim,n", [(4, 2, 64, 128), (2, 1, 33, 7), (3, 3, 1, 1), (2, 1, 128, 64), (2, 2, 70, 130), (8, 1, 256, 256), (4, 4, 16, 20), (2, 1, 65, 40)])
def test_step_shapes(ctx, dt, heads, groups, dim, n):
    _step_case(ctx, dt, heads, groups, dim, n, 4, [2, 0, 5], 6)


@pytest.mark.parametrize("taps", [1, 2, 3, 5, 8])
def test_step_taps(ctx, taps):
    _step_case(ctx, P.BF16, 4, 1, 32, 16, taps, [1, 0], 3, act=taps != 2, gate=taps != 3, calls=3)


def test_step_rows_left_out(ctx):
    """padded rows, and rows that name a slot again"""
    _step_case(ctx, P.BF16, 4, 2, 64, 64, 4, [3, 0xFFFFFFFF, 1, 3, 7, 1, 0], 7, calls=2, pad=5)


def test_step_many_rows(ctx):
    _step_case(ctx, P.BF16, 2, 1, 8, 8, 4, list(np.random.default_rng(1).permutation(400)[:391]), 400)


# ---- values that are not finite, calls together, captured calls ----------------------------------------------------------------------------------------
def _torch_scan(ctx, rows, heads, groups, dim, n, seed=0, slots=1, seqs=None, dt=P.BF16):
    """a scan over torch tensors: (run, tensors)"""
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    kept = {P.BF16: torch.bfloat16, P.F32: torch.float32}[dt]
    inner, ch = heads * dim, heads * dim + 2 * groups * n
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)
    t = dict(xbc=r(rows, ch).to(kept), z=r(rows, inner).to(kept), dt=r(rows, heads).to(kept), a=-1 - 15 * torch.rand(heads, device="cuda", generator=g), d=r(heads), bias=r(heads) - 3,
             state=r(slots, heads, dim, n), out=torch.zeros(rows, inner, device="cuda", dtype=kept))
    tab = _table(seqs or [(0, rows, 0, 0)])
    e = t["xbc"].element_size()
    args = B.StateSpaceScanArgs(x=t["xbc"].data_ptr(), b=t["xbc"].data_ptr() + e * inner, c=t["xbc"].data_ptr() + e * (inner + groups * n), z=t["z"].data_ptr(), dt=t["dt"].data_ptr(),
                                a=t["a"].data_ptr(), d=t["d"].data_ptr(), dt_bias=t["bias"].data_ptr(), state=t["state"].data_ptr(), out=t["out"].data_ptr(), sequences=C.addressof(tab),
                                sequence_count=len(seqs or [0]), rows=rows, slots=slots, heads=heads, groups=groups, head_dim=dim, state_size=n, x_stride=ch, b_stride=ch, c_stride=ch,
                                dt_stride=heads, z_stride=inner, out_stride=inner, dt_min=0.0, dt_max=float("inf"), dt_softplus=1, data_type=dt)
    args.scratch_bytes = ctx.lib.uzu_state_space_scan_scratch_bytes(ctx.h, C.byref(args))
    t["scratch"] = torch.empty(max(16, args.scratch_bytes), dtype=torch.uint8, device="cuda")
    args.scratch = t["scratch"].data_ptr()

    def run():
        torch.cuda.synchronize()
        with ctx.command_buffer("scan") as cmd:
            cmd.encode("uzu_state_space_scan_encode", C.byref(args))
    return run, t, (args, tab)


@pytest.mark.parametrize("dt,dim,n", [(P.BF16, 64, 128), (P.BF16, 128, 64), (P.F32, 20, 12)])
def test_scan_values_that_are_not_finite(ctx, dt, dim, n):
    """an x that is infinite or no number shows in its own column from its token on, a b in its head group's later tokens, a c and a z in their token: nothing else changes"""
    import torch
    rows, heads, groups = 300, 4, 2
    inner = heads * dim
    run, t, keep = _torch_scan(ctx, rows, heads, groups, dim, n, slots=1, dt=dt)
    state0 = t["state"].clone()
    run()
    clean = t["out"].clone()
    clean_state = t["state"].clone()
    assert bool(torch.isfinite(clean).all())
    for name, where, value in [("xbc", (140, dim + 5), float("inf")), ("xbc", (17, 3), float("nan")), ("xbc", (255, inner - 1), -float("inf")), ("xbc", (200, inner + 4), float("inf")),
                               ("xbc", (90, inner + groups * n + n + 2), float("nan")), ("z", (60, 2 * dim + 1), float("nan"))]:
        old = t[name][where].clone()
        t[name][where] = value
        t["state"].copy_(state0)
        run()
        t[name][where] = old
        row, col = where
        hit = torch.zeros(rows, inner, dtype=torch.bool, device="cuda")
        hit_state = torch.zeros_like(t["state"], dtype=torch.bool)
        must = hit.clone()
        if name == "z":
            hit[row, col] = must[row, col] = True
        elif col < inner:
            hit[row:, col] = must[row, col] = True
            hit_state[0, col // dim, col % dim] = True
        elif col < inner + groups * n:      # b of group 0, one column of the state
            hit[row:, :inner // groups] = True
            must[row, :inner // groups] = True
            hit_state[0, :heads // groups, :, col - inner] = True
        else:                               # c of group 1
            hit[row, inner // groups:] = must[row, inner // groups:] = True
        out, state = t["out"], t["state"]
        assert torch.equal(out[~hit], clean[~hit]), (name, where)
        assert not bool(torch.isfinite(out[must]).any()), (name, where)
        assert torch.equal(state[~hit_state], clean_state[~hit_state])


def _captured(ctx, encode):
    """what `encode(cmd)` enqueues, captured once on the context's stream: a function that replays it"""
    import torch
    stream = torch.cuda.ExternalStream(ctx.stream)
    graph = torch.cuda.CUDAGraph()
    h = C.c_void_p()
    B._check(ctx.lib.uzu_command_buffer_create(ctx.h, b"captured", C.byref(h)))
    B._check(ctx.lib.uzu_command_buffer_start_encoding(h))
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        graph.capture_begin(capture_error_mode="relaxed")
        encode(h)
        graph.capture_end()
    B._check(ctx.lib.uzu_command_buffer_end_encoding(h))
    B._check(ctx.lib.uzu_command_buffer_submit(h))
    B._check(ctx.lib.uzu_command_buffer_wait_until_completed(h))
    ctx.lib.uzu_command_buffer_destroy(h)

    def replay():
        with torch.cuda.stream(stream):
            graph.replay()
        torch.cuda.synchronize()
    return replay


class _Mixer:
    """a layer's state space mixer and its experts over torch tensors, as a host program runs them: prompt rows through convolution and scan, then tokens through the step, the
    mixer's output rows through the experts"""

    def __init__(self, ctx, seed=0, heads=8, groups=2, dim=64, n=128, taps=4, slots=6):
        import torch
        g = torch.Generator(device="cuda").manual_seed(seed)
        r = lambda *s: torch.randn(*s, device="cuda", generator=g)
        self.torch, self.ctx, self.g = torch, ctx, g
        self.heads, self.groups, self.dim, self.n, self.taps, self.slots = heads, groups, dim, n, taps, slots
        self.inner, self.ch = heads * dim, heads * dim + 2 * groups * n
        self.w, self.bias = r(self.ch, taps) / 2, 0.1 * r(self.ch)
        self.a, self.d, self.dtb = -1 - 15 * torch.rand(heads, device="cuda", generator=g), r(heads), r(heads) - 3
        self.conv_state = torch.zeros(slots, taps - 1, self.ch, device="cuda", dtype=torch.bfloat16)
        self.state = torch.zeros(slots, heads, dim, n, device="cuda")
        self.tickets = torch.zeros(64 * groups, dtype=torch.int32, device="cuda")
        self.width, self.ff, self.experts, self.top = self.inner, 64, 8, 2
        self.router = (r(8, self.inner) / self.inner ** 0.5).to(torch.bfloat16)
        self.up, self.down = (r(8, 128, self.inner) / self.inner ** 0.5).to(torch.bfloat16), (r(8, self.inner, 64) / 8).to(torch.bfloat16)
        self.kept = []

    def rows(self, count):
        return self.torch.randn(count, self.inner + self.ch + self.heads, device="cuda", generator=self.g).to(self.torch.bfloat16)

    def prompt(self, proj, seqs):
        """(encode, out): proj rows [z | xbc | dt]"""
        t, n = self.torch, proj.shape[0]
        xbc, out, tab = t.empty(n, self.ch, device="cuda", dtype=t.bfloat16), t.zeros(n, self.inner, device="cuda", dtype=t.bfloat16), _table(seqs)
        row, e = proj.shape[1], 2
        conv = B.CausalConvArgs(input=proj.data_ptr() + e * self.inner, output=xbc.data_ptr(), weights=self.w.data_ptr(), bias=self.bias.data_ptr(), state=self.conv_state.data_ptr(),
                                sequences=C.addressof(tab), sequence_count=len(seqs), rows=n, slots=self.slots, channels=self.ch, taps=self.taps, input_stride=row, output_stride=self.ch,
                                activation=B.ACT_SILU, data_type=B.DT_BF16)
        gn = self.groups * self.n
        scan = B.StateSpaceScanArgs(x=xbc.data_ptr(), b=xbc.data_ptr() + e * self.inner, c=xbc.data_ptr() + e * (self.inner + gn), z=proj.data_ptr(), dt=proj.data_ptr() + e * (self.inner + self.ch),
                                    a=self.a.data_ptr(), d=self.d.data_ptr(), dt_bias=self.dtb.data_ptr(), state=self.state.data_ptr(), out=out.data_ptr(), sequences=C.addressof(tab),
                                    sequence_count=len(seqs), rows=n, slots=self.slots, heads=self.heads, groups=self.groups, head_dim=self.dim, state_size=self.n, x_stride=self.ch, b_stride=self.ch,
                                    c_stride=self.ch, dt_stride=row, z_stride=row, out_stride=self.inner, dt_min=0.0, dt_max=float("inf"), dt_softplus=1, data_type=B.DT_BF16)
        scan.scratch_bytes = self.ctx.lib.uzu_state_space_scan_scratch_bytes(self.ctx.h, C.byref(scan))
        scratch = t.empty(max(16, scan.scratch_bytes), dtype=t.uint8, device="cuda")
        scan.scratch = scratch.data_ptr()
        self.kept += [proj, xbc, out, tab, conv, scan, scratch]

        def encode(h):
            self.ctx.lib.uzu_causal_conv_encode(h, C.byref(conv))
            self.ctx.lib.uzu_state_space_scan_encode(h, C.byref(scan))
        return encode, out

    def token(self, proj, slots):
        """(encode, mixer rows, experts' rows)"""
        t, n, e = self.torch, proj.shape[0], 2
        out, mixed = t.zeros(n, self.inner, device="cuda", dtype=t.bfloat16), t.zeros(n, self.inner, device="cuda", dtype=t.bfloat16)
        row = proj.shape[1]
        step = B.StateSpaceStepArgs(xbc=proj.data_ptr() + e * self.inner, dt=proj.data_ptr() + e * (self.inner + self.ch), z=proj.data_ptr(), conv_weights=self.w.data_ptr(), conv_bias=self.bias.data_ptr(),
                                    conv_state=self.conv_state.data_ptr(), a=self.a.data_ptr(), d=self.d.data_ptr(), dt_bias=self.dtb.data_ptr(), state=self.state.data_ptr(), out=out.data_ptr(),
                                    slots=slots.data_ptr(), tickets=self.tickets.data_ptr(), rows=n, slot_count=self.slots, heads=self.heads, groups=self.groups, head_dim=self.dim, state_size=self.n,
                                    taps=self.taps, xbc_stride=row, dt_stride=row, z_stride=row, out_stride=self.inner, dt_min=0.0, dt_max=float("inf"), dt_softplus=1, activation=B.ACT_SILU,
                                    data_type=B.DT_BF16)
        lay = B.ExpertLayerArgs(x=out.data_ptr(), out=mixed.data_ptr(), router=self.router.data_ptr(), up_gate=self.up.data_ptr(), down=self.down.data_ptr(), rows=n, width=self.width, ff=self.ff,
                                experts=self.experts, top=self.top, shared=0, x_stride=self.inner, out_stride=self.inner, score=0, renormalise=0, weight_scale=1.0, activation=B.ACT_SILU,
                                data_type=B.DT_BF16)
        lay.scratch_bytes = self.ctx.lib.uzu_expert_layer_scratch_bytes(C.byref(lay))
        scratch = t.zeros(lay.scratch_bytes, dtype=t.uint8, device="cuda")
        lay.scratch = scratch.data_ptr()
        self.kept += [proj, out, mixed, step, lay, scratch, slots]

        def encode(h):
            self.ctx.lib.uzu_state_space_step_encode(h, C.byref(step))
            self.ctx.lib.uzu_expert_layer_encode(h, C.byref(lay))
        return encode, out, mixed

    def run(self, *encodes):
        self.torch.cuda.synchronize()
        with self.ctx.command_buffer("mixer") as cmd:
            for f in encodes:
                f(cmd.h)


def test_prompt_then_tokens(ctx):
    """three prompts in one pass, then five tokens of each: as if the whole had been one prompt each; the experts read the mixer's rows in the same buffer"""
    import torch
    whole, parted = _Mixer(ctx, seed=3), _Mixer(ctx, seed=3)
    lengths = [150, 1, 260]
    tokens = 5
    rows = [whole.rows(n + tokens) for n in lengths]
    ends = np.cumsum([n + tokens for n in lengths])
    enc, ref = whole.prompt(torch.cat(rows), [(int(e) - n - tokens, n + tokens, 2 * i, 1) for i, (n, e) in enumerate(zip(lengths, ends))])
    whole.run(enc)
    starts = np.cumsum([0] + lengths)
    enc, out = parted.prompt(torch.cat([r[:n] for r, n in zip(rows, lengths)]), [(int(s), n, 2 * i, 1) for i, (n, s) in enumerate(zip(lengths, starts))])
    steps = [parted.token(torch.stack([r[n + k] for r, n in zip(rows, lengths)]), torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda")) for k in range(tokens)]
    parted.run(enc, *[s[0] for s in steps])
    for i, (n, e) in enumerate(zip(lengths, ends)):
        mine = ref[int(e) - n - tokens:int(e)].float()
        assert torch.equal(out[int(starts[i]):int(starts[i]) + n].float(), mine[:n])
        for k in range(tokens):
            got = steps[k][1][i].float()
            # the prompt's path rounds the convolution's rows, scores and the state that is read out to bf16, the step nothing: a few half steps of the row's size
            assert float((got - mine[n + k]).norm() / mine[n + k].norm()) <= 4 * 2.0 ** -8
    assert all(bool(torch.isfinite(s[2]).all()) and bool((s[2] != 0).any()) for s in steps)
    assert torch.equal(whole.conv_state[[0, 2, 4]].view(torch.int16), parted.conv_state[[0, 2, 4]].view(torch.int16))


def test_captured_calls_follow_the_device(ctx):
    """the four calls captured once and replayed: the same bits as run one by one, and a replay follows the slots that the device's list names then"""
    import torch
    eager, replayed = _Mixer(ctx, seed=5), _Mixer(ctx, seed=5)
    prompt, token = eager.rows(200), eager.rows(3)
    seqs = [(0, 130, 1, 1), (130, 70, 3, 0)]
    for m in (eager, replayed):
        m.state.normal_(generator=torch.Generator(device="cuda").manual_seed(1))
        m.conv_state.normal_(generator=torch.Generator(device="cuda").manual_seed(2))
    lists = [[1, 3, 0], [5, -1, 1], [2, 2, 4]]
    outs = []
    first = eager.prompt(prompt, seqs)
    outs_e = []
    for k, sl in enumerate(lists):
        s = eager.token(token, torch.tensor(sl, dtype=torch.int32, device="cuda"))
        eager.run(first[0], s[0])
        outs_e.append((first[1].clone(), s[1].clone(), s[2].clone()))
    slots = torch.tensor(lists[0], dtype=torch.int32, device="cuda")
    warm = _Mixer(ctx, seed=6)
    warm.run(warm.prompt(prompt, seqs)[0], warm.token(token, slots)[0])      # (a kernel's first launch sets its shared memory, which is not captured)
    p, s = replayed.prompt(prompt, seqs), replayed.token(token, slots)

    def both(h):
        p[0](h)
        s[0](h)
    replay = _captured(ctx, both)
    for k, sl in enumerate(lists):
        slots.copy_(torch.tensor(sl, dtype=torch.int32))
        s[1].zero_()
        torch.cuda.synchronize()
        replay()
        outs.append((p[1].clone(), s[1].clone(), s[2].clone()))
        for a, b in zip(outs_e[k], outs[k]):
            assert torch.equal(a.view(torch.int16), b.view(torch.int16)), k
    assert torch.equal(eager.state, replayed.state) and torch.equal(eager.conv_state.view(torch.int16), replayed.conv_state.view(torch.int16))


def test_two_contexts_at_once(ctx):
    """the same calls on the streams of two contexts at the same time, each with its own scratch and tickets"""
    import torch
    with B.Context(0) as other:
        alone = _Mixer(ctx, seed=8)
        prompt, token = alone.rows(700), alone.rows(4)
        sl = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device="cuda")
        p, s = alone.prompt(prompt, [(0, 700, 2, 1)]), alone.token(token, sl)
        alone.run(p[0], s[0], s[0], s[0])
        pairs = []
        for c in (ctx, other):
            m = _Mixer(c, seed=8)
            pairs.append((m, m.prompt(prompt, [(0, 700, 2, 1)]), m.token(token, sl)))
        torch.cuda.synchronize()
        cmds = [m.ctx.command_buffer("both") for m, _, _ in pairs]
        for cmd in cmds:
            cmd.__enter__()
        for _, p2, _ in pairs:
            p2[0](cmds[pairs.index(next(x for x in pairs if x[1] is p2))].h)
        for _ in range(3):
            for cmd, (_, _, s2) in zip(cmds, pairs):
                s2[0](cmd.h)
        for cmd in cmds:
            cmd.__exit__(None, None, None)
        for m, p2, s2 in pairs:
            assert torch.equal(p[1].view(torch.int16), p2[1].view(torch.int16)) and torch.equal(s[1].view(torch.int16), s2[1].view(torch.int16)) and torch.equal(s[2].view(torch.int16), s2[2].view(torch.int16))
            assert torch.equal(alone.state, m.state)


def test_refused_calls_leave_everything_alone(ctx):
    """an invalid call records the error, surfaced at the wait, and launches nothing"""
    run, t, (args, tab) = _torch_scan(ctx, 10, 2, 1, 64, 64)
    before = t["state"].clone()
    args.dt_min = -1.0
    with pytest.raises(B.UzuError, match="dt_min"):
        run()
    args.dt_min = 0.0
    args.heads = 3
    with pytest.raises(B.UzuError):
        run()
    import torch
    assert torch.equal(t["state"], before) and not bool(t["out"].any())
