"""A whole layer of routed experts against its definition in float64."""
import ctypes as C
import math

import numpy as np
import pytest

from tests import state_space_plain as P
from uzu_b200 import binding as B

pytestmark = pytest.mark.gpu

ACTS = {B.ACT_SILU: P.silu, B.ACT_IDENTITY: lambda v: v,
        B.ACT_GELU_EXACT: lambda v: 0.5 * v * (1 + np.vectorize(math.erf)(v / math.sqrt(2))),
        B.ACT_GELU_APPROX: lambda v: 0.5 * v * (1 + np.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)))}


class _Layer:
    def __init__(self, ctx, width, ff, experts, shared, seed=0):
        rng = np.random.default_rng(seed)
        self.ctx, self.width, self.ff, self.experts, self.shared = ctx, width, ff, experts, shared
        k = lambda v: P.to_kept(v, P.BF16)
        self.host = [k(rng.standard_normal((experts, width)) / math.sqrt(width)), k(rng.standard_normal((experts + shared, 2 * ff, width)) / math.sqrt(width)),
                     k(rng.standard_normal((experts + shared, width, ff)) / math.sqrt(ff))]
        self.bias = (0.2 * rng.standard_normal(experts)).astype(np.float32)
        self.bufs = [ctx.upload(v) for v in self.host] + [ctx.upload(self.bias)]
        self.rng = rng

    def run(self, rows, top, dt, score=0, renormalise=0, scale=1.0, act=B.ACT_SILU, x=None, x_pad=0, out_pad=0, scratch=None, results=True):
        ctx, w = self.ctx, self.width
        x = self.rng.standard_normal((rows, w)) if x is None else x
        xk = np.zeros((rows, w + x_pad), P.to_kept(x, dt).dtype)
        xk[:, :w] = P.to_kept(x, dt)
        xb = ctx.upload(xk)
        out = ctx.upload(np.full((rows, w + out_pad), 77, xk.dtype))
        ids, wt = ctx.upload(np.zeros((rows, top), np.uint32)), ctx.upload(np.zeros((rows, top), np.float32))
        a = B.ExpertLayerArgs(x=xb.ptr, out=out.ptr, router=self.bufs[0].ptr, router_bias=self.bufs[3].ptr, up_gate=self.bufs[1].ptr, down=self.bufs[2].ptr, ids=ids.ptr if results else 0,
                              weights=wt.ptr if results else 0, rows=rows, width=w, ff=self.ff, experts=self.experts, top=top, shared=self.shared, x_stride=w + x_pad, out_stride=w + out_pad,
                              score=score, renormalise=renormalise, weight_scale=scale, activation=act, data_type=dt)
        a.scratch_bytes = ctx.lib.uzu_expert_layer_scratch_bytes(C.byref(a))
        sb = scratch or ctx.upload(np.zeros(a.scratch_bytes, np.uint8))
        a.scratch, a.scratch_bytes = sb.ptr, sb.nbytes
        with ctx.command_buffer("experts") as cmd:
            cmd.encode("uzu_expert_layer_encode", C.byref(a))
        got = out.numpy(xk.dtype, xk.shape[:1] + (w + out_pad,))
        assert np.array_equal(got[:, w:], np.full((rows, out_pad), 77, xk.dtype))
        return x, got[:, :w], ids.numpy(np.uint32, (rows, top)), wt.numpy(np.float32, (rows, top)), cmd

    def check(self, rows, top, dt, score=0, renormalise=0, scale=1.0, act=B.ACT_SILU, **kw):
        x, got, ids, weights, cmd = self.run(rows, top, dt, score, renormalise, scale, act, **kw)
        assert cmd.launches == 1
        r, u, d = (P.of_kept(v, P.BF16) for v in self.host)
        ref, rid, rw, mag, gap = P.experts(P.of_kept(P.to_kept(x, dt), dt), r, self.bias.astype(np.float64), u, d, top, self.shared, score, renormalise, scale, ACTS[act])
        assert gap > 1e-6, "the case has two scores that 32 bits do not tell apart"
        assert np.array_equal(ids, rid)
        assert np.abs(weights - rw).max() <= 2e-6 * np.abs(rw).max() + (self.width + 16) * 2.0 ** -24 * 4 * np.abs(rw).max()
        # products of bf16 parts in 32 bits: a rounding for each of the operands' 8 columns (24 of three parts) and the warps' sums; hidden values and rows of
        # f32 as three bf16 parts keep 24 bits, hidden values of bf16 rows 8; the gate's exponential
        part = 2.0 ** -24 * 3 * (self.width + self.ff) / 8 if dt == P.F32 else 2.0 ** -8
        unit = part + 2.0 ** -24 * ((self.width + self.ff) / 8 + 32) + 2.0 ** -20
        _check(P.of_kept(got, dt), ref, unit * mag, dt)


def _check(got, ref, bound, dt):
    assert np.isfinite(got).all()
    worst = (np.abs(got - ref) / (P.HALF_STEP[dt] * (np.abs(ref) + bound) + bound + 1e-30)).max()
    assert worst <= 1, float(worst)


@pytest.mark.parametrize("dt", [P.BF16, P.F32])
@pytest.mark.parametrize("rows", [1, 3, 8, 9, 16, 17, 33, 64])
def test_rows(ctx, dt, rows):
    _Layer(ctx, 256, 136, 16, 1, seed=rows).check(rows, 4, dt)


@pytest.mark.parametrize("width,ff,experts,top,shared", [(8, 8, 1, 1, 0), (64, 520, 3, 3, 2), (1032, 24, 40, 2, 0), (2048, 512, 8, 2, 0), (72, 1000, 512, 16, 16), (520, 8, 33, 16, 1)])
@pytest.mark.parametrize("dt", [P.BF16, P.F32])
def test_shapes(ctx, width, ff, experts, top, shared, dt):
    _Layer(ctx, width, ff, experts, shared, seed=width).check(5, top, dt, score=1)


@pytest.mark.parametrize("score", [0, 1, 2])
@pytest.mark.parametrize("renormalise,scale", [(0, 1.0), (1, 2.5)])
def test_scores(ctx, score, renormalise, scale):
    _Layer(ctx, 128, 64, 24, 1, seed=3).check(12, 5, P.F32, score, renormalise, scale)


@pytest.mark.parametrize("act", list(ACTS))
def test_activations(ctx, act):
    _Layer(ctx, 128, 64, 8, 0, seed=4).check(7, 2, P.F32, act=act)


def test_strides_and_no_results(ctx):
    lay = _Layer(ctx, 128, 64, 8, 0, seed=5)
    lay.check(6, 2, P.BF16, x_pad=3, out_pad=5)
    x, got, *_ = lay.run(6, 2, P.BF16)
    _, again, *_ = lay.run(6, 2, P.BF16, x=x, results=False, x_pad=1)
    assert np.array_equal(got, again)


def test_ties_go_to_the_lower_index(ctx):
    lay = _Layer(ctx, 64, 32, 40, 0, seed=6)
    lay.bufs[0] = ctx.upload(np.zeros((40, 64), np.uint16))
    lay.bufs[3] = ctx.upload(np.where(np.arange(40) % 3 == 0, 1.0, 0.0).astype(np.float32))
    for score in (0, 1, 2):
        _, _, ids, w, _ = lay.run(9, 16, P.BF16, score=score, renormalise=1)
        assert (ids == np.concatenate([np.arange(0, 40, 3), [1, 2]])).all() and np.allclose(w.sum(1), 1, atol=1e-6)


def test_one_expert_for_all(ctx):
    """every token on the same experts: one expert's tokens fill all tiles"""
    lay = _Layer(ctx, 128, 64, 8, 0, seed=7)
    lay.bias = np.array([0, 50, 0, 0, 0, 40, 0, 0], np.float32)
    lay.bufs[3] = ctx.upload(lay.bias)
    lay.check(64, 2, P.BF16)


def test_scratch_is_left_ready(ctx):
    """calls of other sizes one after the other in the same scratch; the same call gives the same bits"""
    a, b = _Layer(ctx, 1024, 256, 16, 0, seed=8), _Layer(ctx, 64, 40, 4, 1, seed=9)
    scratch = ctx.upload(np.zeros(16 << 20, np.uint8))
    x, first, *_ = a.run(11, 4, P.F32, scratch=scratch)
    for rows in (1, 64, 20):
        b.check(rows, 2, P.BF16, scratch=scratch)
        a.check(rows, 3, P.F32, scratch=scratch)
        assert np.array_equal(a.run(11, 4, P.F32, x=x, scratch=scratch)[1], first)


def test_values_that_are_not_finite_stay_in_their_row(ctx):
    lay = _Layer(ctx, 128, 64, 8, 1, seed=10)
    x = lay.rng.standard_normal((10, 128))
    _, clean, *_ = lay.run(10, 2, P.BF16, x=x)
    bad = x.copy()
    bad[3, 5], bad[7, 0] = np.inf, np.nan
    _, got, *_ = lay.run(10, 2, P.BF16, x=bad)
    keep = [r for r in range(10) if r not in (3, 7)]
    assert np.array_equal(got[keep], clean[keep]) and not np.isfinite(P.of_kept(got[[3, 7]], P.BF16)).all()


@pytest.mark.parametrize("score", [0, 1, 2])
@pytest.mark.parametrize("experts,top", [(8, 2), (8, 8), (64, 6), (300, 16)])
def test_choice_of_logits_that_are_not_finite(ctx, experts, top, score):
    """choices of such tokens are distinct experts, NaN last; the other tokens keep theirs (their sums' order may differ: it follows the choice of all)"""
    lay = _Layer(ctx, 128, 64, experts, 0, seed=11)
    x = lay.rng.standard_normal((9, 128))
    _, clean, ids0, w0, _ = lay.run(9, top, P.F32, score=score, x=x)
    r, u, d = (P.of_kept(v, P.BF16) for v in lay.host)
    _, _, _, mag, _ = P.experts(P.of_kept(P.to_kept(x, P.F32), P.F32), r, lay.bias.astype(np.float64), u, d, top, 0, score, 0, 1.0, P.silu)
    bad = x.copy()
    bad[2, 5], bad[4, :], bad[6, 1] = np.inf, np.nan, -np.inf
    _, got, ids, w, _ = lay.run(9, top, P.F32, score=score, x=bad)
    keep = [0, 1, 3, 5, 7, 8]
    assert np.array_equal(ids[keep], ids0[keep]) and np.array_equal(w[keep], w0[keep])
    # both sums are within the unit that `_Layer.check` derives, and their last rounding
    unit = 2.0 ** -24 * 3 * (128 + 64) / 8 + 2.0 ** -24 * ((128 + 64) / 8 + 32) + 2.0 ** -20
    assert (np.abs(got[keep] - clean[keep]) <= 2 * (unit * mag[keep] + P.HALF_STEP[P.F32] * np.abs(clean[keep]) + 1e-30)).all()
    assert ids.max() < experts and all(len(set(r)) == top for r in ids.tolist())
    assert np.array_equal(ids[4], np.arange(top)) and (score == 2 or np.isnan(w[4]).all())
    if score == 1:
        assert np.array_equal(ids[2], np.arange(top)) and np.isnan(w[2]).all()


@pytest.mark.parametrize("dt", [P.BF16, P.F32])
def test_slices_of_the_same_rows(ctx, dt):
    """out beside x in the same wide rows: the same bits as apart, and x stays"""
    lay, rows, w = _Layer(ctx, 128, 64, 8, 1, seed=12), 21, 128
    x, apart, *_ = lay.run(rows, 2, dt)
    wide = np.zeros((rows, 2 * w), P.to_kept(x, dt).dtype)
    wide[:, :w] = P.to_kept(x, dt)
    buf = ctx.upload(wide)
    a = B.ExpertLayerArgs(x=buf.ptr, out=buf.ptr + w * wide.itemsize, router=lay.bufs[0].ptr, router_bias=lay.bufs[3].ptr, up_gate=lay.bufs[1].ptr, down=lay.bufs[2].ptr, rows=rows, width=w, ff=64,
                          experts=8, top=2, shared=1, x_stride=2 * w, out_stride=2 * w, weight_scale=1.0, activation=B.ACT_SILU, data_type=dt)
    a.scratch_bytes = ctx.lib.uzu_expert_layer_scratch_bytes(C.byref(a))
    scratch = ctx.upload(np.zeros(a.scratch_bytes, np.uint8))
    a.scratch = scratch.ptr
    with ctx.command_buffer("experts") as cmd:
        cmd.encode("uzu_expert_layer_encode", C.byref(a))
    got = buf.numpy(wide.dtype, wide.shape)
    assert np.array_equal(got[:, :w], wide[:, :w]) and np.array_equal(got[:, w:], apart)
