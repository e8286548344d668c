"""The experts' layer at the ends of its ranges."""
import numpy as np
import pytest

from tests import state_space_plain as P
from tests.test_expert_layer_gpu import _Layer
from uzu_b200 import binding as B

pytestmark = pytest.mark.gpu


def test_scratch_after_a_wait_that_ran_out(ctx):
    """A counter that starts below zero makes the first wait for all CTAs run out (a second) in those that look after it has come round, while the others go on: the call reports it,
    and the scratch is ready all the same for the next one, whose tiles of `down` several CTAs share."""
    lay = _Layer(ctx, 1024, 256, 16, 0, seed=21)
    scratch = ctx.upload(np.zeros(16 << 20, np.uint8))
    x, clean, *_ = lay.run(11, 4, P.F32, scratch=scratch)
    held = scratch.numpy(np.uint8, (16 << 20,)).copy()
    assert not held[:16384].any()
    for _ in range(2):
        held[:4] = np.array([2 ** 32 - 74], np.uint32).view(np.uint8)
        spoilt = ctx.upload(held)
        try:
            with pytest.raises(B.UzuError, match="code 0x80[1-4]"):
                lay.run(11, 4, P.F32, x=x, scratch=spoilt)
        finally:
            ctx.lib.uzu_debug_set_wait_error(ctx.h, 0)      # (others look for a code that was left)
        assert not spoilt.numpy(np.uint8, (16 << 20,))[:16384].any()
        for _ in range(3):
            assert np.array_equal(lay.run(11, 4, P.F32, x=x, scratch=spoilt)[1], clean)


@pytest.mark.parametrize("score", [0, 1, 2])
@pytest.mark.parametrize("experts", [9, 100, 300])
@pytest.mark.parametrize("low", [-200.0, -np.inf])
def test_logits_that_are_no_number_come_last(ctx, experts, score, low):
    """behind scores that come to 0, whatever their indices (for score 0 they count as -infinity); the chosen weights are numbers"""
    bias = np.full(experts, low, np.float32)
    bias[[0, 3, experts - 2]] = np.nan
    bias[[5, experts - 1]] = 1.0, 2.0
    lay = _Layer(ctx, 64, 32, experts, 0, seed=22)
    lay.bufs[0], lay.bufs[3] = ctx.upload(np.zeros((experts, 64), np.uint16)), ctx.upload(bias)
    if score == 0:
        bias[np.isnan(bias) & (low == -np.inf)] = low
    order = [experts - 1, 5] + [e for e in range(experts) if bias[e] == low] + ([] if (bias == low).sum() == experts - 2 else [0, 3, experts - 2])
    top = min(9, experts)
    _, got, ids, w, _ = lay.run(5, top, P.F32, score=score)
    assert np.array_equal(ids, np.tile(order[:top], (5, 1))) and np.isfinite(w).all() and np.isfinite(got).all()
    assert (w[:, 2:] == 0).all() and (w[:, :2] > 0).all()


def _bf16(v):
    return P.to_kept(np.asarray(v), P.BF16)


def test_f32_values_above_the_largest_of_bf16(ctx):
    """rows and hidden values that are finite in f32 but not as one bf16 part"""
    most = float(np.finfo(np.float32).max)
    lay = _Layer(ctx, 64, 32, 6, 1, seed=23)
    lay.host[0][:, 0] = 0
    lay.host[1][:, :, 0] = _bf16(2.0 ** -126)
    lay.bufs[0], lay.bufs[1] = ctx.upload(lay.host[0]), ctx.upload(lay.host[1])
    x = lay.rng.standard_normal((9, 64))
    x[:, 0] = [most, -most, 3.399e38, -3.3963e38, 3.3895e38, 1.0, 0.0, 3.0e38, most]
    lay.check(9, 2, P.F32, x=x)


def test_f32_hidden_values_above_the_largest_of_bf16(ctx):
    lay = _Layer(ctx, 64, 32, 3, 0, seed=24)
    lay.host[0][:] = 0
    lay.host[1][:] = 0
    lay.host[1][:, :, 0], lay.host[1][:, :, 1] = _bf16(2.0 ** 64 * (1 - 2.0 ** -8)), _bf16(2.0 ** 64 * 2.0 ** -8 * 0.75)
    lay.host[2][:] = _bf16(2.0 ** -126 * np.sign(P.of_kept(lay.host[2], P.BF16)))
    lay.bufs[:3] = [ctx.upload(v) for v in lay.host]
    x = np.zeros((4, 64))
    x[:, 0] = x[:, 1] = [1.0, 0.5, 0.999, 1.0]
    hidden = (2.0 ** 64 * (1 - 2.0 ** -10)) ** 2
    assert 2.0 ** 128 * (1 - 2.0 ** -9) < hidden < float(np.finfo(np.float32).max)      # (the least that rounds to an infinite bf16)
    lay.check(4, 1, P.F32, act=B.ACT_IDENTITY, x=x)


@pytest.mark.parametrize("rows", [1, 7, 16, 30, 64])
def test_bf16_rows_keep_products_of_16_bits(ctx, rows):
    """hidden values that are products of two 8-bit numbers reach `down` whole: differences of them, exact in 32 bits, are the results to the bit"""
    width, ff = 64, 32
    lay = _Layer(ctx, width, ff, 8, 0, seed=25)
    lay.host[0][:] = 0
    lay.host[1][:] = _bf16(1 + lay.rng.integers(0, 128, lay.host[1].shape) / 128)
    down = np.zeros((8, width, ff))
    d = np.arange(width)
    down[:, d, d % ff], down[:, d, (d + 1 + d // ff) % ff] = 1.0, -1.0
    lay.host[2][:] = _bf16(down)
    lay.bufs[:3] = [ctx.upload(v) for v in lay.host]
    x = np.eye(64)[:rows]
    _, got, ids, w, _ = lay.run(rows, 1, P.BF16, act=B.ACT_IDENTITY, x=x)
    assert (w == 1).all()
    y = np.stack([P.of_kept(lay.host[1][ids[r, 0]], P.BF16)[:, r] for r in range(rows)])
    hidden = y[:, :ff] * y[:, ff:]
    ref = hidden[:, d % ff] - hidden[:, (d + 1 + d // ff) % ff]
    assert np.array_equal(got, P.to_kept(ref, P.BF16))


@pytest.mark.parametrize("dt", [P.F32, P.BF16])
@pytest.mark.parametrize("experts,spread", [(512, True), (512, False), (16, False)])
def test_the_longest_lists(ctx, dt, experts, spread):
    """64 rows, 16 chosen and 16 shared: every expert by some rows and the shared ones by all, or the same few experts by all rows"""
    lay = _Layer(ctx, 64, 24, experts, 16, seed=26)
    if spread:      # row r reads its choices from its column
        router = np.full((experts, 64), -8.0)
        r, j = np.arange(64)[:, None], np.arange(16)[None, :]
        router[(8 * r + 5 * j) % experts, np.broadcast_to(r, (64, 16))] = 8 - j / 4
        lay.host[0][:], x = _bf16(router), np.eye(64)
        lay.bias[:] = 0
    else:
        x = 0.01 * lay.rng.standard_normal((64, 64))
        lay.bias[:] = 0
        lay.bias[np.arange(16) * (experts // 16)] = 10 + np.arange(16)
    lay.bufs[0], lay.bufs[3] = ctx.upload(lay.host[0]), ctx.upload(lay.bias)
    lay.check(64, 16, dt, x=x)
    ids = lay.run(64, 16, dt, x=x)[2]
    assert len(np.unique(ids)) == (experts if spread else 16)
