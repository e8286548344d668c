"""Verification of drafted tokens at the ends of its range: temperatures next to 0, logits of any size, decisions that only sums of 64 bits can make."""
import ctypes as C

import numpy as np
import pytest

from tests import state_space_plain as P
from tests.quantized_cache_gpu import NONE, verify
from uzu_b200 import binding as B

pytestmark = pytest.mark.gpu

TYPES = [P.BF16, P.F32, P.F16]


def _drafts(rng, target, draft):
    """the target's favourite, the draft's, any: by turns"""
    n, k = target.shape[0], target.shape[1] - 1
    kinds = [target[:, :k].argmax(2), draft.argmax(2), rng.integers(0, target.shape[2], (n, k))]
    return np.choose(rng.choice(3, (n, k), p=[0.6, 0.3, 0.1]), kinds)


# ---- temperatures and logits at the ends ------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("temperature,draft_temperature", [(2.0 ** -60, 2.0 ** -60), (2.0 ** -50, 1.0), (1.0, 2.0 ** -55), (1e-16, 1e-16), (1e-15, 1e-12), (1e-12, 1e-6), (1e-6, 1e-15), (1e-3, 1e10), (1e38, 3e38)])
def test_any_temperature(ctx, dt, temperature, draft_temperature):
    """the largest logit's weight is 1, however cold it is"""
    rng = np.random.default_rng(17)
    n, k, vocab = 10, 4, 3001
    for lift in (0.0, 30.0):
        target = 8 * rng.standard_normal((n, k + 1, vocab)) + lift
        draft = target[:, :k] + 0.5 * rng.standard_normal((n, k, vocab))
        drafted, u = _drafts(rng, target, draft), rng.random((n, k + 1))
        assert verify(ctx, target, draft, drafted, u, temperature, draft_temperature, dt)[2] >= n - 2
        assert verify(ctx, target, None, drafted, u, temperature, 0.0, dt)[2] >= n - 2
        assert verify(ctx, target[:, :1], None, drafted[:, :0], u[:, :1], temperature, 0.0, dt)[2] >= n - 2


@pytest.mark.parametrize("dt,size", [(P.F32, 1e18), (P.BF16, 1e18), (P.F32, 1e30), (P.BF16, 1e30), (P.F32, 3e38), (P.BF16, 3e38), (P.F16, 6e4)])
@pytest.mark.parametrize("temperature", [1.0, 2.0 ** -60])
def test_any_logits(ctx, dt, size, temperature):
    rng = np.random.default_rng(18)
    n, k, vocab = 10, 3, 2000
    target = size * rng.uniform(-1, 1, (n, k + 1, vocab))
    draft = np.clip(target[:, :k] * rng.uniform(0.9, 1.0, (n, k, vocab)), -size, size)
    drafted, u = _drafts(rng, target, draft), rng.random((n, k + 1))
    for d in (draft, None):
        assert verify(ctx, target, d, drafted, u, temperature, temperature, dt)[2] >= n - 2


# ---- decisions that sums of 32 bits cannot make -----------------------------------------------------------------------------------------------------
def _shares(row, temperature):
    w = np.exp((row - row.max()) / temperature)
    return w / w.sum()


def _run(ctx, target, draft, drafted, u):
    """(accepted, tokens) of f32 logits at temperature 1"""
    n, k1, vocab = target.shape
    t, dr, un = ctx.upload(target.astype(np.float32)), ctx.upload(drafted.astype(np.uint32)), ctx.upload(u.astype(np.float32))
    d = ctx.upload(draft.astype(np.float32)) if draft is not None else None
    tokens, accepted = ctx.upload(np.zeros((n, k1), np.uint32)), ctx.upload(np.zeros(n, np.uint32))
    a = B.DraftVerifyArgs(target_logits=t.ptr, draft_logits=d.ptr if d else 0, drafted=dr.ptr, uniforms=un.ptr, tokens=tokens.ptr, accepted=accepted.ptr, sequences=n, drafts=k1 - 1, vocab=vocab, target_stride=vocab,
                          draft_stride=vocab, temperature=1.0, draft_temperature=1.0, data_type=P.F32)
    with ctx.command_buffer("verify") as cmd:
        cmd.encode("uzu_draft_verify_encode", C.byref(a))
    return accepted.numpy(np.uint32, (n,)), tokens.numpy(np.uint32, (n, k1))


# A weight of the device is within 2^-37 of itself beside roundings of exponents of up to 2^5, some 2^-46; a quotient of two and their sums within 2^-35: 3e-11
CLEAR = 1e-9


@pytest.mark.parametrize("with_draft", [True, False])
@pytest.mark.parametrize("shape", ["random", "rising"])
def test_uniform_numbers_next_to_the_share(ctx, with_draft, shape):
    """u one step or none beside p / q: kept or not as 64 bits have it, draft after draft"""
    rng = np.random.default_rng(19)
    n, k, vocab = (64, 4, 7001) if shape == "random" else (4, 2, 300001)
    target = 2 * rng.standard_normal((n, k + 1, vocab)) if shape == "random" else np.linspace(-20, 0, vocab) + 1e-3 * rng.standard_normal((n, k + 1, vocab))
    draft = target[:, :k] + rng.standard_normal((n, k, vocab))
    target, draft = target.astype(np.float32).astype(np.float64), draft.astype(np.float32).astype(np.float64)
    drafted, u = rng.integers(0, vocab, (n, k)), rng.random((n, k + 1)).astype(np.float32)
    ratio = np.zeros((n, k))
    for i in range(n):
        for j in range(k):
            p, q = _shares(target[i, j], 1.0), _shares(draft[i, j], 1.0) if with_draft else np.ones(vocab)
            x = int(np.argmax(q > 1.5 * p)) if with_draft else int(p.argmax())
            drafted[i, j], ratio[i, j] = x, p[x] / q[x]
            at = np.float32(ratio[i, j])
            u[i, j] = [at, np.nextafter(at, np.float32(0)), np.nextafter(at, np.float32(1))][rng.integers(0, 3)]
    clear = np.abs(u[:, :k] - ratio) > CLEAR * ratio
    keep = u[:, :k] < ratio
    accepted, tokens = _run(ctx, target, draft if with_draft else None, drafted, u)
    seen = 0
    for i in range(n):
        want = k if keep[i].all() else int(np.argmin(keep[i]))
        if not clear[i, :want + 1].all():
            continue
        seen += 1
        assert accepted[i] == want and np.array_equal(tokens[i, :want], drafted[i, :want]) and tokens[i, want] != NONE, (i, accepted[i], want)
    assert seen > n // 2


@pytest.mark.parametrize("vocab", [300, 5000, 40001])
@pytest.mark.parametrize("apart", [1e-4, 1e-6, 3e-7])
def test_a_draft_model_that_is_nearly_the_target(ctx, vocab, apart):
    """what is left of p - q is small, and is where p is above q"""
    rng = np.random.default_rng(20)
    n = 64
    target = (2 * rng.standard_normal((n, 2, vocab))).astype(np.float32)
    draft = (target[:, :1] + apart * rng.standard_normal((n, 1, vocab))).astype(np.float32)
    u = rng.random((n, 2)).astype(np.float32)
    accepted, tokens = _run(ctx, target, draft, np.full((n, 1), vocab), u)      # (no token: refused)
    assert (accepted == 0).all()
    seen = 0
    for i in range(n):
        p, q = _shares(target[i, 0].astype(np.float64), 1.0), _shares(draft[i, 0].astype(np.float64), 1.0)
        r = np.maximum(p - q, 0)
        sums = np.cumsum(r)
        aim = float(u[i, 1]) * sums[-1]
        # shares are off by roundings of exponents of up to 2^5, 2^-47 on both sides together; the series' own error is nearly the same for p and q, and goes with their difference
        if np.abs(sums - aim).min() <= 2.0 ** -46 + 2.0 ** -34 * sums[-1]:
            continue
        seen += 1
        assert tokens[i, 0] == np.flatnonzero(sums > aim)[0] and tokens[i, 1] == NONE, (i, tokens[i], np.flatnonzero(sums > aim)[0])
    assert seen > n // 2
