"""Verification of drafted tokens at the ends of its range: temperatures next to 0, logits of any size."""
import numpy as np
import pytest

from tests import state_space_plain as P
from tests.quantized_cache_gpu import verify

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
