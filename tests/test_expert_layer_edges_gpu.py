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
        with pytest.raises(B.UzuError):
            lay.run(11, 4, P.F32, x=x, scratch=spoilt)
        assert not spoilt.numpy(np.uint8, (16 << 20,))[:16384].any()
        for _ in range(3):
            assert np.array_equal(lay.run(11, 4, P.F32, x=x, scratch=spoilt)[1], clean)
