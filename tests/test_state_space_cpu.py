"""What the state space mixer's and the experts' layer's entries refuse, without a device (the _validate calls make the checks of the _encode ones)."""
import ctypes as C

import pytest

from uzu_b200 import binding as B


def _table(*seqs):
    return (B.RowSequence * max(1, len(seqs)))(*[B.RowSequence(*s) for s in seqs])


def _conv(seqs=((0, 5, 0, 0), (5, 3, 2, 1)), **over):
    t = _table(*seqs)
    a = B.CausalConvArgs(input=1 << 20, output=2 << 20, weights=3 << 20, bias=0, state=4 << 20, sequences=C.addressof(t), sequence_count=len(seqs), rows=8, slots=3, channels=64,
                         taps=4, input_stride=64, output_stride=64, activation=B.ACT_SILU, data_type=B.DT_BF16)
    for k, v in over.items():
        setattr(a, k, v)
    a._keep = t
    return a


def _scan(seqs=((0, 5, 0, 0), (5, 3, 2, 1)), **over):
    t = _table(*seqs)
    a = B.StateSpaceScanArgs(x=1 << 20, dt=2 << 20, b=3 << 20, c=4 << 20, z=5 << 20, a=6 << 20, d=0, dt_bias=0, state=7 << 20, out=8 << 20, sequences=C.addressof(t), sequence_count=len(seqs),
                             rows=8, slots=3, heads=4, groups=2, head_dim=16, state_size=16, x_stride=64, dt_stride=4, b_stride=32, c_stride=32, z_stride=64, out_stride=64, dt_min=0.0,
                             dt_max=float("inf"), dt_softplus=1, data_type=B.DT_BF16)
    for k, v in over.items():
        setattr(a, k, v)
    a._keep = t
    return a


def _step(**over):
    a = B.StateSpaceStepArgs(xbc=1 << 20, dt=2 << 20, z=3 << 20, conv_weights=4 << 20, conv_bias=0, conv_state=5 << 20, a=6 << 20, d=0, dt_bias=0, state=7 << 20, out=8 << 20, slots=9 << 20,
                             tickets=10 << 20, rows=3, slot_count=2, heads=4, groups=2, head_dim=16, state_size=16, taps=4, xbc_stride=128, dt_stride=4, z_stride=64, out_stride=64, dt_min=0.0,
                             dt_max=1.0, dt_softplus=1, activation=B.ACT_SILU, data_type=B.DT_BF16)
    for k, v in over.items():
        setattr(a, k, v)
    return a


def _experts(lib, **over):
    a = B.ExpertLayerArgs(x=1 << 20, out=2 << 20, router=3 << 20, router_bias=0, up_gate=4 << 20, down=5 << 20, ids=0, weights=0, scratch=6 << 20, rows=3, width=64, ff=32, experts=8, top=2,
                          shared=1, x_stride=64, out_stride=64, score=0, renormalise=0, weight_scale=1.0, activation=B.ACT_SILU, data_type=B.DT_BF16)
    a.scratch_bytes = lib.uzu_expert_layer_scratch_bytes(C.byref(a))
    for k, v in over.items():
        setattr(a, k, v)
    return a


def _refused(lib, call, a, part):
    assert getattr(lib, call)(C.byref(a)) == 2 and part in lib.uzu_last_error().decode(), lib.uzu_last_error()


SEQUENCES = [
    (((0, 5, 0, 0), (4, 3, 2, 0)), "share a row"),
    (((5, 3, 2, 0), (0, 6, 0, 0)), "share a row"),
    (((0, 5, 1, 0), (5, 3, 1, 0)), "same slot"),
    (((0, 5, 3, 0),), "slot is not below"),
    (((0, 9, 0, 0),), "behind the last row"),
    (((0xFFFFFFFF, 2, 0, 0),), "behind the last row"),
]


@pytest.mark.parametrize("seqs,part", SEQUENCES)
def test_sequences_refused(lib, seqs, part):
    _refused(lib, "uzu_causal_conv_validate", _conv(seqs), part)
    _refused(lib, "uzu_state_space_scan_validate", _scan(seqs), part)


@pytest.mark.parametrize("seqs", [(), ((0, 0, 0, 0),), ((3, 0, 0, 0), (0, 8, 1, 1)), ((5, 3, 0, 0), (0, 5, 1, 0)), ((2, 1, 2, 0),)])
def test_sequences_taken(lib, seqs):
    assert lib.uzu_causal_conv_validate(C.byref(_conv(seqs))) == 0 and lib.uzu_state_space_scan_validate(C.byref(_scan(seqs))) == 0


def test_null_sequences(lib):
    _refused(lib, "uzu_causal_conv_validate", _conv(sequences=0), "null sequences")
    assert lib.uzu_causal_conv_validate(None) == 2 and lib.uzu_state_space_scan_validate(None) == 2 and lib.uzu_state_space_step_validate(None) == 2 and lib.uzu_expert_layer_validate(None) == 2


@pytest.mark.parametrize("over,part", [
    (dict(taps=0), "taps"), (dict(taps=9), "taps"), (dict(channels=0), "channels"), (dict(input_stride=63), "shorter"), (dict(output_stride=63), "shorter"), (dict(data_type=3), "data_type"),
    (dict(activation=B.ACT_GELU_EXACT), "activation"), (dict(input=0), "null"), (dict(output=0), "null"), (dict(weights=0), "null"), (dict(state=0), "null"), (dict(input=(1 << 20) + 1), "aligned"),
    (dict(weights=(3 << 20) + 2), "aligned"), (dict(output=1 << 20), "overlap"), (dict(output=(1 << 20) + 64), "overlap"), (dict(state=(1 << 20) + 8), "overlap"),
    (dict(output=(1 << 20) - 896), "overlap")])
def test_conv_refused(lib, over, part):
    _refused(lib, "uzu_causal_conv_validate", _conv(**over), part)


def test_conv_slices_of_one_row(lib):
    """input and output side by side in the same wide rows do not overlap; one element closer they do"""
    wide = dict(input=1 << 20, input_stride=200, output_stride=200)
    assert lib.uzu_causal_conv_validate(C.byref(_conv(output=(1 << 20) + 128, **wide))) == 0
    assert lib.uzu_causal_conv_validate(C.byref(_conv(output=(1 << 20) + 2 * 136, **wide))) == 0
    _refused(lib, "uzu_causal_conv_validate", _conv(output=(1 << 20) + 126, **wide), "overlap")
    _refused(lib, "uzu_causal_conv_validate", _conv(output=(1 << 20) + 2 * 137, **wide), "overlap")
    assert lib.uzu_causal_conv_validate(C.byref(_conv(output=(1 << 20) - 128, **wide))) == 0
    _refused(lib, "uzu_causal_conv_validate", _conv(output=(1 << 20) - 126, **wide), "overlap")


@pytest.mark.parametrize("over,part", [
    (dict(heads=0), "heads"), (dict(groups=3), "groups"), (dict(groups=0), "groups"), (dict(head_dim=0), "head_dim"), (dict(head_dim=257), "head_dim"), (dict(state_size=0), "state_size"),
    (dict(state_size=257), "state_size"), (dict(dt_min=-1.0), "dt_min"), (dict(dt_min=float("nan")), "dt_min"), (dict(dt_max=-1.0), "dt_m"), (dict(dt_max=float("nan")), "dt_m"),
    (dict(x_stride=63), "shorter"), (dict(dt_stride=3), "shorter"), (dict(b_stride=31), "shorter"), (dict(c_stride=31), "shorter"), (dict(z_stride=63), "shorter"), (dict(out_stride=63), "shorter"),
    (dict(x=0), "null"), (dict(dt=0), "null"), (dict(b=0), "null"), (dict(c=0), "null"), (dict(a=0), "null"), (dict(state=0), "null"), (dict(out=0), "null"), (dict(state=(7 << 20) + 2), "aligned"),
    (dict(z=(5 << 20) + 1), "aligned"), (dict(out=1 << 20), "overlap"), (dict(out=5 << 20), "overlap"), (dict(state=1 << 20), "overlap"), (dict(state=8 << 20), "overlap"), (dict(data_type=9), "data_type"),
    (dict(scratch=8), "scratch")])
def test_scan_refused(lib, over, part):
    _refused(lib, "uzu_state_space_scan_validate", _scan(**over), part)


@pytest.mark.parametrize("over,part", [
    (dict(taps=0), "taps"), (dict(taps=9), "taps"), (dict(rows=65536), "rows"), (dict(slots=0), "slots"), (dict(xbc_stride=127), "shorter"), (dict(dt_stride=3), "shorter"), (dict(z_stride=1), "shorter"),
    (dict(out_stride=63), "shorter"), (dict(tickets=0), "null"), (dict(conv_state=0), "null"), (dict(state=0), "null"), (dict(xbc=0), "null"), (dict(tickets=(10 << 20) + 2), "aligned"),
    (dict(out=1 << 20), "overlap"), (dict(state=1 << 20), "overlap"), (dict(conv_state=8 << 20), "overlap"), (dict(conv_state=7 << 20), "overlap"), (dict(activation=B.ACT_SOFTPLUS), "activation"),
    (dict(groups=3), "groups"), (dict(head_dim=300), "head_dim")])
def test_step_refused(lib, over, part):
    _refused(lib, "uzu_state_space_step_validate", _step(**over), part)


def test_step_taken(lib):
    assert lib.uzu_state_space_step_validate(C.byref(_step())) == 0
    assert lib.uzu_state_space_step_validate(C.byref(_step(rows=2, slots=0))) == 0
    assert lib.uzu_state_space_step_validate(C.byref(_step(taps=1, conv_state=0, tickets=0))) == 0
    assert lib.uzu_state_space_step_validate(C.byref(_step(rows=0, xbc=0))) == 0


@pytest.mark.parametrize("over,part", [
    (dict(rows=65), "64 rows"), (dict(width=60), "multiples of 8"), (dict(ff=36), "multiples of 8"), (dict(ff=0), "multiples of 8"), (dict(width=65544), "multiples of 8"), (dict(experts=0), "experts"),
    (dict(experts=513), "experts"), (dict(shared=17), "shared"), (dict(top=0), "top"), (dict(top=9), "top"), (dict(score=3), "score"), (dict(activation=5), "activation"), (dict(x_stride=63), "shorter"),
    (dict(out_stride=8), "shorter"), (dict(x=0), "null"), (dict(router=0), "null"), (dict(down=0), "null"), (dict(scratch=0), "null"), (dict(up_gate=(4 << 20) + 8), "aligned"), (dict(data_type=2), "data_type"),
    (dict(scratch=(6 << 20) + 16), "scratch"), (dict(scratch_bytes=16), "scratch"), (dict(out=(1 << 20) + 128), "overlap"), (dict(ids=(7 << 20) + 1), "aligned")])
def test_experts_refused(lib, over, part):
    _refused(lib, "uzu_expert_layer_validate", _experts(lib, **over), part)


def test_experts_taken(lib):
    assert lib.uzu_expert_layer_validate(C.byref(_experts(lib))) == 0 and lib.uzu_expert_layer_validate(C.byref(_experts(lib, rows=0, x=0))) == 0
    assert lib.uzu_expert_layer_scratch_bytes(C.byref(_experts(lib, width=60))) == 0


def test_experts_side_by_side(lib):
    """x and out as slices of the same wide rows: side by side they share nothing, a column less apart they do"""
    base = 1 << 20
    beside = dict(x=base, out=base + 64 * 2, x_stride=128, out_stride=128)
    assert lib.uzu_expert_layer_validate(C.byref(_experts(lib, **beside))) == 0
    assert lib.uzu_expert_layer_validate(C.byref(_experts(lib, **{**beside, "x": base + 64 * 2, "out": base}))) == 0
    _refused(lib, "uzu_expert_layer_validate", _experts(lib, **{**beside, "out": base + 63 * 2}), "overlap")
    _refused(lib, "uzu_expert_layer_validate", _experts(lib, **{**beside, "out_stride": 129}), "overlap")
