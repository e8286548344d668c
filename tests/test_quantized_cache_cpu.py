"""What the 8-bit cache's and the draft verification's entries refuse, without a device (the _validate calls make the checks of the _encode ones), and the codes of their plain form."""
import ctypes as C
import math

import numpy as np
import pytest

from tests import quantized_cache_plain as P
from uzu_b200 import binding as B

M = 1 << 20


def _cache(**over):
    a = dict(key_codes=16 * M, value_codes=32 * M, key_scales=48 * M, value_scales=49 * M, key_weights=50 * M, blocks=8, kv_heads=2, block_tokens=32, head_dim=64, code_type=B.CACHE_CODE_I8)
    return B.QuantizedCache(**{**a, **over})


def _sequences(**over):
    a = dict(tables=60 * M, lengths=61 * M, row_offsets=62 * M, count=3, table_stride=4, rows=9, max_rows=5, max_length=128)
    return B.CacheSequences(**{**a, **over})


def _make(kind, **over):
    cache, seqs = _cache(**over.pop("cache", {})), _sequences(**over.pop("sequences", {}))
    rows = dict(keys=70 * M, values=71 * M, key_stride=128, value_stride=128, data_type=B.DT_BF16)
    a = {"append": lambda: B.QuantizedCacheAppendArgs(cache=cache, sequences=seqs, new_lengths=72 * M, **rows),
         "read": lambda: B.QuantizedCacheReadArgs(cache=cache, sequences=seqs, **rows),
         "attention": lambda: B.QuantizedCacheAttentionArgs(cache=cache, sequences=seqs, query=70 * M, out=71 * M, sinks=0, scratch=80 * M, scratch_bytes=1 << 16, heads=4, query_row_stride=256,
                                                            query_head_stride=64, out_stride=256, scale=0.125, data_type=B.DT_BF16),
         "evict": lambda: B.QuantizedCacheEvictArgs(cache=cache, sequences=seqs, new_lengths=72 * M, indices=73 * M, scratch=80 * M, scratch_bytes=1 << 16, budget=40, keep_first=4, keep_last=8)}[kind]()
    for k, v in over.items():
        setattr(a, k, v)
    return a


def _verify(**over):
    a = B.DraftVerifyArgs(target_logits=16 * M, draft_logits=17 * M, drafted=18 * M, draft_counts=0, uniforms=19 * M, tokens=20 * M, accepted=21 * M, sequences=2, drafts=3, vocab=1000,
                          target_stride=1000, draft_stride=1000, temperature=1.0, draft_temperature=1.0, data_type=B.DT_BF16)
    for k, v in over.items():
        setattr(a, k, v)
    return a


KINDS = ["append", "read", "attention", "evict"]


def _status(lib, kind, a):
    return getattr(lib, f"uzu_{kind}_validate" if kind == "draft_verify" else f"uzu_quantized_cache_{kind}_validate")(C.byref(a))


def _refused(lib, kind, a, part):
    assert _status(lib, kind, a) == 2 and part in lib.uzu_last_error().decode(), lib.uzu_last_error()


@pytest.mark.parametrize("kind", KINDS)
def test_taken(lib, kind):
    assert _status(lib, kind, _make(kind)) == 0, lib.uzu_last_error()
    assert _status(lib, kind, _make(kind, sequences=dict(count=0, tables=0, lengths=0, row_offsets=0))) == 0
    assert getattr(lib, f"uzu_quantized_cache_{kind}_validate")(None) == 2


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("over,part", [
    (dict(code_type=2), "code_type"), (dict(block_tokens=8), "block_tokens"), (dict(block_tokens=48), "block_tokens"), (dict(block_tokens=128), "block_tokens"), (dict(head_dim=0), "head_dim"),
    (dict(head_dim=72), "head_dim"), (dict(head_dim=272), "head_dim"), (dict(kv_heads=0), "heads"), (dict(blocks=0), "blocks"), (dict(key_codes=0), "null"), (dict(value_scales=0), "null"),
    (dict(value_codes=32 * M + 8), "aligned"), (dict(key_scales=48 * M + 2), "aligned"), (dict(key_weights=50 * M + 1), "aligned")])
def test_cache_refused(lib, kind, over, part):
    _refused(lib, kind, _make(kind, cache=over), part)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("over,part", [
    (dict(tables=0), "null"), (dict(lengths=0), "null"), (dict(lengths=61 * M + 2), "aligned"), (dict(table_stride=0), "at least 1"), (dict(max_length=0), "at least 1"), (dict(max_length=1 << 31), "below 2^31"),
    (dict(count=65536), "65535")])
def test_sequences_refused(lib, kind, over, part):
    _refused(lib, kind, _make(kind, sequences=over), part)


@pytest.mark.parametrize("kind", ["append", "read"])
@pytest.mark.parametrize("over,part", [
    (dict(data_type=3), "data_type"), (dict(key_stride=127), "shorter"), (dict(value_stride=1), "shorter"), (dict(keys=70 * M + 1), "aligned"), (dict(values=32 * M + 64), "overlap"),
    (dict(keys=50 * M), "overlap"), (dict(sequences=dict(row_offsets=0)), "null"), (dict(sequences=dict(rows=1 << 31)), "below 2^31")])
def test_rows_refused(lib, kind, over, part):
    _refused(lib, kind, _make(kind, **over), part)


@pytest.mark.parametrize("over,part", [(dict(keys=0), "null"), (dict(new_lengths=61 * M), "new_lengths"), (dict(new_lengths=72 * M + 2), "aligned"), (dict(new_lengths=70 * M + 128), "new_lengths"),
                                       (dict(cache=dict(value_codes=16 * M + 16)), "overlaps itself"), (dict(cache=dict(key_scales=61 * M)), "which sequences")])
def test_append_refused(lib, over, part):
    _refused(lib, "append", _make("append", **over), part)


def test_append_without_lengths_out(lib):
    assert _status(lib, "append", _make("append", new_lengths=0)) == 0


@pytest.mark.parametrize("over,part", [(dict(values=70 * M + 64), "overlap"), (dict(values=61 * M), "which sequences")])
def test_read_refused(lib, over, part):
    _refused(lib, "read", _make("read", **over), part)


def test_read_of_one_kind(lib):
    assert _status(lib, "read", _make("read", keys=0)) == 0 and _status(lib, "read", _make("read", values=0, keys=0)) == 0
    # keys and values as slices of the same wide rows
    assert _status(lib, "read", _make("read", values=70 * M + 256, key_stride=256, value_stride=256)) == 0
    _refused(lib, "read", _make("read", values=70 * M + 254, key_stride=256, value_stride=256), "overlap")


@pytest.mark.parametrize("over,part", [
    (dict(data_type=3), "data_type"), (dict(heads=3), "heads"), (dict(heads=0), "heads"), (dict(scale=math.nan), "scale"), (dict(scale=math.inf), "scale"), (dict(softcap=-1.0), "softcap"),
    (dict(softcap=math.inf), "softcap"), (dict(out_stride=255), "shorter"), (dict(weight_rows=1, cache=dict(key_weights=0)), "key_weights"), (dict(query=0), "null"), (dict(out=0), "null"),
    (dict(scratch=0), "null"), (dict(scratch=80 * M + 16), "scratch"), (dict(out=70 * M), "overlap"), (dict(out=70 * M + 510), "overlap"), (dict(out=16 * M), "overlap"), (dict(query=50 * M), "overlap"),
    (dict(scratch=71 * M), "overlap"), (dict(scratch=60 * M), "overlap"), (dict(out=62 * M), "overlap"), (dict(query=70 * M + 1), "aligned"), (dict(sinks=90 * M + 2), "aligned"), (dict(sinks=71 * M), "overlap"),
    (dict(heads=65536 * 2), "heads"), (dict(sequences=dict(rows=(1 << 31) - 1, max_rows=(1 << 31) - 1)), "too many rows")])
def test_attention_refused(lib, over, part):
    _refused(lib, "attention", _make("attention", **over), part)


def test_attention_slices_of_one_row(lib):
    assert _status(lib, "attention", _make("attention", out=70 * M + 512, query_row_stride=512, out_stride=512)) == 0
    # head-major queries
    assert _status(lib, "attention", _make("attention", query_row_stride=64, query_head_stride=64 * 9)) == 0


@pytest.mark.parametrize("over,part", [
    (dict(cache=dict(key_weights=0)), "key_weights"), (dict(budget=0), "budget"), (dict(budget=1 << 31), "budget"), (dict(budget=11), "more than budget"), (dict(keep_first=0xFFFFFFFF, keep_last=2), "more than budget"),
    (dict(new_lengths=0), "null"), (dict(scratch=0), "null"), (dict(scratch=80 * M + 8), "scratch"), (dict(new_lengths=61 * M), "overlaps"), (dict(indices=72 * M), "overlap"), (dict(indices=80 * M), "overlap"),
    (dict(indices=32 * M), "overlaps"), (dict(indices=73 * M + 1), "aligned")])
def test_evict_refused(lib, over, part):
    _refused(lib, "evict", _make("evict", **over), part)


def test_evict_taken(lib):
    assert _status(lib, "evict", _make("evict", indices=0, sequences=dict(row_offsets=0, rows=0, max_rows=0))) == 0
    assert _status(lib, "evict", _make("evict", budget=12)) == 0


@pytest.mark.parametrize("over,part", [
    (dict(data_type=3), "data_type"), (dict(drafts=17), "16 drafts"), (dict(vocab=0), "vocab"), (dict(vocab=1 << 31), "vocab"), (dict(target_stride=999), "shorter"), (dict(draft_stride=999), "shorter"),
    (dict(temperature=-1.0), "temperature"), (dict(temperature=math.nan), "temperature"), (dict(temperature=math.inf), "temperature"), (dict(temperature=1e-30), "temperature"),
    (dict(draft_temperature=0.0), "draft_temperature"), (dict(draft_temperature=math.nan), "draft_temperature"), (dict(target_logits=0), "null"), (dict(drafted=0), "null"), (dict(uniforms=0), "null"),
    (dict(tokens=0), "null"), (dict(accepted=0), "null"), (dict(target_logits=16 * M + 1), "aligned"), (dict(tokens=20 * M + 2), "aligned"), (dict(accepted=20 * M + 4), "overlap"), (dict(tokens=18 * M), "overlaps"),
    (dict(accepted=19 * M), "overlaps"), (dict(sequences=(1 << 24) + 1), "sequences")])
def test_verify_refused(lib, over, part):
    _refused(lib, "draft_verify", _verify(**over), part)


def test_verify_taken(lib):
    for over in (dict(), dict(draft_logits=0, draft_stride=0, draft_temperature=0.0), dict(temperature=0.0, uniforms=0, draft_temperature=0.0), dict(drafts=0, drafted=0, draft_logits=0), dict(sequences=0, tokens=0)):
        assert _status(lib, "draft_verify", _verify(**over)) == 0, (over, lib.uzu_last_error())
    assert lib.uzu_draft_verify_validate(None) == 2


@pytest.mark.parametrize("code", [P.I8, P.E4M3])
def test_plain_codes(code):
    """every code stands for itself; halfway between two the even one is taken; a scale brings the largest magnitude just into the range"""
    values = P.stands_for(np.arange(256, dtype=np.uint8), code)
    values = np.unique(values[np.isfinite(values) & (np.abs(values) <= P.LARGEST[code])])
    assert np.array_equal(P.stands_for(P.coded(values, code), code), values)
    half = (values[1:] + values[:-1]) / 2
    for x, lo, hi in zip(half, values[:-1], values[1:]):
        got = P.coded(np.array([x]), code)
        assert got[0] % 2 == 0 and P.stands_for(got, code)[0] in (lo, hi)
    top = P.LARGEST[code]
    assert P.scale_of(np.array([top]), code) == 1 and P.scale_of(np.array([-np.nextafter(top, 1e9)]), code) == 2 and P.scale_of(np.array([top / 2, 1e-9]), code) == 0.5
    assert P.scale_of(np.zeros(3), code) == 0 and P.scale_of(np.array([1e-40]), code) == 2.0 ** -100 and math.isnan(P.scale_of(np.array([np.inf]), code)) and math.isnan(P.scale_of(np.array([2.0 ** 96]), code))
