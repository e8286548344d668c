"""The 8-bit cache's entries against their definitions in float64: rows in and out, attention, weights, eviction, and a run of them together."""
import ctypes as C

import numpy as np
import pytest

from tests import quantized_cache_plain as Q
from tests import state_space_plain as P
from tests.quantized_cache_gpu import NONE, Served, verify
from uzu_b200 import binding as B

pytestmark = pytest.mark.gpu

ALL = 0xFFFFFFFF
CODES = [Q.I8, Q.E4M3]
TYPES = [P.BF16, P.F32, P.F16]


# ---- rows in and out ------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("block,heads,dim", [(16, 3, 80), (32, 2, 64), (64, 2, 256), (64, 1, 16)])
def test_append(ctx, code, dt, block, heads, dim):
    """new sequences, begun blocks, blocks that are full, sequences without rows; then single tokens, whose blocks keep or raise their scale; all read back"""
    s = Served(ctx, code, block, heads, dim, [0, 5, block, 2 * block - 1, 7], room=4 * block + 20)
    after = s.append([block + 3, 2 * block + 1, 1, 2, 0], dt)
    assert s.same()
    for n in range(4):
        s.set_lengths(after)
        after = s.append([1, 1, 0, 1, 1], dt)
        assert s.same()
    s.read([0] * 5, [int(n) for n in after], dt)
    s.read([3, 0, 1, 40, 5], [4, 0, 7, 3, 2], P.BF16)


@pytest.mark.parametrize("dt", TYPES)
def test_rows_off_alignment(ctx, dt):
    s = Served(ctx, Q.I8, 32, 2, 48, [3, 31])
    s.append([40, 9], dt, stride=103, shift=1)
    assert s.same()
    s.read([0, 2], [43, 30], dt, stride=101, shift=3)
    s.read([0, 2], [43, 30], dt, kinds=(True, False))
    s.read([0, 2], [43, 30], dt, kinds=(False, True))


@pytest.mark.parametrize("code", CODES)
def test_scales_that_grow(ctx, code):
    """token by token into one block, each a little or a lot larger than the ones before"""
    s = Served(ctx, code, 16, 2, 32, [0])
    for t in range(20):
        s.set_lengths([t])
        x = [s.rng.standard_normal((1, 64)) * 2.0 ** min(60, [0, 0, 1, 1, 2, 9, 9, 3, 30, 60][t // 2]) for _ in range(2)]
        s.append([1], P.F32, values=[np.concatenate([v, v]) for v in x], tail=1)
        assert s.same(), t


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dt", TYPES)
def test_values_at_the_ends(ctx, code, dt):
    """zeros, the smallest and the largest numbers, halves between codes, values that are not finite; a block's scale of NaN stays until the block is begun again"""
    s = Served(ctx, code, 16, 8, 16, [0, 4], room=64)
    x = np.zeros((2, 16 + 4, 8, 16))
    top = Q.LARGEST[code]
    x[:, :, 0] = 0.0
    x[:, :, 1] = 2.0 ** -140
    x[:, :, 2] = np.linspace(-top, top, 16) + 0.5
    x[:, :, 3] = 1e30 if dt != P.F16 else 6e4
    x[:, 3, 4] = np.inf
    x[:, 5, 5, 3] = np.nan
    x[:, :, 6] = top
    x[:, :, 7] = np.arange(16) + 0.5
    s.append([16, 2], dt, values=[v.reshape(20, 128) for v in x], tail=2)
    assert s.same() and np.isnan(s.plain.scales[0][s.table[0, 0], [4, 5]]).all()
    s.set_lengths([16, 6])
    s.append([3, 3], dt)
    assert s.same()
    s.set_lengths([0, 0])
    s.append([2, 17], dt)
    assert s.same() and np.isfinite(s.plain.scales[0][s.table[0, 0]]).all()


def test_huge_f32_rows(ctx):
    s = Served(ctx, Q.E4M3, 16, 2, 16, [0, 0])
    x = np.full((20, 32), 1.0)
    x[3, 5], x[12, 20] = 2.0 ** 95.9, -2.0 ** 96
    s.append([10, 8], P.F32, values=[x, x[::-1].copy()])
    assert s.same() and np.isnan(s.plain.scales[0]).any()


@pytest.mark.parametrize("code", CODES)
def test_blocks_that_are_none_and_lengths_behind_the_end(ctx, code):
    """rows for a block number that is none, and tokens behind max_length, are dropped"""
    s = Served(ctx, code, 16, 2, 32, [10, 70, 0, 500], room=90, missing=[(0, 1), (1, 5), (2, 0)])
    s.append([30, 40, 20, 3], P.BF16)
    assert s.same()
    s.append([30, 40, 20, 3], P.BF16, max_length=50, new_lengths=True)
    assert s.same()
    s.read([0, 60, 0, 90], [40, 50, 20, 30], P.F32)
    s.read([0, 60, 0, 90], [40, 50, 20, 30], P.F32, max_length=50)


# ---- attention ------------------------------------------------------------------------------------------------------------------------------------
SHAPES = [(16, 3, 6, 80), (32, 2, 8, 64), (64, 2, 8, 128), (64, 2, 4, 256), (32, 1, 16, 16), (16, 2, 2, 192), (32, 2, 14, 128)]


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("block,kv,heads,dim", SHAPES)
def test_single_tokens(ctx, code, dt, block, kv, heads, dim):
    """one row for each sequence, from an empty cache on, tokens behind the last are no numbers"""
    s = Served(ctx, code, block, kv, dim, [0, 1, 15, 16, 17, 100, 333], room=340, garbage=0x7F)
    s.set_lengths([0] * 7)
    s.append([1, 2, 16, 17, 18, 101, 334], P.F32)
    s.set_lengths([0, 1, 15, 16, 17, 100, 333])
    s.attend([1] * 7, heads, dt, weight_rows=ALL)
    s.attend([1, 0, 1, 0, 0, 1, 1], heads, dt)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("window,first,cap,sink", [(0, 0, 0.0, False), (40, 0, 0.0, True), (33, 5, 20.0, False), (1, 0, 0.0, True), (16, 20, 5.0, True), (7, 200, 0.0, False)])
def test_drafted_tokens_and_prompts(ctx, code, dt, window, first, cap, sink):
    s = Served(ctx, code, 32, 2, 64, [0, 3, 90, 200, 64, 41], room=300)
    rows = [5, 17, 1, 4, 0, 33]
    s.append(rows, P.F32)
    sinks = s.rng.standard_normal(8) * 2 if sink else None
    s.attend(rows, 8, dt, window=window, first=first, cap=cap, sinks=sinks, weight_rows=3)
    s.attend(rows, 8, dt, window=window, first=first, cap=cap, sinks=sinks, weight_rows=ALL, head_major=True)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rows", [[300], [129, 77], [128, 1, 64]])
@pytest.mark.parametrize("block,kv,heads,dim", [(64, 2, 8, 128), (16, 2, 4, 64), (32, 1, 2, 256), (32, 2, 6, 96), (16, 1, 8, 16), (32, 1, 3, 80)])
def test_prompts(ctx, dt, rows, block, kv, heads, dim):
    s = Served(ctx, Q.I8 if dim != 64 else Q.E4M3, block, kv, dim, [int(7 + 61 * i) for i in range(len(rows))], room=500)
    s.append(rows, P.F32)
    s.attend(rows, heads, dt, weight_rows=20)
    s.attend(rows, heads, dt, window=50, first=3, cap=10.0)


@pytest.mark.parametrize("dt", TYPES)
def test_rows_anywhere(ctx, dt):
    """rows off alignment, wider than their heads; more max_rows and max_length than there are, and less"""
    s = Served(ctx, Q.I8, 32, 2, 48, [37, 80], room=200)
    s.append([3, 2], dt)
    s.attend([3, 2], 4, dt, stride=197, shift=1, weight_rows=2)
    s.attend([3, 2], 4, dt, max_rows=40)
    s.attend([3, 2], 4, dt, max_length=64, weight_rows=2)
    got = s.attend([3, 2], 4, dt, max_rows=1, check=False)[0]
    assert (got[1] == 7).all() and (got[2] == 7).all() and (got[4] == 7).all() and (got[[0, 3]] != 7).any(1).all()


def test_no_rows_and_no_block(ctx):
    """a sequence whose blocks are all none sees nothing: zeros"""
    s = Served(ctx, Q.E4M3, 16, 1, 32, [0, 20, 30], room=40, missing=[(1, 0), (1, 1), (2, 0)])
    s.attend([0, 2, 3], 2, P.BF16, weight_rows=ALL)
    got, grown = s.attend([0, 2, 3], 2, P.BF16, check=False, sinks=[0.0, 1.0])
    assert (got[:2] == 0).all() and (got[2:5] != 0).any()
    s.attend([0, 0, 0], 2, P.BF16)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("rows", [[1, 1], [40, 33]])
def test_blocks_of_very_different_size(ctx, code, rows):
    """scales from 2^-60 to 2^40 side by side: what a row sees of the small ones is as exact as if the large ones were not there"""
    s = Served(ctx, code, 16, 2, 64, [100, 60], room=160)
    s.append(rows, P.F32)
    for i in range(2):
        for k in range(len(s.table[0])):
            s.plain.scales[1][s.table[i, k]] = 2.0 ** [-60, 40, -5, -30, 20][(k + i) % 5]
            s.plain.scales[0][s.table[i, k]] *= [1, 2.0 ** -40, 4][k % 3]
    s.scales = [ctx.upload(x.astype(np.float32)) for x in s.plain.scales]
    # windows that leave rows with small blocks alone
    for window in (0, 20, 33):
        s.attend(rows, 8, P.F32, window=window, weight_rows=4)
        s.attend(rows, 8, P.BF16, window=window)


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("rows", [[1, 1], [20, 30], [90, 70]])
def test_a_block_that_is_no_number(ctx, which, rows):
    """rows that see a token of it are NaN, in its head, and no others"""
    s = Served(ctx, Q.I8, 16, 2, 64, [100, 40], room=200)
    s.append(rows, P.F32)
    s.plain.scales[which][s.table[0, 2], 1] = np.nan
    s.plain.scales[which][s.table[1, 3], 0] = np.nan
    s.scales = [ctx.upload(x.astype(np.float32)) for x in s.plain.scales]
    got = s.attend(rows, 4, P.BF16)
    assert np.isnan(got).any() and not np.isnan(got).all()
    s.attend(rows, 4, P.BF16, window=30)
    # (of single tokens, none sees one here)
    got = s.attend(rows, 4, P.F32, window=50, first=8, weight_rows=ALL if which == 0 else 0)
    assert np.isnan(got).any() == (rows[0] > 1) and not np.isnan(got).all()


@pytest.mark.parametrize("dt", TYPES)
def test_weights_of_a_row_that_is_no_number(ctx, dt):
    """keys that such a row does not see get theirs from the others: behind it, and before its window"""
    for kv, heads, rows in ((1, 2, [6]), (1, 4, [40])):
        s = Served(ctx, Q.I8, 16, kv, 64, [100], room=200)
        s.append(rows, P.F32)
        x = s.rng.standard_normal((rows[0], heads * 64))
        x[2, 7] = np.nan
        y = np.delete(x, 2, 0)
        before = s.device_weights()
        got, grown = s.attend(rows, heads, dt, tail=0, query=x, window=20, weight_rows=ALL, check=False)
        assert np.isnan(got[2, :64]).all() and np.isfinite(np.delete(got, 2, 0)).all()
        tokens = np.arange(100 + rows[0])
        seen = (tokens <= 102) & (102 - tokens < 20)
        of = grown[s.table[0][tokens // 16], 0, tokens % 16]
        assert np.array_equal(np.isnan(of), seen), np.flatnonzero(np.isnan(of) != seen)
        assert len(y) and np.isfinite(before).all()


@pytest.mark.parametrize("dt", TYPES)
def test_queries_at_the_ends(ctx, dt):
    """queries that are zero, tiny, huge or not finite"""
    s = Served(ctx, Q.I8, 32, 1, 64, [50], room=100)
    s.append([8], P.F32)
    x = s.rng.standard_normal((8, 64))
    x[0] = 0
    x[1] *= 1e-5 if dt == P.F16 else 1e-30
    x[2] *= 30 if dt == P.F16 else 1e4
    x[3, 7] = np.inf
    x[4, 3] = np.nan
    x[5] *= np.exp2(-np.arange(64) / 4)
    x[6, 0] = 200
    ref = [i for i in range(8) if i not in (3, 4)]
    got = s.attend([8], 1, dt, tail=0, query=x, check=False)[0]
    assert np.isnan(got[3:5]).all() and np.isfinite(got[ref]).all()
    y = x.copy()
    y[3:5] = 0
    s.attend([8], 1, dt, tail=0, query=y)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rows", [[1, 8], [9, 3]])
def test_many_heads_of_one(ctx, dt, rows):
    """heads of one key head: few rows of many pairs, beside a sequence whose rows are not few"""
    s = Served(ctx, Q.E4M3, 32, 1, 64, [200, 77], room=300)
    s.append(rows, P.F32)
    s.attend(rows, 100, dt, weight_rows=ALL)
    s.attend(rows, 100, dt, window=40, first=3, weight_rows=2)


def test_long_and_many(ctx):
    """more keys than one CTA takes, more sequences than CTAs, and the other way round; the same bits twice"""
    s = Served(ctx, Q.I8, 64, 2, 128, [3000], room=3100)
    s.append([1], P.F32)
    s.attend([1], 8, P.BF16, weight_rows=ALL)
    s.set_lengths([2950])
    a = s.attend([3], 8, P.F32, query=np.ones((5, 1024)), check=False)[0]
    b = s.attend([3], 8, P.F32, query=np.ones((5, 1024)), check=False)[0]
    assert np.array_equal(a, b)
    s = Served(ctx, Q.E4M3, 16, 4, 32, [int(x) for x in np.random.default_rng(0).integers(0, 60, 300)], room=64)
    s.append([1] * 300, P.F32)
    s.attend([1] * 300, 4, P.BF16, weight_rows=1)


def test_a_cache_of_more_than_4_gb(ctx):
    """offsets behind 2^32 in both directions"""
    kv, block, dim, blocks = 8, 64, 128, 66000
    rng = np.random.default_rng(0)
    last = np.array([[blocks - 2, 5, blocks - 1]], np.uint32)
    codes = [ctx.buffer(blocks * kv * block * dim, B.BUFFER_DEVICE) for _ in range(2)]
    scales = [ctx.buffer(blocks * kv * 4, B.BUFFER_DEVICE) for _ in range(2)]
    table, length, new = ctx.upload(last), ctx.upload(np.array([0], np.uint32)), ctx.upload(np.zeros(1, np.uint32))
    offsets = ctx.upload(np.array([0, 150], np.uint32))
    cache = B.QuantizedCache(key_codes=codes[0].ptr, value_codes=codes[1].ptr, key_scales=scales[0].ptr, value_scales=scales[1].ptr, blocks=blocks, kv_heads=kv, block_tokens=block, head_dim=dim, code_type=Q.I8)
    seqs = B.CacheSequences(tables=table.ptr, lengths=length.ptr, row_offsets=offsets.ptr, count=1, table_stride=3, rows=150, max_rows=150, max_length=192)
    x = [P.to_kept(rng.standard_normal((150, kv * dim)), P.BF16) for _ in range(2)]
    rows = [ctx.upload(v) for v in x]
    back = [ctx.upload(np.zeros_like(v)) for v in x]
    q, out = ctx.upload(P.to_kept(rng.standard_normal((150, kv * dim)), P.BF16)), ctx.upload(np.zeros((150, kv * dim), np.uint16))
    common = dict(cache=cache, sequences=seqs)
    append = B.QuantizedCacheAppendArgs(keys=rows[0].ptr, values=rows[1].ptr, new_lengths=new.ptr, key_stride=kv * dim, value_stride=kv * dim, data_type=P.BF16, **common)
    read = B.QuantizedCacheReadArgs(keys=back[0].ptr, values=back[1].ptr, key_stride=kv * dim, value_stride=kv * dim, data_type=P.BF16, **common)
    att = B.QuantizedCacheAttentionArgs(query=q.ptr, out=out.ptr, heads=kv, query_row_stride=kv * dim, query_head_stride=dim, out_stride=kv * dim, scale=dim ** -0.5, data_type=P.BF16, **common)
    att.scratch_bytes = ctx.lib.uzu_quantized_cache_attention_scratch_bytes(ctx.h, C.byref(att))
    scratch = ctx.upload(np.zeros(att.scratch_bytes, np.uint8))
    att.scratch = scratch.ptr
    with ctx.command_buffer("far") as cmd:
        cmd.encode("uzu_quantized_cache_append_encode", C.byref(append))
        cmd.encode("uzu_quantized_cache_read_encode", C.byref(read))
        cmd.encode("uzu_quantized_cache_attention_encode", C.byref(att))
    small = Q.Cache(3, kv, block, dim, Q.I8)
    k, v = (P.of_kept(a, P.BF16).reshape(150, kv, dim) for a in x)
    small.append(np.arange(3), 0, (k, v), 192)
    for w in range(2):
        want = small.numbers(w, np.arange(3), np.arange(150))[0].reshape(150, -1)
        assert np.array_equal(P.of_kept(back[w].numpy(np.uint16, (150, kv * dim)), P.BF16), want)
    ref, bound, _, _ = small.attend(np.arange(3), 0, P.of_kept(q.numpy(np.uint16, (150, kv * dim)), P.BF16).reshape(150, kv, dim), 192, float(np.float32(dim ** -0.5)), tensor=True)
    got = P.of_kept(out.numpy(np.uint16, (150, kv * dim)), P.BF16).reshape(ref.shape)
    assert (np.abs(got - ref) <= P.HALF_STEP[P.BF16] * (np.abs(ref) + bound) + bound).all()
    for b in codes + scales:
        b.close()


# ---- eviction -------------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("block,heads,dim", [(16, 3, 48), (32, 2, 64), (64, 2, 256)])
@pytest.mark.parametrize("budget,first,last", [(100, 4, 20), (33, 0, 0), (64, 30, 34), (1, 0, 0), (299, 0, 1), (96, 96, 0)])
def test_evict(ctx, code, block, heads, dim, budget, first, last):
    s = Served(ctx, code, block, heads, dim, [300, 0, 101, 100, 297, budget, budget + 1], room=310)
    s.plain.weights = np.round(s.plain.weights * 4) / 4      # (many alike)
    s.weights = ctx.upload(s.plain.weights.astype(np.float32))
    s.evict(budget, first, last)
    s.evict(budget, first, last, indices=False)


def test_evict_special_weights(ctx):
    """NaN behind everything, zeros of both signs alike, infinities, all the same"""
    s = Served(ctx, Q.I8, 16, 4, 32, [200, 150], room=210)
    w = s.plain.weights
    w[:, 0] = 1.0
    w[:, 1] = np.where(s.rng.random(w[:, 1].shape) < 0.7, np.nan, w[:, 1])
    w[:, 2] = np.where(s.rng.random(w[:, 2].shape) < 0.5, 0.0, -0.0)
    w[:, 3] = s.rng.choice([np.inf, -np.inf, -1.0, 1e-45, 0.0], w[:, 3].shape)
    s.plain.weights = w.astype(np.float32).astype(np.float64)      # (1e-45 is not a number of 32 bits)
    s.weights = ctx.upload(w.astype(np.float32))
    s.evict(90, 2, 3)


@pytest.mark.parametrize("code", CODES)
def test_evict_without_blocks_and_without_numbers(ctx, code):
    s = Served(ctx, code, 16, 2, 32, [200, 150, 500], room=210, missing=[(0, 2), (0, 7), (1, 0), (2, 12)])
    s.plain.scales[0][s.table[0, 5], 1] = np.nan
    s.plain.scales[1][s.table[1, 3]] = 0.0
    s.plain.scales[1][s.table[0, 9], 0] = 2.0 ** 30
    s.scales = [ctx.upload(x.astype(np.float32)) for x in s.plain.scales]
    s.evict(90, 2, 3)
    s.evict(60, 0, 40, max_length=85)


@pytest.mark.parametrize("lengths,budget", [([60000], 20000), ([42000, 3, 41000], 41500), ([9000] * 6, 4096)])
def test_evict_long(ctx, lengths, budget):
    """more weights than shared memory holds, many blocks that wait for one another"""
    s = Served(ctx, Q.I8, 32, 2, 16, lengths, room=max(lengths))
    s.evict(budget, 4, budget // 8)


# ---- together -------------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("code", CODES)
def test_a_served_batch(ctx, code):
    """prompts, answers token by token with their weights summed up, cut by weight, drafted tokens of which some are kept: as a server runs them"""
    kv, heads, dim = 2, 8, 64
    s = Served(ctx, code, 32, kv, dim, [0, 0, 0], room=260)
    s.plain.weights[:] = 0
    s.weights = ctx.upload(s.plain.weights.astype(np.float32))
    rows = [150, 70, 33]
    after = s.append(rows, P.BF16)
    s.attend(rows, heads, P.BF16, weight_rows=16)
    for _ in range(3):
        s.set_lengths(after)
        after = s.append([1, 1, 1], P.BF16)
        s.attend([1, 1, 1], heads, P.BF16, weight_rows=ALL)
    s.set_lengths(after)
    after = s.evict(64, 4, 16)
    assert after == [64, 64, 36]
    s.set_lengths(after)
    s.append([5, 5, 5], P.BF16)
    s.attend([5, 5, 5], heads, P.BF16, weight_rows=ALL)
    rng = np.random.default_rng(1)
    target = 2 * rng.standard_normal((3, 5, 500))
    draft = target[:, :4] + 0.3 * rng.standard_normal((3, 4, 500))
    accepted, _, clear = verify(ctx, target, draft, draft.argmax(2), rng.random((3, 5)), 1.0, 1.0, P.BF16)
    assert clear
    # the refused tokens' places are taken by what comes next
    after = [int(n + 1 + a) for n, a in zip(after, accepted)]
    s.set_lengths(after)
    s.append([1, 1, 1], P.BF16)
    s.attend([1, 1, 1], heads, P.BF16)
    s.read([0, 0, 0], [n + 1 for n in after], P.BF16)


def test_captured_calls_follow_the_device(ctx):
    """append and attention captured once: a replay follows the lengths, offsets and tables that the device holds then"""
    from tests.test_state_space_gpu import _captured
    kv, heads, dim = 2, 8, 64
    s, ref = (Served(ctx, Q.I8, 32, kv, dim, [40, 99], room=200, seed=3) for _ in range(2))
    x = [s.rng.standard_normal((4, kv * dim)) for _ in range(2)]
    q = s.rng.standard_normal((4, heads * dim))
    qb, out = ctx.upload(P.to_kept(q, P.BF16)), ctx.upload(np.zeros((4, heads * dim), np.uint16))
    rows = [ctx.upload(P.to_kept(v, P.BF16)) for v in x]
    offsets = ctx.upload(np.array([0, 2, 4], np.uint32))
    seqs = B.CacheSequences(tables=s.tables.ptr, lengths=s.length_buffer.ptr, row_offsets=offsets.ptr, count=2, table_stride=s.table.shape[1], rows=4, max_rows=4, max_length=s.room)
    append = B.QuantizedCacheAppendArgs(cache=s.cache(), sequences=seqs, keys=rows[0].ptr, values=rows[1].ptr, new_lengths=s.new_lengths.ptr, key_stride=kv * dim, value_stride=kv * dim, data_type=P.BF16)
    att = B.QuantizedCacheAttentionArgs(cache=s.cache(), sequences=seqs, query=qb.ptr, out=out.ptr, heads=heads, query_row_stride=heads * dim, query_head_stride=dim, out_stride=heads * dim,
                                        weight_rows=ALL, scale=0.125, data_type=P.BF16)
    att.scratch_bytes = ctx.lib.uzu_quantized_cache_attention_scratch_bytes(ctx.h, C.byref(att))
    scratch = ctx.upload(np.zeros(att.scratch_bytes, np.uint8))
    att.scratch = scratch.ptr

    def both(cmd):
        ctx.lib.uzu_quantized_cache_append_encode(cmd, C.byref(append))
        ctx.lib.uzu_quantized_cache_attention_encode(cmd, C.byref(att))

    ref.attend([2, 2], heads, P.BF16, query=np.concatenate([q, q[:0]]), tail=0, weight_rows=ALL, check=False)      # (a kernel's first launch sets its shared memory, which is not captured)
    ref = Served(ctx, Q.I8, 32, kv, dim, [40, 99], room=200, seed=3)
    ref.rng = np.random.default_rng(0)
    replay = _captured(ctx, both)
    for lengths, parts in (([40, 99], [2, 2]), ([42, 101], [1, 3]), ([43, 104], [4, 0])):
        C.memmove(s.length_buffer.cpu_ptr, np.array(lengths + [0], np.uint32).ctypes.data, 12)
        C.memmove(offsets.cpu_ptr, np.cumsum([0] + parts).astype(np.uint32).ctypes.data, 12)
        replay()
        ref.set_lengths(lengths)
        ref.append(parts, P.BF16, values=x, tail=0)
        ref.attend(parts, heads, P.BF16, query=q, tail=0, weight_rows=ALL, scale=0.125)
        s.plain = ref.plain
        assert s.same()
        assert np.array_equal(s.device_weights(), ref.device_weights())
        want = ref.attend(parts, heads, P.BF16, query=q, tail=0, scale=0.125)
        assert np.array_equal(P.of_kept(out.numpy(np.uint16, (4, heads * dim)), P.BF16), want)


@pytest.mark.parametrize("code", CODES)
def test_captured_evictions(ctx, code):
    """what a call counts and waits for begins anew in every replay, and the lengths are those that the device holds then"""
    from tests.test_state_space_gpu import _captured
    s = Served(ctx, code, 32, 2, 64, [190, 77, 64], room=200, seed=4)
    s.evict(64, 4, 16)      # (a kernel's first launch sets its shared memory, which is not captured)
    args = s.last
    replay = _captured(ctx, lambda cmd: ctx.lib.uzu_quantized_cache_evict_encode(cmd, C.byref(args)))
    for lengths in ([150, 3, 200], [64, 65, 0], [199, 199, 199]):
        C.memmove(s.length_buffer.cpu_ptr, np.array(lengths + [0], np.uint32).ctypes.data, 16)
        replay()
        after = [s.plain.evict(s.table[i], min(n, s.capacity()), 64, 4, 16)[1] for i, n in enumerate(lengths)]
        assert s.new_lengths.numpy(np.uint32, (4,)).tolist() == after + [77]
        assert s.same()
        assert np.array_equal(s.device_weights(), s.plain.weights)


def test_captured_prompts(ctx):
    """both kernels of a pass of prompts and single tokens: a replay gives what a call gives"""
    from tests.test_state_space_gpu import _captured
    heads = 8
    s = Served(ctx, Q.I8, 32, 2, 64, [40, 99], room=300, seed=5)
    s.append([90, 90], P.BF16)
    q = s.rng.standard_normal((180, heads * 64))
    kw = dict(query=q, tail=0, max_rows=170)
    s.attend([90, 90], heads, P.BF16, **kw)
    args, out, offsets, lengths = s.last, s.kept[-3], s.kept[-6], s.length_buffer
    assert offsets.ptr == args.sequences.row_offsets and out.ptr == args.out
    replay = _captured(ctx, lambda cmd: ctx.lib.uzu_quantized_cache_attention_encode(cmd, C.byref(args)))
    for held, rows in (([40, 99], [90, 90]), ([100, 20], [10, 170]), ([10, 128], [179, 1])):
        C.memmove(lengths.cpu_ptr, np.array(held + [0], np.uint32).ctypes.data, 12)
        C.memmove(offsets.cpu_ptr, np.cumsum([0] + rows).astype(np.uint32).ctypes.data, 12)
        replay()
        got = out.get()[0]
        s.set_lengths(held)
        n = min(rows[0], 170)      # (rows behind max_rows are left out)
        if n < rows[0]:
            want = s.attend(rows, heads, P.BF16, check=False, **kw)[0]
            assert np.array_equal(got[:n], want[:n]) and np.array_equal(got[rows[0]:], want[rows[0]:])
        else:
            assert np.array_equal(got, s.attend(rows, heads, P.BF16, **kw))


def test_refused_calls_are_errors_of_their_buffer(ctx):
    s = Served(ctx, Q.I8, 32, 2, 64, [40], room=100)
    s.attend([1], 8, P.BF16)
    a = s.last
    before = s.codes[0].numpy(np.uint8)
    for over in (dict(heads=3), dict(scratch_bytes=64), dict(out=0)):
        bad = B.QuantizedCacheAttentionArgs.from_buffer_copy(a)
        for k, v in over.items():
            setattr(bad, k, v)
        with pytest.raises(B.UzuError):
            s.run("bad", ("uzu_quantized_cache_attention_encode", bad))
    s.evict(20, 0, 0)
    bad = B.QuantizedCacheEvictArgs.from_buffer_copy(s.last)
    bad.scratch_bytes = 16
    with pytest.raises(B.UzuError):
        s.run("bad", ("uzu_quantized_cache_evict_encode", bad))
    assert len(before) and s.same()


# ---- verification -----------------------------------------------------------------------------------------------------------------------------------
def _case(rng, n, k, vocab, near=0.5, spread=2.0):
    target = spread * rng.standard_normal((n, k + 1, vocab))
    draft = target[:, :k] + near * rng.standard_normal((n, k, vocab))
    gumbel = -np.log(-np.log(rng.random((n, k, vocab))))
    return target, draft, (draft + gumbel).argmax(2) if k else np.zeros((n, 0), np.int64), rng.random((n, k + 1))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("vocab", [1, 2, 255, 1000, 32001, 70000])
@pytest.mark.parametrize("k", [0, 1, 4, 16])
def test_verify(ctx, dt, vocab, k):
    rng = np.random.default_rng(vocab + k)
    target, draft, drafted, u = _case(rng, 5, k, vocab)
    clear = [verify(ctx, target, draft if k else None, drafted, u, 1.0, 1.0, dt)[2], verify(ctx, target, None, drafted, u, 0.75, 0.0, dt)[2], verify(ctx, target, draft if k else None, drafted, u, 0.0, 1.0, dt)[2],
             verify(ctx, target, draft if k else None, drafted, u, 1.5, 0.5, dt, stride=vocab + 5, shift=1)[2]]
    assert sum(clear) >= 15


def test_verify_counts_and_strange_drafts(ctx):
    """fewer drafts than the rows hold, drafts that are no tokens, the same logits on both sides, numbers at the ends of the range"""
    rng = np.random.default_rng(5)
    target, draft, drafted, u = _case(rng, 6, 4, 3000)
    drafted[1, 2], drafted[2, 0] = 3000, NONE
    draft[3] = target[3, :4]
    u[4], u[5] = 0.0, np.float32(1 - 2.0 ** -24)
    for temperature in (1.0, 0.0):
        verify(ctx, target, draft, drafted, u, temperature, 1.0, P.F32, counts=[4, 3, 1, 9, 0, 2])
        verify(ctx, target, None, drafted, u, temperature, 1.0, P.BF16, counts=[0, 0, 4, 4, 4, 4])


def test_verify_rows_without_a_distribution(ctx):
    """masked tokens have no weight; a NaN, +infinity or nothing at all ends the sequence's tokens"""
    rng = np.random.default_rng(6)
    target, draft, drafted, u = _case(rng, 9, 3, 2000, near=0.1)
    u[:, :3] *= 0.2      # (kept, if they can be)
    target[0, 0, 100:] = -np.inf
    target[1, 1] = -np.inf
    target[2, 0, 1999] = np.inf
    target[3, 2, 7] = np.nan
    draft[4, 1, 3] = np.nan
    draft[5, 0] = -np.inf
    target[6, 3, 0] = np.nan
    target[7, 0, 1:] = -np.inf
    target[8, :, :1990] = -np.inf
    for temperature in (1.0, 0.0):
        for d in (draft, None):
            accepted, tokens, clear = verify(ctx, target, d, drafted, u, temperature, 1.0, P.BF16)
            assert clear >= 7 and accepted[2] == 0 and tokens[2, 0] == NONE


def test_verify_a_certain_draft_with_all_of_p(ctx):
    """nothing is left beside it: it comes as the token behind if it is not kept"""
    target = np.full((2, 2, 300), -np.inf)
    target[:, 0, 7], target[0, 1, 9], target[1, 1] = 1.0, 0.0, 0.0
    u = np.array([[1.0, 0.5], [0.25, 0.999]])      # (the first is outside the range: the draft is not kept)
    got = verify(ctx, target, None, np.full((2, 1), 7), u, 1.0, 1.0, P.F32)
    assert got[1][0].tolist() == [7, NONE] and got[0].tolist() == [0, 1] and got[1][1, 0] == 7


def test_captured_verification(ctx):
    """a replay reads the drafts and uniform numbers that the device holds then"""
    from tests.test_state_space_gpu import _captured
    n, k, vocab = 3, 4, 5000
    rng = np.random.default_rng(11)
    target, draft, drafted, u = _case(rng, n, k, vocab)
    t, d = (ctx.upload(x.reshape(-1, vocab).astype(np.float32)) for x in (target, draft))
    dr, un = ctx.upload(drafted.astype(np.uint32)), ctx.upload(u.astype(np.float32))
    tokens, accepted = ctx.upload(np.zeros((n, k + 1), np.uint32)), ctx.upload(np.zeros(n, np.uint32))
    verify(ctx, target, draft, drafted, u, 1.0, 1.0, P.F32)
    a = B.DraftVerifyArgs(target_logits=t.ptr, draft_logits=d.ptr, drafted=dr.ptr, uniforms=un.ptr, tokens=tokens.ptr, accepted=accepted.ptr, sequences=n, drafts=k, vocab=vocab, target_stride=vocab,
                          draft_stride=vocab, temperature=1.0, draft_temperature=1.0, data_type=P.F32)
    replay = _captured(ctx, lambda cmd: ctx.lib.uzu_draft_verify_encode(cmd, C.byref(a)))
    for _ in range(3):
        drafted, u = rng.integers(0, vocab, (n, k)), rng.random((n, k + 1))
        drafted[0] = draft[0].argmax(1)
        held = [np.ascontiguousarray(drafted, np.uint32), np.ascontiguousarray(u, np.float32)]
        for buffer, x in zip((dr, un), held):
            C.memmove(buffer.cpu_ptr, x.ctypes.data, x.nbytes)
        replay()
        acc, tok, _ = verify(ctx, target, draft, drafted, u, 1.0, 1.0, P.F32)
        assert np.array_equal(accepted.numpy(np.uint32, (n,)), acc) and np.array_equal(tokens.numpy(np.uint32, (n, k + 1)), tok)


def test_verify_draws_the_target(ctx):
    """kept or drawn anew, first tokens are spread as the target's distribution: every interval of the uniform numbers has its share"""
    rng = np.random.default_rng(7)
    n, vocab = 4096, 8
    one, other = rng.standard_normal((1, 1, vocab)), rng.standard_normal((1, 1, vocab))
    target, draft = np.repeat(np.repeat(one, 2, 1), n, 0), np.repeat(other, n, 0)
    q = np.exp(other[0, 0]) / np.exp(other[0, 0]).sum()
    drafted = rng.choice(vocab, (n, 1), p=q)
    _, tokens, _ = verify(ctx, target, draft, drafted, rng.random((n, 2)), 1.0, 1.0, P.F32)
    p = np.exp(one[0, 0]) / np.exp(one[0, 0]).sum()
    share = np.bincount(tokens[:, 0], minlength=vocab) / n
    assert np.abs(share - p).max() < 5 * np.sqrt(0.25 / n)      # (five standard deviations)
