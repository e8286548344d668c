"""An 8-bit cache on the device beside its plain form, and the calls on it."""
import ctypes as C

import numpy as np

from tests import quantized_cache_plain as Q
from tests import state_space_plain as P
from tests.test_state_space_gpu import _np, _Rows
from uzu_b200 import binding as B

NONE = 0xFFFFFFFF


class Served:
    """A cache, its tables and the lengths of its sequences, on the device and in float64."""

    def __init__(self, ctx, code, block, heads, dim, lengths, room=200, seed=0, garbage=None, spare=3, missing=()):
        rng = self.rng = np.random.default_rng(seed)
        self.ctx, self.n, self.code = ctx, len(lengths), code
        per = -(-room // block) + 1
        blocks = per * self.n + spare
        self.plain = Q.Cache(blocks, heads, block, dim, code, rng, garbage)
        order = rng.permutation(blocks)
        self.table = order[:per * self.n].reshape(self.n, per).astype(np.uint32)
        for i, k in missing:
            self.table[i, k] = [blocks, NONE, blocks + 1][k % 3]
        self.lengths, self.room = list(lengths), per * block
        self.codes = [ctx.upload(c) for c in self.plain.codes]
        self.scales = [ctx.upload(s.astype(np.float32)) for s in self.plain.scales]
        self.weights = ctx.upload(self.plain.weights.astype(np.float32))
        self.tables = ctx.upload(self.table)
        self.length_buffer = ctx.upload(np.array(lengths + [0], np.uint32))
        self.new_lengths = ctx.upload(np.full(self.n + 1, 77, np.uint32))
        self.kept = []

    def cache(self, weights=True):
        p = self.plain
        return B.QuantizedCache(key_codes=self.codes[0].ptr, value_codes=self.codes[1].ptr, key_scales=self.scales[0].ptr, value_scales=self.scales[1].ptr, key_weights=self.weights.ptr if weights else 0,
                                blocks=p.blocks, kv_heads=p.heads, block_tokens=p.block, head_dim=p.dim, code_type=p.code)

    def sequences(self, rows=(), total=None, max_rows=None, max_length=None, lengths=None):
        offsets = self.ctx.upload(np.concatenate([[0], np.cumsum(rows if len(rows) else [0] * self.n)]).astype(np.uint32))
        at = self.length_buffer if lengths is None else self.ctx.upload(np.array(lengths, np.uint32))
        self.kept += [offsets, at]
        return B.CacheSequences(tables=self.tables.ptr, lengths=at.ptr, row_offsets=offsets.ptr, count=self.n, table_stride=self.table.shape[1], rows=sum(rows) if total is None else total,
                                max_rows=max(rows, default=0) if max_rows is None else max_rows, max_length=self.room if max_length is None else max_length)

    def capacity(self, max_length=None):
        return min(self.room, max_length or self.room)

    def set_lengths(self, lengths):
        self.lengths = list(lengths)
        self.length_buffer = self.ctx.upload(np.array(list(lengths) + [0], np.uint32))
        self.kept.append(self.length_buffer)

    def run(self, name, *calls):
        with self.ctx.command_buffer(name) as cmd:
            for fn, args in calls:
                cmd.encode(fn, C.byref(args))

    def same(self, only_tokens=False):
        """the device's cache is the plain form's, bit for bit: all of it, or what stands for numbers (tokens of the sequences)"""
        p = self.plain
        for w in range(2):
            got = self.codes[w].numpy(np.uint8, p.codes[w].shape)
            assert np.array_equal(got, p.codes[w]), (w, np.argwhere(got != p.codes[w])[:4])
            s = self.scales[w].numpy(np.float32, p.scales[w].shape).astype(np.float64)
            assert np.array_equal(s, p.scales[w], equal_nan=True), (w, s[s != p.scales[w]][:4], p.scales[w][s != p.scales[w]][:4])
        return True

    def device_weights(self):
        return self.weights.numpy(np.float32, self.plain.weights.shape).astype(np.float64)

    # ---- append ----
    def append(self, rows, dt, values=None, stride=0, shift=0, tail=2, max_length=None, new_lengths=True):
        p = self.plain
        width, total = p.heads * p.dim, sum(rows) + tail
        x = values if values is not None else [self.rng.standard_normal((total, width)) * np.exp2(self.rng.integers(-3, 3, (total, 1))) for _ in range(2)]
        k, v = (_Rows(self.ctx, a, dt, stride=stride, shift=shift) for a in x)
        a = B.QuantizedCacheAppendArgs(cache=self.cache(), sequences=self.sequences(rows, total, max_length=max_length), keys=k.ptr, values=v.ptr, new_lengths=self.new_lengths.ptr if new_lengths else 0,
                                       key_stride=k.stride, value_stride=v.stride, data_type=dt)
        self.run("append", ("uzu_quantized_cache_append_encode", a))
        at, after = 0, []
        for i, n in enumerate(rows):
            mine = [P.of_kept(P.to_kept(b[at:at + n], dt), dt).reshape(n, p.heads, p.dim) for b in x]
            after.append(p.append(self.table[i], self.lengths[i], mine, self.capacity(max_length)))
            at += n
        if new_lengths:
            assert self.new_lengths.numpy(np.uint32, (self.n + 1,)).tolist() == after + [77]
        return after

    # ---- attention ----
    def attend(self, rows, heads, dt, stride=0, shift=0, tail=2, window=0, first=0, cap=0.0, sinks=None, weight_rows=0, scale=None, head_major=False, max_length=None, query=None, check=True, max_rows=None):
        p = self.plain
        total, width = sum(rows) + tail, heads * p.dim
        scale = np.float32(p.dim ** -0.5 if scale is None else scale)
        x = 1.5 * self.rng.standard_normal((total, width)) if query is None else query
        if head_major:
            q = _Rows(self.ctx, x.reshape(total, heads, p.dim).transpose(1, 0, 2).reshape(heads * total, p.dim), dt, shift=shift)
            strides = dict(query_row_stride=p.dim, query_head_stride=total * p.dim)
        else:
            q = _Rows(self.ctx, x, dt, stride=stride, shift=shift)
            strides = dict(query_row_stride=q.stride, query_head_stride=p.dim)
        out = _Rows(self.ctx, np.full((total, width), 7.0), dt, stride=stride, shift=shift)
        before = out.raw().copy()
        s = self.ctx.upload(np.asarray(sinks, np.float32)) if sinks is not None else None
        a = B.QuantizedCacheAttentionArgs(cache=self.cache(), sequences=self.sequences(rows, total, max_length=max_length, max_rows=max_rows), query=q.ptr, out=out.ptr, sinks=s.ptr if s else 0, heads=heads,
                                          out_stride=out.stride, window=window, keep_first=first, weight_rows=weight_rows, scale=scale, softcap=cap, data_type=dt, **strides)
        a.scratch_bytes = self.ctx.lib.uzu_quantized_cache_attention_scratch_bytes(self.ctx.h, C.byref(a))
        scratch = self.ctx.upload(np.zeros(a.scratch_bytes, np.uint8))
        a.scratch = scratch.ptr
        weights = self.device_weights()
        self.run("attention", ("uzu_quantized_cache_attention_encode", a))
        got, raw = out.get()
        self.kept += [q, out, s, scratch]
        self.last = a
        if not check:
            return got, self.device_weights() - weights
        # f32 queries are two f16 parts of 11 bits: 22, each product's half step 2^-23. more than 8 bf16 rows of more than 64 pairs go to the tensor cores' kernel
        tensor = dt == P.BF16 and p.dim <= 128 and scale > 0 and not shift and (stride or 8) % 8 == 0
        at, grown, grown_bound = 0, np.zeros_like(weights), np.zeros_like(weights)
        for i, n in enumerate(rows):
            mine = P.of_kept(P.to_kept(x[at:at + n], dt), dt).reshape(n, heads, p.dim)
            capn = self.capacity(max_length)
            ref, bound, grow, gb = p.attend(self.table[i], self.lengths[i], mine, capn, float(scale), window, first, cap, sinks, weight_rows, 2.0 ** -22 if dt == P.F32 else 0.0,
                                                tensor and n > 8 and n * heads // p.heads > 64, dt != P.F32)
            mine_got = got[at:at + n].reshape(n, heads, p.dim)
            assert np.array_equal(np.isnan(mine_got), np.isnan(ref)), (i, np.argwhere(np.isnan(mine_got) != np.isnan(ref))[:4])
            with np.errstate(invalid="ignore"):
                tol = P.HALF_STEP[dt] * (np.abs(ref) + bound) + P.TINY[dt] + bound
                bad = np.abs(mine_got - ref) > tol
            assert not bad.any(), (i, int(bad.sum()), np.argwhere(bad)[0].tolist(), mine_got[bad][:3], ref[bad][:3], bound[bad][:3])
            tokens = np.arange(len(grow))
            b = self.table[i][tokens // p.block]
            for j in tokens[b < p.blocks]:
                grown[b[j], :, j % p.block] += grow[j]
                grown_bound[b[j], :, j % p.block] += gb[j]
            at += n
        # rows of no sequence, and what is beside rows, keep what they held
        assert np.array_equal(raw[at:], before[at:]) and np.array_equal(raw[:, width:], before[:, width:])
        after = self.device_weights()
        if not weight_rows:
            assert np.array_equal(after, weights)
        else:
            want = weights + grown
            assert np.array_equal(np.isnan(after), np.isnan(want))
            with np.errstate(invalid="ignore"):
                # (one addition for each tile of 16 pairs)
                worst = np.abs(after - want) - grown_bound - 2.0 ** -24 * (1 + max(rows) * heads / 16) * (np.abs(want) + 1e-30)
            assert not (worst > 0).any(), (float(np.nanmax(worst)), np.argwhere(worst > 0)[:3])
            self.plain.weights = after.copy()
        return got

    # ---- read, evict ----
    def read(self, begin, rows, dt, kinds=(True, True), max_length=None, stride=0, shift=0):
        p = self.plain
        total, width = sum(rows) + 2, p.heads * p.dim
        out = [_Rows(self.ctx, np.full((total, width), 3.0), dt, stride=stride, shift=shift) for _ in range(2)]
        a = B.QuantizedCacheReadArgs(cache=self.cache(False), sequences=self.sequences(rows, total, lengths=begin, max_length=max_length), keys=out[0].ptr if kinds[0] else 0, values=out[1].ptr if kinds[1] else 0,
                                     key_stride=out[0].stride, value_stride=out[1].stride, data_type=dt)
        self.run("read", ("uzu_quantized_cache_read_encode", a))
        for w in range(2):
            want = np.full((total, width), 3.0)
            at = 0
            for i, n in enumerate(rows):
                if kinds[w]:
                    tokens = np.arange(begin[i], min(begin[i] + n, self.capacity(max_length)))
                    x, there = p.numbers(w, self.table[i], tokens)
                    want[at + np.flatnonzero(there)] = x[there].reshape(-1, width)
                at += n
            got, raw = out[w].get()
            assert np.array_equal(got, P.of_kept(P.to_kept(want, dt), dt), equal_nan=True), w
        return True

    def evict(self, budget, first, last, indices=True, max_length=None):
        p = self.plain
        idx = self.ctx.upload(np.full((self.n, p.heads, budget), 5, np.uint32))
        a = B.QuantizedCacheEvictArgs(cache=self.cache(), sequences=self.sequences(max_length=max_length), new_lengths=self.new_lengths.ptr, indices=idx.ptr if indices else 0, budget=budget, keep_first=first,
                                      keep_last=last)
        a.scratch_bytes = self.ctx.lib.uzu_quantized_cache_evict_scratch_bytes(self.ctx.h, C.byref(a))
        scratch = self.ctx.upload(np.full(a.scratch_bytes, 0xA5, np.uint8))
        a.scratch = scratch.ptr
        self.run("evict", ("uzu_quantized_cache_evict_encode", a))
        self.kept += [idx, scratch]
        self.last = a
        after = []
        got = idx.numpy(np.uint32, (self.n, p.heads, budget))
        for i in range(self.n):
            keep, n = p.evict(self.table[i], min(self.lengths[i], self.capacity(max_length)), budget, first, last)
            after.append(n)
            if indices:
                assert np.array_equal(got[i, :, :n], keep) and (got[i, :, n:] == NONE).all(), i
        assert self.new_lengths.numpy(np.uint32, (self.n + 1,)).tolist() == after + [77]
        self.same()
        assert np.array_equal(self.device_weights(), p.weights, equal_nan=True)
        return after


def verify(ctx, target, draft, drafted, uniforms, temperature, draft_temperature, dt, counts=None, stride=0, shift=0):
    """target [n, k + 1, vocab], draft [n, k, vocab] or None. (accepted, tokens) of the device, checked against the plain form where its decisions are clear"""
    n, k1, vocab = target.shape
    k = k1 - 1
    t = _Rows(ctx, target.reshape(n * k1, vocab), dt, stride=stride, shift=shift)
    d = _Rows(ctx, draft.reshape(n * k, vocab), dt, stride=stride, shift=shift) if draft is not None else None
    dr, un = ctx.upload(drafted.astype(np.uint32)), ctx.upload(uniforms.astype(np.float32))
    tokens, accepted = ctx.upload(np.full((n + 1, k1), 9, np.uint32)), ctx.upload(np.full(n + 1, 9, np.uint32))
    cn = ctx.upload(np.asarray(counts, np.uint32)) if counts is not None else None
    a = B.DraftVerifyArgs(target_logits=t.ptr, draft_logits=d.ptr if d else 0, drafted=dr.ptr, draft_counts=cn.ptr if cn else 0, uniforms=un.ptr, tokens=tokens.ptr, accepted=accepted.ptr, sequences=n, drafts=k,
                          vocab=vocab, target_stride=t.stride, draft_stride=d.stride if d else 0, temperature=temperature, draft_temperature=draft_temperature, data_type=dt)
    with ctx.command_buffer("verify") as cmd:
        cmd.encode("uzu_draft_verify_encode", C.byref(a))
    acc, tok = accepted.numpy(np.uint32, (n + 1,)), tokens.numpy(np.uint32, (n + 1, k1))
    assert acc[n] == 9 and (tok[n] == 9).all()
    kept = lambda x: P.of_kept(P.to_kept(x, dt), dt)
    clear = 0
    for i in range(n):
        m = k if counts is None else min(k, int(counts[i]))
        with np.errstate(invalid="ignore", over="ignore"):
            want, token, sure = Q.verify(kept(target[i, :m + 1]), kept(draft[i, :m]) if draft is not None else None, drafted[i, :m].astype(np.int64), np.append(uniforms[i, :m], uniforms[i, k]).astype(np.float32).astype(np.float64),
                                         float(np.float32(temperature)), float(np.float32(draft_temperature)))
        if not sure:
            continue
        clear += 1
        assert acc[i] == want, (i, acc[i], want, tok[i])
        assert tok[i].tolist() == drafted[i, :want].tolist() + [token] + [Q.NO_INDEX] * (k - want), (i, want, token, tok[i])
    return acc[:n], tok[:n], clear


__all__ = ["Served", "verify", "_np", "NONE"]
