"""A cache of 8 bits, the attention that reads it, eviction from it, and the verification of drafted tokens, as measured cases.

  append   new key and value rows of packed sequences into a paged cache of 8-bit codes, one scale per block of tokens and head, and the rows read back
  attend   attention over that cache: single tokens, drafted tokens, prompts; optionally the attention weight of every cached token is summed up
  evict    a long sequence cut down to the tokens that had the most weight, the first and the last ones, and the kept tokens read back
  verify   drafted tokens accepted or refused against the target's probabilities from given random numbers, and the next token drawn

A pass goes through the entry points of `uzu_b200.binding` (a command buffer that the state keeps open, as a host program that brings its own
graph encodes into it), or through elementary torch operations that say the same.
"""
from __future__ import annotations

import math

import torch

own = False

F32, F64 = torch.float32, torch.float64
TYPES = {"bf16": (torch.bfloat16, 0), "f32": (torch.float32, 1), "f16": (torch.float16, 2)}
CODES = {"i8": 0, "e4m3": 1}
LARGEST = {"i8": 127.0, "e4m3": 448.0}
ALL = 0xFFFFFFFF
NO_TOKEN = 0xFFFFFFFF
TAIL = 3          # rows behind the last sequence: of a padded pass, left as they are
SPARE = 3         # blocks of the pool beyond what the sequences may take


def listed():
    return [
        # a served batch decodes: every sequence's new token enters the cache
        {"name": "append-step", "kind": "append", "type": "bf16", "code": "i8", "kv_heads": 8, "dim": 128, "block": 32, "sequences": 64, "cached": 64 * 2048, "rows": 64},
        # five prompts of different lengths behind what their sequences hold
        {"name": "append-prompts", "kind": "append", "type": "bf16", "code": "e4m3", "kv_heads": 8, "dim": 128, "block": 64, "sequences": 5, "cached": 3001, "rows": 16384},
        # one user's answer: latency counts
        {"name": "attend-1", "kind": "attend", "type": "bf16", "code": "e4m3", "heads": 32, "kv_heads": 8, "dim": 128, "block": 64, "sequences": 1, "cached": 4099, "rows": 1, "window": 0, "first": 0, "cap": 0.0, "weights": 0},
        # one answer behind a very long document
        {"name": "attend-long", "kind": "attend", "type": "bf16", "code": "i8", "heads": 32, "kv_heads": 8, "dim": 128, "block": 64, "sequences": 1, "cached": 131071, "rows": 1, "window": 0, "first": 0, "cap": 0.0, "weights": 0},
        # a served batch, whose cache is cut by weight from time to time
        {"name": "attend-batch", "kind": "attend", "type": "bf16", "code": "i8", "heads": 32, "kv_heads": 8, "dim": 128, "block": 32, "sequences": 64, "cached": 64 * 4096, "rows": 64, "window": 0, "first": 0, "cap": 0.0, "weights": ALL},
        # four drafted tokens and the last one of each of sixteen sequences, a window that keeps the first tokens, capped scores
        {"name": "attend-drafts", "kind": "attend", "type": "bf16", "code": "e4m3", "heads": 32, "kv_heads": 8, "dim": 64, "block": 32, "sequences": 16, "cached": 16 * 6000, "rows": 80, "window": 4096, "first": 4, "cap": 50.0, "weights": 0},
        # a short turn on a small model kept in 32 bits; the last rows of a prompt say which keys matter
        {"name": "attend-turn", "kind": "attend", "type": "f32", "code": "i8", "heads": 8, "kv_heads": 2, "dim": 256, "block": 16, "sequences": 1, "cached": 1003, "rows": 77, "window": 0, "first": 0, "cap": 0.0, "weights": 32},
        # three prompts' next parts, ragged
        {"name": "attend-prompts", "kind": "attend", "type": "bf16", "code": "i8", "heads": 32, "kv_heads": 8, "dim": 128, "block": 64, "sequences": 3, "cached": 12000, "rows": 6144, "window": 0, "first": 0, "cap": 0.0, "weights": 0},
        # one sequence has reached its limit
        {"name": "evict-1", "kind": "evict", "code": "i8", "kv_heads": 8, "dim": 128, "block": 32, "sequences": 1, "cached": 9001, "budget": 4096, "first": 4, "last": 512},
        # a batch of long ones
        {"name": "evict-16", "kind": "evict", "code": "e4m3", "kv_heads": 8, "dim": 128, "block": 64, "sequences": 16, "cached": 16 * 16000, "budget": 8000, "first": 4, "last": 1000},
        # one user's answer, drafted by a small model
        {"name": "verify-1", "kind": "verify", "type": "bf16", "sequences": 1, "drafts": 4, "vocab": 128256, "drafted": "model", "temperature": 0.75},
        # a served batch
        {"name": "verify-64", "kind": "verify", "type": "bf16", "sequences": 64, "drafts": 4, "vocab": 128256, "drafted": "model", "temperature": 1.0},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "attend", "evict", "verify"])
    if kind == "verify":
        n = _log(rng, 1, 64)
        return {"kind": kind, "type": rng.choice(["bf16", "bf16", "f32", "f16"]), "sequences": n, "drafts": rng.randint(1, 8 if n < 24 else 4), "vocab": rng.choice([32000, 50257, 128256, 151936 if n < 32 else 999]),
                "drafted": rng.choice(["model", "model", "text"]), "temperature": rng.choice([0.0, 0.5, 0.75, 1.0, 1.25])}
    heads, kv, dim = rng.choice([(32, 8, 128), (32, 8, 128), (32, 8, 64), (8, 2, 256), (24, 8, 64), (16, 16, 80), (40, 8, 128), (28, 4, 128), (16, 1, 96), (12, 3, 192)])
    case = {"kind": kind, "code": rng.choice(["i8", "e4m3"]), "kv_heads": kv, "dim": dim, "block": rng.choice([16, 32, 64])}
    if kind == "evict":
        n = _log(rng, 1, 16)
        mean = _log(rng, 200, 12000)
        budget = max(8, int(mean * rng.uniform(0.2, 0.95)))
        return {**case, "sequences": n, "cached": n * mean, "budget": budget, "first": rng.choice([0, 4, 4]), "last": rng.choice([0, budget // 8, budget // 3])}
    case["type"] = rng.choice(["bf16", "bf16", "bf16", "f32", "f16"])
    if kind == "append":
        n, rows = _log(rng, 1, 64), _log(rng, 1, 8192)
        return {**case, "sequences": min(n, rows), "cached": _log(rng, 1, 60000), "rows": rows}
    case.update(heads=heads, window=rng.choice([0, 0, 0, 128, 1000]), first=rng.choice([0, 4]), cap=rng.choice([0.0, 0.0, 30.0]), weights=rng.choice([0, 0, ALL, 16]))
    shape = rng.choice(["one", "batch", "drafts", "prompt"])
    if shape == "one":
        return {**case, "sequences": 1, "cached": _log(rng, 1, 100000), "rows": 1}
    if shape == "prompt":
        n = rng.randint(1, 4)
        rows = _log(rng, 9 * n, 2048 if case["type"] == "bf16" else 600)
        return {**case, "sequences": n, "cached": _log(rng, 1, 8000), "rows": rows, "weights": min(case["weights"], 64)}
    n = _log(rng, 2, 64)
    return {**case, "sequences": n, "cached": n * _log(rng, 8, 3000), "rows": n * (1 if shape == "batch" else rng.randint(2, 8))}


# ---- inputs -------------------------------------------------------------------------------------------------------------------------------------
def _spread(total, n, g, least):
    """`total` cut into n parts of at least `least`, unlike one another"""
    w = torch.rand(n, generator=g).double() + 0.4
    ends = (w.cumsum(0) / w.sum() * (total - least * n)).round().long().tolist()
    return [b - a + least for a, b in zip([0] + ends[:-1], ends)]


def _lengths(case, seed):
    """Tokens that each sequence has in the cache, and its rows of the pass. Steps and drafts have the same rows for each, prompts their own."""
    g = torch.Generator().manual_seed(seed * 7919 + 13)
    n, rows = case["sequences"], case.get("rows", 0)
    cached = _spread(case["cached"], n, g, 0)
    if rows and rows % n == 0 and rows // n <= 8:
        return cached, [rows // n] * n
    return cached, _spread(rows, n, g, min(1, rows // n)) if rows else [0] * n


def _pages(case, seed):
    """The plan of a pass: tables, lengths, offsets on the device, and the host's numbers."""
    cached, rows = _lengths(case, seed)
    bt, n = case["block"], case["sequences"]
    held = [-(-(c + r) // bt) for c, r in zip(cached, rows)]
    stride, blocks = max(max(held), 1) + 1, (case["cached"] + case.get("rows", 0)) // bt + n + SPARE      # (as many as the lengths can take)
    g = torch.Generator().manual_seed(seed * 104729 + 7)
    order = torch.randperm(blocks, generator=g)
    table = torch.full((n, stride), 0x7FFFFFFF, dtype=torch.int32)      # (no block)
    at = 0
    for i, k in enumerate(held):
        table[i, :k] = order[at:at + k].int()
        at += k
    offsets = torch.tensor([0] + rows).cumsum(0)
    return {"cached": cached, "rows": rows, "blocks": blocks, "stride": stride, "table": table.cuda(), "lengths": torch.tensor(cached, dtype=torch.int32).cuda(), "offsets": offsets.int().cuda(),
            "first": offsets.tolist()}


def _tensors(case, seed):
    """The inputs of a case, from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    kept = TYPES[case.get("type", "bf16")][0]

    def randn(*shape, dtype=F32):
        return torch.randn(*shape, device="cuda", dtype=dtype, generator=g)

    def rand(*shape):
        return torch.rand(*shape, device="cuda", generator=g)

    t = {}
    if case["kind"] == "verify":
        n, k, v = case["sequences"], case["drafts"], case["vocab"]
        target = 3.0 * randn(n, k + 1, v)
        t["uniforms"] = rand(n, k + 1)
        if case["drafted"] == "model":
            draft = target[:, :k] + 0.6 * randn(n, k, v)                 # a smaller model's, near the target's
            t["draft_logits"] = draft.to(kept)
            heat = max(case["temperature"], 0.5)
            t["drafted"] = (draft / heat - torch.log(-torch.log(rand(n, k, v).clamp(1e-20, 1 - 1e-7)))).argmax(2).int()
        else:                                                            # copied from the text: often the likeliest token
            t["drafted"] = torch.where(rand(n, k) < 0.7, target[:, :k].argmax(2), (rand(n, k) * v).long()).int()
            target.scatter_add_(2, t["drafted"].long()[..., None], torch.full((n, k, 1), 6.0, device="cuda"))
        t["target"] = target.to(kept)
        return t
    plan = _pages(case, seed)
    blocks, h, bt, d = plan["blocks"], case["kv_heads"], case["block"], case["dim"]
    loud = torch.exp(0.4 * randn(h, 1, d))                               # keys have channels that are louder than others
    for what, factor in (("key", loud), ("value", 1.0)):
        x = randn(blocks, h, bt, d, dtype=torch.bfloat16).float() * factor
        if case["code"] == "i8":
            t[what + "_codes"] = (x * 24).round_().clamp_(-127, 127).to(torch.int8).view(torch.uint8)
        else:
            t[what + "_codes"] = (x * 60).clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
        t[what + "_scales"] = torch.ldexp(torch.ones(blocks, h, device="cuda"), (rand(blocks, h) * 3).int() - (5 if case["code"] == "i8" else 7))
        del x
    # sums of attention weight: most tokens have little, many have the same
    t["key_weights"] = (-8 * torch.log(rand(blocks, h, bt).clamp_min(1e-9))).round_().div_(16)
    n = (plan["first"][-1] if "rows" in case else 0) + TAIL
    if case["kind"] == "append":
        t["keys"], t["values"] = (randn(h, d) .exp().sqrt() * randn(n, h, d)).reshape(n, h * d).to(kept), randn(n, h * d).to(kept)
    elif case["kind"] == "attend":
        t["query"] = (1.5 * randn(n, case["heads"] * d)).to(kept)
    return t


class _State:
    """What a host program keeps: its buffers, the argument blocks and a command buffer that it encodes into."""

    def __init__(self, case, tensors):
        self.case, self.t, self.handle = case, tensors, None

    def __del__(self):
        if self.handle is not None:
            lib = _ctx().lib
            for call in (lib.uzu_command_buffer_end_encoding, lib.uzu_command_buffer_submit, lib.uzu_command_buffer_wait_until_completed):
                call(self.handle)
            lib.uzu_command_buffer_destroy(self.handle)


_context = None


def _ctx():
    global _context
    if _context is None:
        from uzu_b200 import binding as B
        _context = B.Context(0)
    return _context


def _read_plan(case, plan):
    """What is read back: the rows of the pass with those before them in their first block, or the kept tokens. (first token, rows) of each sequence."""
    if case["kind"] == "append":
        begin = [c // case["block"] * case["block"] for c in plan["cached"]]
        return begin, [c + r - b if r else 0 for c, r, b in zip(plan["cached"], plan["rows"], begin)]
    return [0] * case["sequences"], [min(c, case["budget"]) for c in plan["cached"]]


def _read_bound(case):
    """rows that a read back has at most, whatever the lengths are"""
    return case["rows"] + case["sequences"] * (case["block"] - 1) if case["kind"] == "append" else case["sequences"] * case["budget"]


def prepare(case, seed):
    t = _tensors(case, seed)
    st = _State(case, t)
    k = case["kind"]
    if k == "verify":
        n = case["sequences"]
        t["tokens"] = torch.zeros(n, case["drafts"] + 1, dtype=torch.int32, device="cuda")
        t["accepted"] = torch.zeros(n, dtype=torch.int32, device="cuda")
        if own:
            _arguments(st)
        return st
    plan = st.plan = _pages(case, seed)
    t["table"], t["lengths"], t["offsets"] = plan["table"], plan["lengths"], plan["offsets"]
    if k == "attend":
        t["out"] = torch.zeros_like(t["query"])
    else:
        begin, count = _read_plan(case, plan)
        st.begin, st.count = begin, count
        ends = torch.tensor([0] + count).cumsum(0)
        t["read_lengths"], t["read_offsets"] = torch.tensor(begin, dtype=torch.int32).cuda(), ends.int().cuda()
        st.read_rows = int(ends[-1])
        # 8-bit codes times a power of two are numbers of 16 bits
        t["read_keys"], t["read_values"] = (torch.zeros(_read_bound(case), case["kv_heads"] * case["dim"], dtype=torch.bfloat16, device="cuda") for _ in range(2))
        token = torch.cat([torch.arange(b, b + c) for b, c in zip(begin, count)]).long()
        of = torch.repeat_interleave(torch.arange(case["sequences"]), torch.tensor(count))
        st.read_at = plan["table"].cpu()[of, token // case["block"]].long().cuda(), (token % case["block"]).cuda()
        t["new_lengths"] = torch.zeros(case["sequences"], dtype=torch.int32, device="cuda")
    if k == "evict":
        t["indices"] = torch.zeros(case["sequences"], case["kv_heads"], case["budget"], dtype=torch.int32, device="cuda")
    if k == "append":
        # blocks that take rows: sequence, first token, whether the block is begun
        bt, todo = case["block"], []
        for i, (c, r) in enumerate(zip(plan["cached"], plan["rows"])):
            for b in range(c // bt, -(-(c + r) // bt) if r else c // bt):
                todo.append((i, b, c, r, plan["first"][i]))
        i, b, c, r, first = (torch.tensor(v) for v in zip(*todo))
        token = b[:, None] * bt + torch.arange(bt)[None, :]
        st.new = ((token >= c[:, None]) & (token < (c + r)[:, None])).cuda()
        st.old = (token < c[:, None]).cuda()
        st.row = torch.where(st.new.cpu(), first[:, None] + token - c[:, None], 0).cuda()
        st.block = plan["table"].cpu()[i, b].long().cuda()
    if own:
        _arguments(st)
    return st


def run(st):
    return _own(st) if own else PLAIN[st.case["kind"]](st.case, st, st.t)


# ---- the framework's operators ---------------------------------------------------------------------------------------------------------------------
def _arguments(st):
    import ctypes as C

    from uzu_b200 import binding as B
    c, t, k = st.case, st.t, st.case["kind"]
    kept = TYPES[c.get("type", "bf16")][1]
    lib = _ctx().lib
    p = {n: v.data_ptr() for n, v in t.items()}
    st.calls = []
    if k == "verify":
        args = B.DraftVerifyArgs(target_logits=p["target"], draft_logits=p.get("draft_logits", 0), drafted=p["drafted"], draft_counts=0, uniforms=p["uniforms"], tokens=p["tokens"], accepted=p["accepted"],
                                 sequences=c["sequences"], drafts=c["drafts"], vocab=c["vocab"], target_stride=c["vocab"], draft_stride=c["vocab"], temperature=c["temperature"],
                                 draft_temperature=max(c["temperature"], 0.5), data_type=kept)
        st.calls.append((lib.uzu_draft_verify_encode, args))
    else:
        cache = B.QuantizedCache(key_codes=p["key_codes"], value_codes=p["value_codes"], key_scales=p["key_scales"], value_scales=p["value_scales"], key_weights=p["key_weights"],
                                 blocks=st.plan["blocks"], kv_heads=c["kv_heads"], block_tokens=c["block"], head_dim=c["dim"], code_type=CODES[c["code"]])
        width, longest = c["kv_heads"] * c["dim"], max(a + b for a, b in zip(st.plan["cached"], st.plan["rows"]))

        def sequences(lengths, offsets, rows, most):
            return B.CacheSequences(tables=p["table"], lengths=p[lengths], row_offsets=p[offsets], count=c["sequences"], table_stride=st.plan["stride"], rows=rows, max_rows=most, max_length=max(longest, 1))

        def scratch(args, size):
            args.scratch_bytes = size(_ctx().h, C.byref(args))
            t["scratch"] = torch.zeros(max(16, args.scratch_bytes), dtype=torch.uint8, device="cuda")
            args.scratch = t["scratch"].data_ptr()

        if k == "append":
            st.calls.append((lib.uzu_quantized_cache_append_encode, B.QuantizedCacheAppendArgs(
                cache=cache, sequences=sequences("lengths", "offsets", t["keys"].shape[0], max(st.plan["rows"])), keys=p["keys"], values=p["values"], new_lengths=p["new_lengths"], key_stride=width,
                value_stride=width, data_type=kept)))
        elif k == "attend":
            args = B.QuantizedCacheAttentionArgs(
                cache=cache, sequences=sequences("lengths", "offsets", t["query"].shape[0], max(st.plan["rows"])), query=p["query"], out=p["out"], sinks=0, heads=c["heads"],
                query_row_stride=c["heads"] * c["dim"], query_head_stride=c["dim"], out_stride=c["heads"] * c["dim"], window=c["window"], keep_first=c["first"], weight_rows=c["weights"],
                scale=c["dim"] ** -0.5, softcap=c["cap"], data_type=kept)
            scratch(args, lib.uzu_quantized_cache_attention_scratch_bytes)
            st.calls.append((lib.uzu_quantized_cache_attention_encode, args))
        else:
            args = B.QuantizedCacheEvictArgs(cache=cache, sequences=B.CacheSequences(tables=p["table"], lengths=p["lengths"], count=c["sequences"], table_stride=st.plan["stride"], max_length=longest),
                                             new_lengths=p["new_lengths"], indices=p["indices"], budget=c["budget"], keep_first=c["first"], keep_last=c["last"])
            scratch(args, lib.uzu_quantized_cache_evict_scratch_bytes)
            st.calls.append((lib.uzu_quantized_cache_evict_encode, args))
        if k != "attend":
            st.calls.append((lib.uzu_quantized_cache_read_encode, B.QuantizedCacheReadArgs(
                cache=cache, sequences=sequences("read_lengths", "read_offsets", _read_bound(c), max(max(st.count), 1)), keys=p["read_keys"], values=p["read_values"], key_stride=width,
                value_stride=width, data_type=0)))
    st.refs = [(call, C.byref(args)) for call, args in st.calls]
    h = C.c_void_p()
    B._check(lib.uzu_command_buffer_create(_ctx().h, b"operator", C.byref(h)))
    B._check(lib.uzu_command_buffer_start_encoding(h))
    st.handle = h


OUTPUTS = {"append": ("read_keys", "read_values", "new_lengths"), "attend": ("out", "key_weights"), "evict": ("read_keys", "read_values", "key_weights", "indices", "new_lengths"), "verify": ("tokens", "accepted")}


def _outputs(st):
    return [st.t[n] for n in OUTPUTS[st.case["kind"]] if n != "key_weights" or st.case["kind"] == "evict" or st.case["weights"]]


def _own(st):
    for call, args in st.refs:
        call(st.handle, args)
    return _outputs(st)


# ---- the plain forms ---------------------------------------------------------------------------------------------------------------------------------
def _values(codes, code):
    return codes.view(torch.int8 if code == "i8" else torch.float8_e4m3fn).float()


def _round(x, code):
    """32-bit numbers within the codes' range, as codes"""
    return (torch.round(x).to(torch.int8) if code == "i8" else x.to(torch.float8_e4m3fn)).view(torch.uint8)


def _scale(most, code):
    """the smallest power of two that brings `most` into the codes' range; 0 for 0"""
    f, e = torch.frexp(most)
    e = e - 7 + (f > 127 / 128).int() if code == "i8" else e - 9 + (f > 0.875).int()
    return torch.where(most > 0, torch.ldexp(torch.ones_like(most), e.clamp_min(-100)), 0.0)


def _inverse(scale):
    return torch.where(scale > 0, 1 / scale.clamp_min(2.0 ** -100), 0.0)


def _plain_read(c, st, t):
    block, at = st.read_at
    for what in ("key", "value"):
        x = _values(t[what + "_codes"][block, :, at], c["code"]) * t[what + "_scales"][block][..., None]
        t["read_" + what + "s"][:st.read_rows] = x.reshape(st.read_rows, -1).to(torch.bfloat16)


def _plain_append(c, st, t):
    h, d, code = c["kv_heads"], c["dim"], c["code"]
    for what in ("key", "value"):
        codes, scales = t[what + "_codes"], t[what + "_scales"]
        x = torch.where(st.new[..., None, None], t[what + "s"][st.row].float().reshape(*st.row.shape, h, d), 0.0).transpose(1, 2)      # [blocks, heads, tokens, dim]
        begun = st.old[:, :1]
        old = torch.where(begun, scales[st.block], 0.0)
        scale = torch.maximum(old, _scale(x.abs().amax((2, 3)), code))
        inverse = _inverse(scale)[..., None, None]
        was = codes[st.block]
        again = _round(_values(was, code).nan_to_num() * (old[..., None, None] * inverse), code)
        codes[st.block] = torch.where(st.new[:, None, :, None], _round(x * inverse, code), torch.where(st.old[:, None, :, None], again, was))
        scales[st.block] = scale
    weights = t["key_weights"][st.block]
    t["key_weights"][st.block] = torch.where(st.new[:, None], 0.0, weights)
    t["new_lengths"].copy_(t["lengths"] + t["offsets"].diff())
    _plain_read(c, st, t)
    return _outputs(st)


def _plain_attend(c, st, t):
    g, d, bt = c["kv_heads"], c["dim"], c["block"]
    per, kept = c["heads"] // g, t["out"].dtype
    cached, rows, first = st.plan["cached"], st.plan["rows"], st.plan["first"]
    n = len(rows)
    # sequences of few rows side by side, others one by one, some rows at a time
    few = max(rows) * per <= 64
    for ids in ([list(range(n))] if few else [[i] for i in range(n)]):
        longest, most = max(cached[i] + rows[i] for i in ids), max(rows[i] for i in ids)
        if not most:
            continue
        blocks = -(-longest // bt)
        table = t["table"][ids][:, :blocks].long()
        there = table < st.plan["blocks"]
        table = torch.where(there, table, 0)
        k, v = (_values(t[w + "_codes"][table], c["code"]).nan_to_num() * t[w + "_scales"][table][..., None, None] for w in ("key", "value"))      # [n, blocks, g, bt, d]
        k, v = (x.transpose(1, 2).reshape(len(ids), g, blocks * bt, d) for x in (k, v))
        length, m, start = (torch.tensor([x[i] for i in ids], device="cuda")[:, None] for x in (cached, rows, first))
        j = torch.arange(blocks * bt, device="cuda")
        step = most if few else max(1, (1 << 28) // (c["heads"] * blocks * bt))
        for begin in range(0, most, step):
            row = torch.arange(begin, min(begin + step, most), device="cuda")[None, :]
            live = row < m
            at = torch.where(live, start + row, 0)
            q = t["query"][at].float().reshape(len(ids), row.shape[1], g, per, d)
            s = torch.einsum("nrgpd,ngjd->ngprj", q, k) * d ** -0.5
            if c["cap"]:
                s = c["cap"] * torch.tanh(s / c["cap"])
            index = (length + row)[..., None]
            seen = (j <= index) & live[..., None]
            if c["window"]:
                seen &= (index - j < c["window"]) | (j < c["first"])
            seen = seen[:, None, None]
            s = torch.where(seen, s, -math.inf)
            s = torch.exp(s - s.amax(-1, keepdim=True).clamp_min(-1e30))
            s = torch.where(seen, s / s.sum(-1, keepdim=True).clamp_min(1e-30), 0.0)
            o = torch.einsum("ngprj,ngjd->nrgpd", s, v).reshape(len(ids), row.shape[1], -1)
            t["out"][at[live]] = o[live].to(kept)
            if c["weights"]:
                last = (row >= m - min(c["weights"], most)) & live
                w = (s * last[:, None, None, :, None]).sum((2, 3)).reshape(len(ids), g, blocks, bt).transpose(1, 2)
                t["key_weights"].index_put_((table[there],), w[there], accumulate=True)
            del s
    return _outputs(st)


def _plain_evict(c, st, t):
    g, d, bt, budget, code = c["kv_heads"], c["dim"], c["block"], c["budget"], c["code"]
    t["new_lengths"].copy_(t["lengths"].clamp_max(budget))
    t["indices"].fill_(-1)
    for i, length in enumerate(st.plan["cached"]):
        if length <= budget:
            t["indices"][i, :, :length] = torch.arange(length, device="cuda", dtype=torch.int32)
            continue
        table = t["table"][i, :-(-length // bt)].long()
        w = t["key_weights"][table].transpose(0, 1).reshape(g, -1)[:, :length].clone()
        w[:, :c["first"]] = math.inf
        w[:, length - c["last"]:] = math.inf
        keep = torch.sort(torch.sort(w, dim=1, descending=True, stable=True)[1][:, :budget], dim=1)[0]            # [g, budget]
        t["indices"][i] = keep
        block, at, head = table[keep // bt], keep % bt, torch.arange(g, device="cuda")[:, None]
        blocks = -(-budget // bt)
        live = (torch.arange(blocks * bt, device="cuda") < budget).reshape(1, blocks, bt)
        weights = t["key_weights"][block, head, at]
        to = table[:blocks]

        def filled(x):
            return torch.nn.functional.pad(x, [0, 0] * (x.dim() - 2) + [0, blocks * bt - budget]).reshape(g, blocks, bt, *x.shape[2:])

        for what in ("key", "value"):
            codes, scales = t[what + "_codes"], t[what + "_scales"]
            x = filled(_values(codes[block, head, at], code) * scales[block, head][..., None])
            scale = _scale(x.abs().amax((2, 3)), code)
            codes[to] = torch.where(live[..., None], _round(x * _inverse(scale)[..., None, None], code), codes[to].transpose(0, 1)).transpose(0, 1)
            scales[to] = scale.T
        t["key_weights"][to] = torch.where(live, filled(weights), t["key_weights"][to].transpose(0, 1)).transpose(0, 1)
    _plain_read(c, st, t)
    return _outputs(st)


def _plain_verify(c, st, t):
    n, k, v = c["sequences"], c["drafts"], c["vocab"]
    drafted = t["drafted"].long()
    if c["temperature"] == 0:
        best = t["target"].float().argmax(2)
        wrong = best[:, :k] != drafted
        count = torch.where(wrong.any(1), wrong.int().argmax(1), k)
        token = torch.gather(best, 1, count[:, None])[:, 0]
    else:
        def weights(logits, heat, kind):
            x = logits.to(kind)
            return torch.exp((x - x.amax(-1, keepdim=True)) / heat)

        w = weights(t["target"], c["temperature"], F32)
        p = torch.gather(w[:, :k], 2, drafted[..., None])[..., 0] / w[:, :k].sum(2)
        q = torch.ones_like(p)
        if "draft_logits" in t:
            w = weights(t["draft_logits"], max(c["temperature"], 0.5), F32)
            q = torch.gather(w, 2, drafted[..., None])[..., 0] / w.sum(2)
        del w
        refused = ~(t["uniforms"][:, :k] * q < p)
        count = torch.where(refused.any(1), refused.int().argmax(1), k)
        # the token behind, in 64 bits: the border between two tokens depends on a sum over the vocabulary
        seq, at = torch.arange(n, device="cuda"), count.clamp_max(k - 1)
        r = weights(t["target"][seq, count], c["temperature"], F64)
        r = r / r.sum(1, keepdim=True)
        if "draft_logits" in t:
            q = weights(t["draft_logits"][seq, at], max(c["temperature"], 0.5), F64)
            q = q / q.sum(1, keepdim=True)
        else:
            q = torch.zeros_like(r).scatter_(1, drafted[seq, at][:, None], 1.0)
        r = torch.where((count < k)[:, None], (r - q).clamp_min(0.0), r)
        sums = r.cumsum(1)
        aim = t["uniforms"][:, k].double()[:, None] * sums[:, -1:]
        token = (sums <= aim).sum(1).clamp_max(v - 1)
    place = torch.arange(k + 1, device="cuda")[None, :]
    tokens = torch.where(place < count[:, None], torch.nn.functional.pad(drafted, (0, 1)), torch.where(place == count[:, None], token[:, None], -1))
    t["tokens"].copy_(tokens)
    t["accepted"].copy_(count)
    return _outputs(st)


PLAIN = {"append": _plain_append, "attend": _plain_attend, "evict": _plain_evict, "verify": _plain_verify}


# ---- what a pass cannot do without -------------------------------------------------------------------------------------------------------------------
def work(case):
    k, n = case["kind"], case["sequences"]
    e = 4 if case.get("type") == "f32" else 2
    if k == "verify":
        rows = (case["drafts"] + 1) * n
        read = rows + (case["drafts"] * n if case["drafted"] == "model" and case["temperature"] else 0)
        return {"bytes": read * case["vocab"] * e + rows * 12, "flops": 4 * read * case["vocab"]}
    g, d = case["kv_heads"], case["dim"]
    token = 2 * g * (d + 4 / case["block"])                              # codes and scales of a token's keys and values
    if k == "append":
        rows = case["rows"]
        # rows read, codes written; codes read back with those before them in their first block, numbers written
        back = rows + min(n * (case["block"] - 1) / 2, case["cached"])
        return {"bytes": rows * (2 * g * d * e + token + 4 * g) + back * (token + 2 * g * d * 2), "flops": 4 * rows * g * d}
    if k == "evict":
        kept = min(case["cached"], n * case["budget"])
        return {"bytes": case["cached"] * g * 4 + kept * (2 * token + g * 12) + kept * (token + 2 * g * d * 2), "flops": kept * 4 * g * d}
    rows, cached = case["rows"], case["cached"] / n
    mine = rows / n
    seen = cached + (mine + 1) / 2                                       # of a row, on average
    if case["window"]:
        seen = min(seen, case["window"] + case["first"])
    tokens = min(cached + mine, seen + mine) * n
    summed = min(case["weights"], mine) * n
    return {"bytes": tokens * (token + (8 * g if case["weights"] else 0)) + 2 * rows * case["heads"] * d * e, "flops": case["heads"] * seen * (rows * 4 * d + summed)}


# ---- in 64 bits, from the definitions ----------------------------------------------------------------------------------------------------------------
def _stands_for(codes, code):
    return codes.view(torch.int8).double() if code == "i8" else codes.view(torch.float8_e4m3fn).double()


def _step_of(x, code):
    """the smallest power of two s with |x| <= LARGEST s for all of x, from 2^-100 on"""
    most = float(x.abs().max()) if x.numel() else 0.0
    if most == 0:
        return 0.0
    s = 2.0 ** -100
    e = max(-100, math.ceil(math.log2(most / LARGEST[code])) - 2)
    s = 2.0 ** e
    while LARGEST[code] * s < most:
        s *= 2
    return s


def _coded(x, s, code):
    """x to the nearest code times s, ties to even"""
    if s == 0:
        return torch.zeros_like(x)
    y = x / s
    if code == "i8":
        return torch.round(y) * s
    quantum = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(y / quantum) * quantum * s


def exact(case, seed):
    t = _tensors(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "evict": _exact_evict, "verify": _exact_verify}[case["kind"]](case, seed, t)


def _exact_append(c, seed, t):
    plan, bt, g, d = _pages(c, seed), c["block"], c["kv_heads"], c["dim"]
    begin, count = _read_plan(c, plan)
    if sum(-(-n // bt) for n in count) * g > 6000:
        return None
    out = [torch.zeros(_read_bound(c), g * d, dtype=F64, device="cuda") for _ in range(2)]
    at = 0
    for i, (b0, n) in enumerate(zip(begin, count)):
        have, row = plan["cached"][i], plan["first"][i]
        for b in range(b0 // bt, -(-(b0 + n) // bt) if n else b0 // bt):
            block = int(plan["table"][i, b])
            lo, hi = b * bt, min((b + 1) * bt, b0 + n)
            olds = max(0, min(have - lo, hi - lo))
            for o, what in zip(out, ("key", "value")):
                rows = t[what + "s"][row + lo + olds - have:row + hi - have].double().reshape(-1, g, d)
                for h in range(g):
                    was = float(t[what + "_scales"][block, h]) if olds else 0.0
                    old = _stands_for(t[what + "_codes"][block, h, :olds], c["code"]) * was
                    s = max(was, _step_of(rows[:, h], c["code"]))
                    o[at + lo - b0:at + hi - b0, h * d:(h + 1) * d] = torch.cat([_coded(old, s, c["code"]), _coded(rows[:, h], s, c["code"])])
        at += n
    return [*out, torch.tensor([a + b for a, b in zip(plan["cached"], plan["rows"])], dtype=torch.int32, device="cuda")]


def _exact_attend(c, seed, t):
    plan, bt, g, d = _pages(c, seed), c["block"], c["kv_heads"], c["dim"]
    per = c["heads"] // g
    out, sums = torch.zeros(t["query"].shape, dtype=F64, device="cuda"), t["key_weights"].double()
    for i, (cached, m, first) in enumerate(zip(plan["cached"], plan["rows"], plan["first"])):
        if not m:
            continue
        length = cached + m
        j = torch.arange(length, device="cuda")
        block, at = plan["table"][i].long()[j // bt], j % bt
        for h in range(g):
            k, v = (_stands_for(t[w + "_codes"][block, h, at], c["code"]) * t[w + "_scales"][block, h].double()[:, None] for w in ("key", "value"))
            for r0 in range(0, m, 256):
                r = torch.arange(r0, min(r0 + 256, m), device="cuda")
                index = (cached + r)[:, None]
                hide = j[None, :] > index
                if c["window"]:
                    hide |= (index - j >= c["window"]) & (j >= c["first"])
                q = t["query"][first + r].double().reshape(len(r), c["heads"], d)[:, h * per:(h + 1) * per]
                s = torch.matmul(q.transpose(0, 1), k.T) / math.sqrt(d)
                if c["cap"]:
                    s = torch.tanh(s / c["cap"]) * c["cap"]
                s = torch.softmax(s.masked_fill(hide, -math.inf), -1)
                out[first + r, h * per * d:(h + 1) * per * d] = torch.matmul(s, v).transpose(0, 1).reshape(len(r), per * d)
                mine = r >= m - min(c["weights"], m)
                sums[block, h, at] += s[:, mine].sum((0, 1))
    return [out, sums] if c["weights"] else [out]


def _exact_evict(c, seed, t):
    plan, bt, g, d, budget = _pages(c, seed), c["block"], c["kv_heads"], c["dim"], c["budget"]
    kept = [min(n, budget) for n in plan["cached"]]
    if sum(-(-n // bt) for n in kept) * g > 6000:
        return None
    out = [torch.zeros(_read_bound(c), g * d, dtype=F64, device="cuda") for _ in range(2)]
    weights, indices = t["key_weights"].double(), torch.full((c["sequences"], g, budget), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(plan["cached"]):
        j = torch.arange(n, device="cuda")
        block, place = plan["table"][i].long()[j // bt], j % bt
        for h in range(g):
            w = t["key_weights"][block, h, place].cpu().tolist()
            middle = range(c["first"], n - c["last"])
            best = sorted(middle, key=lambda a: (-w[a], a))[:max(0, budget - c["first"] - c["last"])]
            keep = sorted(best + list(range(c["first"])) + list(range(n - c["last"], n))) if n > budget else list(range(n))
            indices[i, h, :len(keep)] = torch.tensor(keep, dtype=torch.int32)
            from_ = torch.tensor(keep, device="cuda", dtype=torch.long)
            if n > budget:
                weights[block[:budget], h, place[:budget]] = t["key_weights"][block[from_], h, place[from_]].double()
            for o, what in zip(out, ("key", "value")):
                x = _stands_for(t[what + "_codes"][block[from_], h, place[from_]], c["code"]) * t[what + "_scales"][block[from_], h].double()[:, None]
                if n > budget:
                    x = torch.cat([_coded(p, _step_of(p, c["code"]), c["code"]) for p in x.split(bt)])
                o[at:at + len(keep), h * d:(h + 1) * d] = x
        at += kept[i]
    return [*out, weights, indices.cuda(), torch.tensor(kept, dtype=torch.int32, device="cuda")]


def _exact_verify(c, seed, t):
    n, k, v = c["sequences"], c["drafts"], c["vocab"]
    tokens, accepted = torch.full((n, k + 1), -1, dtype=torch.int32), torch.zeros(n, dtype=torch.int32)
    heat = c["temperature"]
    for i in range(n):
        drafted, u = t["drafted"][i].tolist(), t["uniforms"][i].tolist()
        for a in range(k + 1):
            row = t["target"][i, a].double()
            if heat == 0:
                token = int((row == row.max()).nonzero()[0])
                if a < k and token == drafted[a]:
                    tokens[i, a] = token
                    continue
            else:
                p = torch.softmax(row / heat, 0)
                if a < k:
                    q = torch.softmax(t["draft_logits"][i, a].double() / max(heat, 0.5), 0) if "draft_logits" in t else torch.nn.functional.one_hot(torch.tensor(drafted[a], device="cuda"), v).double()
                    if u[a] * float(q[drafted[a]]) < float(p[drafted[a]]):
                        tokens[i, a] = drafted[a]
                        continue
                    p = torch.relu(p - q)
                sums = p.cumsum(0)
                token = min(v - 1, int(torch.searchsorted(sums, u[k] * sums[-1:], right=True)))
            tokens[i, a], accepted[i] = token, a
            break
    return [tokens.cuda(), accepted.cuda()]
