"""The operators of a state space mixer and of the routed experts behind it, as measured cases.

  conv     the short causal convolution over the packed rows of a pass's sequences, its last inputs kept per slot
  scan     the selective state space scan over packed rows: one decay per head and token, state carried in and out per slot
  step     one token of each running sequence through convolution, scan and gate
  experts  a whole layer of routed experts for a few tokens: router, chosen experts, shared experts, weighted sum

A pass goes through the entry points of `uzu_b200.binding` (a command buffer that the state keeps open, as a host program that brings its own
graph encodes into it), or through elementary torch operations that say the same.
"""
from __future__ import annotations

import math

import torch

own = False

F32, F64 = torch.float32, torch.float64
TYPES = {"bf16": (torch.bfloat16, 0), "f32": (torch.float32, 1), "f16": (torch.float16, 2)}
TAIL = 3          # rows behind the last sequence: of a padded pass, left as they are


def listed():
    return [
        # a short turn in a running chat: latency counts
        {"name": "conv-turn", "kind": "conv", "type": "bf16", "channels": 4352, "taps": 4, "sequences": 1, "rows": 37},
        # sixteen prompts of different lengths in one pass, a wide model
        {"name": "conv-packed", "kind": "conv", "type": "bf16", "channels": 10240, "taps": 4, "sequences": 16, "rows": 16384},
        # a short turn
        {"name": "scan-turn", "kind": "scan", "type": "bf16", "heads": 64, "groups": 1, "dim": 64, "state": 128, "sequences": 1, "rows": 200},
        # several prompts, ragged
        {"name": "scan-packed", "kind": "scan", "type": "bf16", "heads": 64, "groups": 1, "dim": 64, "state": 128, "sequences": 9, "rows": 8192},
        # one long document on a wide model
        {"name": "scan-long", "kind": "scan", "type": "bf16", "heads": 128, "groups": 8, "dim": 64, "state": 128, "sequences": 1, "rows": 16384},
        # a small model kept in 32 bits, an odd length and a small state
        {"name": "scan-f32", "kind": "scan", "type": "f32", "heads": 24, "groups": 1, "dim": 64, "state": 64, "sequences": 2, "rows": 1001},
        # one user's answer
        {"name": "step-1", "kind": "step", "type": "bf16", "heads": 64, "groups": 1, "dim": 64, "state": 128, "taps": 4, "rows": 1},
        # a served batch
        {"name": "step-64", "kind": "step", "type": "bf16", "heads": 80, "groups": 1, "dim": 64, "state": 128, "taps": 4, "rows": 64},
        # a large batch on a wide model
        {"name": "step-256", "kind": "step", "type": "bf16", "heads": 128, "groups": 8, "dim": 64, "state": 128, "taps": 4, "rows": 256},
        # one decoded token of a model with few large experts
        {"name": "experts-1", "kind": "experts", "type": "bf16", "width": 4096, "ff": 14336, "experts": 8, "top": 2, "shared": 0, "score": "chosen", "rows": 1},
        # a small batch, many small experts and two shared ones
        {"name": "experts-16", "kind": "experts", "type": "bf16", "width": 2048, "ff": 1408, "experts": 64, "top": 6, "shared": 2, "score": "all", "rows": 16},
        # a batch on f32 rows, nearly every expert is chosen by some token
        {"name": "experts-48-f32", "kind": "experts", "type": "f32", "width": 2048, "ff": 768, "experts": 128, "top": 8, "shared": 0, "score": "sigmoid", "rows": 48},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(["conv", "scan", "scan", "step", "experts"])
    kept = rng.choice(["bf16", "bf16", "bf16", "f32", "f16"])
    if kind == "conv":
        rows = _log(rng, 1, 16384)
        return {"kind": kind, "type": kept, "channels": rng.choice([512, 1536 + 7, 2304, 4352, 6144]), "taps": rng.choice([2, 3, 4, 4, 4, 7]), "sequences": rng.randint(1, min(rows, 24)), "rows": rows}
    if kind == "scan":
        heads, groups = rng.choice([(8, 1), (40, 1), (32, 2), (64, 1), (64, 8), (80, 1), (128, 8)])
        dim, state = rng.choice([(64, 128), (64, 128), (64, 128), (64, 64), (128, 128), (32, 16), (64, 40), (80, 64)])
        rows = min(_log(rng, 1, 12000), 16384 * 128 * 64 // (heads * dim) // 2)
        return {"kind": kind, "type": kept, "heads": heads, "groups": groups, "dim": dim, "state": state, "sequences": rng.randint(1, min(rows, 8)), "rows": rows}
    if kind == "step":
        heads, groups = rng.choice([(8, 1), (40, 1), (32, 2), (64, 1), (64, 8), (80, 1), (128, 8)])
        dim, state = rng.choice([(64, 128), (64, 128), (64, 64), (128, 128), (32, 16), (64, 40)])
        return {"kind": kind, "type": kept, "heads": heads, "groups": groups, "dim": dim, "state": state, "taps": rng.choice([2, 4, 4, 4]), "rows": min(_log(rng, 1, 256), 256 * 128 * 64 // (heads * dim))}
    width, ff, experts, top, shared = rng.choice([(4096, 14336, 8, 2, 0), (2048, 1408, 64, 6, 2), (2048, 768, 128, 8, 0), (1024, 512, 32, 8, 0), (1536, 1000, 16, 1, 1)])
    return {"kind": kind, "type": rng.choice(["bf16", "bf16", "f32"]), "width": width, "ff": ff, "experts": experts, "top": top, "shared": shared,
            "score": rng.choice(["chosen", "all", "sigmoid"]), "rows": _log(rng, 1, 4 if width == 4096 else 64)}


def _lengths(case, seed):
    """Rows of each sequence, the first row of each, its slot and whether it starts from nothing: spread around the mean, the sum as the case says."""
    g = torch.Generator().manual_seed(seed * 7919 + 13)
    n, rows = case["sequences"], case["rows"]
    w = (torch.rand(n, generator=g) + 0.3).cumsum(0)
    ends = [int(round(float(v) * rows / float(w[-1]))) for v in w]
    ends[-1] = rows
    first = [0] + ends[:-1]
    slots = torch.randperm(n + 2, generator=g)[:n].tolist()
    fresh = [(i + seed) % 3 == 0 and n > 1 for i in range(n)]
    return [(a, b - a, s, int(f)) for a, b, s, f in zip(first, ends, slots, fresh)]


def _channels(case):
    return case["heads"] * case["dim"] + 2 * case["groups"] * case["state"]


def _parameters(case, randn, rand):
    """Decay rates of 1 .. 16, step sizes of 0.001 .. 0.1, as trained mixers have them."""
    h = case["heads"]
    size = torch.exp(math.log(1e-3) + rand(h) * (math.log(0.1) - math.log(1e-3)))
    return {"a": -(1 + 15 * rand(h)), "d": 1 + 0.2 * randn(h), "dt_bias": size + torch.log(-torch.expm1(-size))}


def _tensors(case, seed):
    """The inputs of a case, from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    kept = TYPES[case["type"]][0]

    def randn(*shape, dtype=F32):
        return torch.randn(*shape, device="cuda", dtype=dtype, generator=g)

    def rand(*shape):
        return torch.rand(*shape, device="cuda", generator=g)

    k, t = case["kind"], {}
    if k == "conv":
        n, ch, taps = case["rows"] + TAIL, case["channels"], case["taps"]
        t["input"] = randn(n, ch).to(kept)
        t["weights"] = randn(ch, taps) / math.sqrt(taps)
        t["bias"] = 0.1 * randn(ch)
        t["state"] = randn(case["sequences"] + 2, taps - 1, ch).to(kept)
    elif k in ("scan", "step"):
        h, p, s = case["heads"], case["dim"], case["state"]
        n, ch, inner = case["rows"] + (TAIL if k == "scan" else 0), _channels(case), h * p
        # the input projection's row: gate, what the convolution takes, step sizes
        proj = randn(n, inner + ch + h, dtype=F32 if kept == F32 else kept)
        proj[:, inner + ch:] *= 0.5
        t["proj"] = proj
        t.update(_parameters(case, randn, rand))
        slots = case["sequences"] + 2 if k == "scan" else case["rows"] + 2
        t["state"] = 0.3 * randn(slots, h, p, s)
        if k == "scan":
            xbc = randn(n, ch, dtype=F32)
            t["xbc"] = (xbc * torch.sigmoid(xbc)).to(kept)
        else:
            t["weights"] = randn(ch, case["taps"]) / math.sqrt(case["taps"])
            t["bias"] = 0.1 * randn(ch)
            t["conv_state"] = randn(slots, case["taps"] - 1, ch).to(kept)
            order = torch.randperm(slots, device="cuda", generator=g)[:case["rows"]]
            if case["rows"] > 4:
                order[case["rows"] // 2] = -1      # a row of a padded batch
            t["slots"] = order.to(torch.int32)
    else:
        w, f, e = case["width"], case["ff"], case["experts"] + case["shared"]
        t["x"] = randn(case["rows"], w).to(kept)
        t["router"] = (randn(case["experts"], w) / math.sqrt(w)).to(torch.bfloat16)
        t["router_bias"] = 0.1 * randn(case["experts"])
        t["up_gate"] = randn(e, 2 * f, w, dtype=torch.bfloat16).div_(math.sqrt(w))
        t["down"] = randn(e, w, f, dtype=torch.bfloat16).div_(math.sqrt(f))
    return t


class _State:
    """What a host program keeps: its buffers, the argument block and a command buffer that it encodes into."""

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


def prepare(case, seed):
    t = _tensors(case, seed)
    st = _State(case, t)
    k = case["kind"]
    if k in ("conv", "scan"):
        st.sequences = _lengths(case, seed)
        longest = max(n for _, n, _, _ in st.sequences)
        at = torch.arange(longest)[None, :]
        first, n, slot, fresh = (torch.tensor(v)[:, None] for v in zip(*st.sequences))
        st.valid = (at < n).cuda()
        st.index = torch.where(at < n, first + at, 0).cuda()
        st.slot, st.fresh, st.n = slot[:, 0].cuda(), (fresh[:, 0] != 0).cuda(), n[:, 0].cuda()
    if k == "conv":
        t["out"] = torch.zeros_like(t["input"])
    elif k == "experts":
        t["out"] = torch.zeros_like(t["x"])
        t["ids"] = torch.zeros(case["rows"], case["top"], dtype=torch.int32, device="cuda")
        t["weights"] = torch.zeros(case["rows"], case["top"], device="cuda")
    else:
        t["out"] = torch.zeros(t["proj"].shape[0], case["heads"] * case["dim"], dtype=TYPES[case["type"]][0], device="cuda")
        if k == "step":
            st.live = torch.nonzero(t["slots"] >= 0)[:, 0]
    if own:
        _arguments(st)
    return st


def run(st):
    return _own(st) if own else PLAIN[st.case["kind"]](st.case, st, st.t)


# ---- the framework's operators ---------------------------------------------------------------------------------------------------------------
def _arguments(st):
    import ctypes as C

    from uzu_b200 import binding as B
    c, t, k = st.case, st.t, st.case["kind"]
    kept = TYPES[c["type"]][1]
    lib = _ctx().lib
    p = {n: v.data_ptr() for n, v in t.items()}
    if k in ("conv", "scan"):
        st.host = (B.RowSequence * len(st.sequences))(*[B.RowSequence(first_row=a, rows=n, slot=s, fresh=f) for a, n, s, f in st.sequences])
        packed = dict(sequences=C.addressof(st.host), sequence_count=len(st.sequences), rows=c["rows"] + TAIL, slots=c["sequences"] + 2, data_type=kept)
    if k == "conv":
        args = B.CausalConvArgs(input=p["input"], weights=p["weights"], bias=p["bias"], output=p["out"], state=p["state"], channels=c["channels"], taps=c["taps"],
                                input_stride=c["channels"], output_stride=c["channels"], activation=B.ACT_SILU, **packed)
        st.call = lib.uzu_causal_conv_encode
    elif k == "experts":
        args = B.ExpertLayerArgs(x=p["x"], router=p["router"], router_bias=p["router_bias"], up_gate=p["up_gate"], down=p["down"], out=p["out"], ids=p["ids"], weights=p["weights"],
                                 rows=c["rows"], width=c["width"], ff=c["ff"], experts=c["experts"], top=c["top"], shared=c["shared"], x_stride=c["width"], out_stride=c["width"],
                                 score={"chosen": 0, "all": 1, "sigmoid": 2}[c["score"]], renormalise=int(c["score"] == "sigmoid"), weight_scale=1.0, activation=B.ACT_SILU, data_type=kept)
        st.call = lib.uzu_expert_layer_encode
        args.scratch_bytes = lib.uzu_expert_layer_scratch_bytes(C.byref(args))
    else:
        e = t["proj"].element_size()
        h, inner, gs, ch = c["heads"], c["heads"] * c["dim"], c["groups"] * c["state"], _channels(c)
        row = inner + ch + h
        common = dict(dt=p["proj"] + (inner + ch) * e, z=p["proj"], a=p["a"], d=p["d"], dt_bias=p["dt_bias"], state=p["state"], out=p["out"], heads=h, groups=c["groups"], head_dim=c["dim"],
                      state_size=c["state"], dt_stride=row, z_stride=row, out_stride=inner, dt_min=0.0, dt_max=float("inf"), dt_softplus=1)
        if k == "scan":
            args = B.StateSpaceScanArgs(x=p["xbc"], b=p["xbc"] + inner * e, c=p["xbc"] + (inner + gs) * e, x_stride=ch, b_stride=ch, c_stride=ch, **common, **packed)
            st.call = lib.uzu_state_space_scan_encode
            args.scratch_bytes = lib.uzu_state_space_scan_scratch_bytes(_ctx().h, C.byref(args))
        else:
            t["tickets"] = torch.zeros(c["rows"] * c["groups"], dtype=torch.int32, device="cuda")
            args = B.StateSpaceStepArgs(xbc=p["proj"] + inner * e, conv_weights=p["weights"], conv_bias=p["bias"], conv_state=p["conv_state"], slots=p["slots"], tickets=t["tickets"].data_ptr(),
                                        rows=c["rows"], slot_count=c["rows"] + 2, taps=c["taps"], xbc_stride=row, activation=B.ACT_SILU, data_type=kept, **common)
            st.call = lib.uzu_state_space_step_encode
    if k in ("scan", "experts"):
        t["scratch"] = torch.zeros(max(16, args.scratch_bytes), dtype=torch.uint8, device="cuda")
        args.scratch = t["scratch"].data_ptr()
    st.args, st.ref = args, C.byref(args)
    h = C.c_void_p()
    B._check(lib.uzu_command_buffer_create(_ctx().h, b"operator", C.byref(h)))
    B._check(lib.uzu_command_buffer_start_encoding(h))
    st.handle = h


def _own(st):
    st.call(st.handle, st.ref)
    t = st.t
    return [t[n] for n in {"conv": ("out", "state"), "scan": ("out", "state"), "step": ("out", "conv_state", "state"), "experts": ("out", "ids", "weights")}[st.case["kind"]]]


# ---- the plain forms ---------------------------------------------------------------------------------------------------------------------------
def _silu(x):
    return x / (1 + torch.exp(-x))


def _softplus(x):
    return torch.where(x > 20, x, torch.log1p(torch.exp(torch.clamp(x, max=20.0))))


def _plain_conv(c, st, t):
    taps, kept = c["taps"], t["input"].dtype
    old = torch.where(st.fresh[:, None, None], 0.0, t["state"][st.slot].float())
    u = torch.where(st.valid[..., None], t["input"][st.index].float(), 0.0)
    u = torch.cat([old, u], 1)                                                      # [sequences, taps - 1 + longest, channels]
    y = torch.einsum("nltc,ct->nlc", u.unfold(1, taps, 1).transpose(2, 3), t["weights"]) + t["bias"]
    t["out"][st.index[st.valid]] = _silu(y)[st.valid].to(kept)
    last = st.n[:, None] + torch.arange(taps - 1, device="cuda")[None, :]
    t["state"][st.slot] = torch.gather(u, 1, last[..., None].expand(-1, -1, u.shape[2])).to(kept)
    return [t["out"], t["state"]]


def _plain_scan(c, st, t):
    h, p, s, g = c["heads"], c["dim"], c["state"], c["groups"]
    inner, ch = h * p, _channels(c)
    n, longest = st.valid.shape
    q = 256 if longest > 256 else max(1, longest)
    chunks = -(-longest // q)
    valid = torch.nn.functional.pad(st.valid, (0, chunks * q - longest))
    index = torch.nn.functional.pad(st.index, (0, chunks * q - longest))

    def rows(v, *shape):
        return torch.where(valid.reshape(n, chunks * q, *[1] * len(shape)), v[index].reshape(n, chunks * q, *shape).float(), 0.0).reshape(n, chunks, q, *shape)

    x = rows(t["xbc"][:, :inner], h, p)
    b, cc = rows(t["xbc"][:, inner:inner + g * s], g, s), rows(t["xbc"][:, inner + g * s:], g, s)
    dt = torch.where(valid.reshape(n, chunks, q, 1), _softplus(rows(t["proj"][:, inner + ch:], h) + t["dt_bias"]), 0.0)
    steps = dt.double() * t["a"].double()
    sums = steps.cumsum(2)                                                           # logarithms of the decays, from the chunk's start on
    whole = sums[:, :, -1]
    scores = torch.einsum("ncigs,ncjgs->ncgij", cc, b)
    seen = torch.ones(q, q, dtype=torch.bool, device="cuda").tril()
    logs = sums.permute(0, 1, 3, 2)
    decay = torch.where(seen, torch.exp((logs[..., :, None] - logs[..., None, :]).float()), 0.0)
    weights = (decay.reshape(n, chunks, g, h // g, q, q) * scores[:, :, :, None]).reshape(n, chunks, h, q, q)
    del decay, scores
    xd = x * dt[..., None]
    y = torch.einsum("nchij,ncjhp->ncihp", weights, xd)
    del weights
    to_end = torch.exp((whole[:, :, None] - sums).float())
    added = torch.einsum("ncjgs,ncjgkp->ncgkps", b, (xd * to_end[..., None]).reshape(n, chunks, q, g, h // g, p)).reshape(n, chunks, h, p, s)
    start = torch.where(st.fresh[:, None, None, None], 0.0, t["state"][st.slot])
    parts = torch.cat([start[:, None], added], 1)                                    # the state at a chunk's start: those before it, decayed
    ends = torch.nn.functional.pad(whole.cumsum(1), (0, 0, 1, 0))
    between = ends[:, :, None] - ends[:, None, :]
    between = torch.where(torch.ones(chunks + 1, chunks + 1, dtype=torch.bool, device="cuda").tril()[None, :, :, None], torch.exp(between.float()), 0.0)
    states = torch.einsum("nzch,nchps->nzhps", between, parts)
    y += torch.einsum("ncigs,ncgkps,ncigk->ncigkp", cc, states[:, :-1].reshape(n, chunks, g, h // g, p, s), torch.exp(sums.float()).reshape(n, chunks, q, g, h // g)).reshape(y.shape)
    y += t["d"][:, None] * x
    y *= _silu(rows(t["proj"][:, :inner], h, p))
    t["out"][index[valid]] = y.reshape(n, chunks * q, inner)[valid].to(t["out"].dtype)
    t["state"][st.slot] = states[:, -1]
    return [t["out"], t["state"]]


def _plain_step(c, st, t):
    h, p, s, g, taps = c["heads"], c["dim"], c["state"], c["groups"], c["taps"]
    inner, ch = h * p, _channels(c)
    slot, kept = t["slots"][st.live].long(), t["out"].dtype
    row = t["proj"][st.live].float()
    u = torch.cat([t["conv_state"][slot].float(), row[:, None, inner:inner + ch]], 1)
    v = _silu(torch.einsum("rtc,ct->rc", u, t["weights"]) + t["bias"])
    x, b, cc = v[:, :inner].reshape(-1, h, p), v[:, inner:inner + g * s].reshape(-1, g, s), v[:, inner + g * s:].reshape(-1, g, s)
    dt = _softplus(row[:, inner + ch:] + t["dt_bias"])
    state = t["state"][slot] * torch.exp(dt * t["a"])[..., None, None]
    state += (dt[..., None] * x)[..., None] * b.repeat_interleave(h // g, 1)[:, :, None, :]
    y = torch.einsum("rhps,rhs->rhp", state, cc.repeat_interleave(h // g, 1)) + t["d"][:, None] * x
    t["out"][st.live] = (y.reshape(-1, inner) * _silu(row[:, :inner])).to(kept)
    t["conv_state"][slot] = u[:, 1:].to(kept)
    t["state"][slot] = state
    return [t["out"], t["conv_state"], t["state"]]


def _choose(c, logits):
    """Experts by their score, the lower index where two are alike, and their weights."""
    if c["score"] == "sigmoid":
        score = 1 / (1 + torch.exp(-logits))
    elif c["score"] == "all":
        score = torch.exp(logits - logits.amax(1, keepdim=True))
        score = score / score.sum(1, keepdim=True)
    else:
        score = logits
    ids = torch.sort(score, dim=1, descending=True, stable=True)[1][:, :c["top"]]
    w = torch.gather(score, 1, ids)
    if c["score"] == "chosen":
        w = torch.exp(w - w.amax(1, keepdim=True))
    if c["score"] != "all":
        w = w / w.sum(1, keepdim=True)
    return ids, w


def _plain_experts(c, st, t):
    x, f, rows, e = t["x"].float(), c["ff"], c["rows"], c["experts"]
    ids, w = _choose(c, x @ t["router"].float().T + t["router_bias"])
    every = torch.cat([ids, torch.arange(e, e + c["shared"], device="cuda").expand(rows, -1)], 1)
    factor = torch.cat([w, torch.ones(rows, c["shared"], device="cuda")], 1)
    if every.numel() < e + c["shared"]:                                              # few pairs: their experts alone
        up = torch.einsum("rkfw,rw->rkf", t["up_gate"][every].float(), x)
        hidden = _silu(up[..., f:]) * up[..., :f] * factor[..., None]
        out = torch.einsum("rkwf,rkf->rw", t["down"][every].float(), hidden)
    else:                                                                            # all experts for all rows
        up = torch.einsum("efw,rw->erf", t["up_gate"].float(), x)
        share = torch.zeros(rows, e + c["shared"], device="cuda").scatter_(1, every, factor)
        out = torch.einsum("ewf,erf->rw", t["down"].float(), _silu(up[..., f:]) * up[..., :f] * share.T[..., None])
    t["out"].copy_(out)
    t["ids"].copy_(ids)
    t["weights"].copy_(w)
    return [t["out"], t["ids"], t["weights"]]


PLAIN = {"conv": _plain_conv, "scan": _plain_scan, "step": _plain_step, "experts": _plain_experts}


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------------------------------
def work(case):
    e = 4 if case["type"] == "f32" else 2
    k = case["kind"]
    if k == "conv":
        values = case["rows"] * case["channels"]
        return {"bytes": 2 * values * e + 2 * case["sequences"] * (case["taps"] - 1) * case["channels"] * e + case["channels"] * (case["taps"] + 1) * 4, "flops": 2 * case["taps"] * values}
    if k == "experts":
        r, w, f, n = case["rows"], case["width"], case["ff"], case["experts"]
        met = n * (1 - (1 - case["top"] / n) ** r) + case["shared"]                  # experts that some row chooses, on average
        pairs = r * (case["top"] + case["shared"])
        return {"bytes": met * 3 * w * f * 2 + n * w * 2 + 2 * r * w * e + r * case["top"] * 8, "flops": pairs * 6 * w * f + 2 * r * w * n}
    h, p, s, r = case["heads"], case["dim"], case["state"], case["rows"]
    inner, ch = h * p, _channels(case)
    states = (r if k == "step" else case["sequences"]) * h * p * s * 4 * 2
    values = r * (2 * inner + ch + h) * e
    flops = 5 * r * h * p * s                                                        # decay, add, read out
    if k == "step":
        return {"bytes": states + values + 2 * r * (case["taps"] - 1) * ch * e + ch * (case["taps"] + 1) * 4, "flops": flops + 2 * case["taps"] * r * ch}
    return {"bytes": states + values, "flops": flops}


# ---- in 64 bits, from the definitions -------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    t = {n: v.double() if v.is_floating_point() else v for n, v in _tensors(case, seed).items()}
    return {"conv": _exact_conv, "scan": _exact_scan, "step": _exact_step, "experts": _exact_experts}[case["kind"]](case, seed, t)


def _exact_conv(c, seed, t):
    taps, out, state = c["taps"], torch.zeros_like(t["input"]), t["state"].clone()
    for first, n, slot, fresh in _lengths(c, seed):
        u = torch.cat([torch.zeros_like(state[slot]) if fresh else state[slot], t["input"][first:first + n]])
        y = sum(u[j:j + n] * t["weights"][:, j] for j in range(taps)) + t["bias"]
        out[first:first + n] = y * torch.sigmoid(y)
        state[slot] = u[n:]
    return [out, state]


def _exact_scan(c, seed, t):
    h, p, s, g = c["heads"], c["dim"], c["state"], c["groups"]
    inner, ch = h * p, _channels(c)
    x = t["xbc"][:, :inner].reshape(-1, h, p)
    b, cc = (v.reshape(-1, g, s) for v in (t["xbc"][:, inner:inner + g * s], t["xbc"][:, inner + g * s:]))
    dt = torch.nn.functional.softplus(t["proj"][:, inner + ch:] + t["dt_bias"], threshold=50)
    decay, xd = torch.exp(dt * t["a"]), dt[..., None] * x
    out, state = torch.zeros(t["proj"].shape[0], inner, dtype=F64, device="cuda"), t["state"].clone()
    for first, n, slot, fresh in _lengths(c, seed):
        now = torch.zeros_like(state[slot]) if fresh else state[slot].clone()
        now = now.reshape(g, h // g, p, s)
        y = torch.empty(n, g, (h // g) * p, dtype=F64, device="cuda")
        for i in range(first, first + n):                                            # the recurrence, token by token
            now *= decay[i].reshape(g, h // g, 1, 1)
            now.add_(xd[i].reshape(g, h // g, p, 1) * b[i].reshape(g, 1, 1, s))
            torch.matmul(now.reshape(g, -1, s), cc[i].reshape(g, s, 1), out=y[i - first].unsqueeze(-1))
        rows = slice(first, first + n)
        z = t["proj"][rows, :inner]
        out[rows] = (y.reshape(n, inner) + (t["d"][:, None] * x[rows]).reshape(n, inner)) * z * torch.sigmoid(z)
        state[slot] = now.reshape(h, p, s)
    return [out, state]


def _exact_step(c, seed, t):
    h, p, s, g, taps = c["heads"], c["dim"], c["state"], c["groups"], c["taps"]
    inner, ch = h * p, _channels(c)
    out, conv, state = torch.zeros(c["rows"], inner, dtype=F64, device="cuda"), t["conv_state"].clone(), t["state"].clone()
    for r, slot in enumerate(t["slots"].tolist()):
        if slot < 0:
            continue
        u = torch.cat([conv[slot], t["proj"][r:r + 1, inner:inner + ch]])
        v = sum(u[j] * t["weights"][:, j] for j in range(taps)) + t["bias"]
        v = v * torch.sigmoid(v)
        x = v[:inner].reshape(h, p)
        b, cc = (v[inner + i * g * s:inner + (i + 1) * g * s].reshape(g, 1, 1, s) for i in (0, 1))
        dt = torch.nn.functional.softplus(t["proj"][r, inner + ch:] + t["dt_bias"], threshold=50)
        now = (torch.exp(dt * t["a"])[:, None, None] * state[slot]).reshape(g, h // g, p, s) + (dt[:, None] * x).reshape(g, h // g, p, 1) * b
        y = (now * cc).sum(-1).reshape(h, p) + t["d"][:, None] * x
        z = t["proj"][r, :inner]
        out[r] = y.reshape(-1) * z * torch.sigmoid(z)
        conv[slot], state[slot] = u[1:], now.reshape(h, p, s)
    return [out, conv, state]


def _exact_experts(c, seed, t):
    logits = torch.nn.functional.linear(t["x"], t["router"], t["router_bias"])
    if c["score"] == "sigmoid":
        score = torch.sigmoid(logits)
    else:
        score = torch.softmax(logits, 1) if c["score"] == "all" else logits
    w, ids = torch.topk(score, c["top"], dim=1)
    if c["score"] != "all":
        w = torch.softmax(w, 1) if c["score"] == "chosen" else w / w.sum(1, keepdim=True)
    out = torch.zeros_like(t["x"])
    for e in range(c["experts"] + c["shared"]):
        mine = (ids == e).nonzero() if e < c["experts"] else None
        r = torch.arange(c["rows"], device="cuda") if mine is None else mine[:, 0]
        if len(r):
            up, gate = torch.nn.functional.linear(t["x"][r], t["up_gate"][e]).split(c["ff"], 1)
            y = torch.nn.functional.linear(gate * torch.sigmoid(gate) * up, t["down"][e])
            out[r] += y if mine is None else y * w[mine[:, 0], mine[:, 1]][:, None]
    return [out, None, w]
