"""The state space mixer's and the experts' layer's definitions in float64 (numpy), each beside a bound of what rounding in 32 bits may add: the same
sums over absolute values."""
import numpy as np

BF16, F32, F16 = 0, 1, 2
HALF_STEP = {BF16: 2.0 ** -8, F32: 2.0 ** -24, F16: 2.0 ** -11}      # a rounding is off by at most this part of the value
TINY = {BF16: 2.0 ** -133, F32: 2.0 ** -149, F16: 2.0 ** -25}        # ... or by this, below the type's normal numbers


def to_kept(x, dt):
    """float array -> what the device holds."""
    x = np.asarray(x, np.float32)
    if dt == F32:
        return x
    if dt == F16:
        return x.astype(np.float16)
    u = x.view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def of_kept(v, dt):
    if dt == BF16:
        return (v.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return v.astype(np.float64)


def silu(x):
    with np.errstate(over="ignore"):
        return x / (1 + np.exp(-x))


def softplus(x):
    return np.where(x > 30, x, np.log1p(np.exp(np.minimum(x, 30))))


def conv(u, w, bias, state, sequences, act=True):
    """u [rows, channels], state [slots, taps - 1, channels]; returns out (nan where no sequence is), state, bound of sum |w u| + |bias|."""
    taps = w.shape[1]
    out, mag, state = np.full(u.shape, np.nan), np.zeros(u.shape), state.copy()
    for first, n, slot, fresh in sequences:
        v = np.concatenate([np.zeros_like(state[slot]) if fresh else state[slot], u[first:first + n]])
        y, m = np.zeros((n, u.shape[1])) + bias, np.zeros((n, u.shape[1])) + np.abs(bias)
        for j in range(taps):
            y = y + v[j:j + n] * w[:, j]
            m = m + np.abs(v[j:j + n] * w[:, j])
        out[first:first + n], mag[first:first + n] = silu(y) if act else y, m
        state[slot] = v[n:]
    return out, state, mag


def steps(dt, bias, use_softplus=True, lo=0.0, hi=np.inf):
    v = dt + bias
    return np.clip(softplus(v) if use_softplus else v, lo, hi)


def scan(x, step, b, c, z, a, d, state, sequences):
    """x, z [rows, heads, dim], step [rows, heads], b, c [rows, groups, n], state [slots, heads, dim, n]; z may be None. Returns out, state and the
    magnitudes of both (the recurrence over absolute values; out's before the gate)."""
    h, g = x.shape[1], b.shape[1]
    b, c = np.repeat(b, h // g, 1), np.repeat(c, h // g, 1)
    out, mag = np.full(x.shape, np.nan), np.zeros(x.shape)
    state, smag = state.copy(), np.abs(state)
    for first, n, slot, fresh in sequences:
        s = np.zeros_like(state[slot]) if fresh else state[slot]
        m = np.abs(s)
        for t in range(first, first + n):
            f = np.exp(step[t] * a)[:, None, None]
            add = (step[t][:, None] * x[t])[:, :, None] * b[t][:, None, :]
            s, m = f * s + add, f * m + np.abs(add)
            out[t] = (s * c[t][:, None, :]).sum(-1) + d[:, None] * x[t]
            mag[t] = (m * np.abs(c[t])[:, None, :]).sum(-1) + np.abs(d[:, None] * x[t])
        state[slot], smag[slot] = s, m
    if z is not None:
        out = out * silu(z)
    return out, state, mag, smag


def experts(x, router, bias, up_gate, down, top, shared, score, renormalise, scale, act):
    """Returns out, ids, weights, magnitudes of out, and the smallest gap between a chosen and a left-out score."""
    f = up_gate.shape[1] // 2
    e = router.shape[0]
    logits = x @ router.T + bias
    if score == 2:
        s = 1 / (1 + np.exp(-logits))
    elif score == 1:
        s = np.exp(logits - logits.max(1, keepdims=True))
        s /= s.sum(1, keepdims=True)
    else:
        s = logits
    order = np.argsort(-s, axis=1, kind="stable")
    ids = order[:, :top]
    w = np.take_along_axis(s, ids, 1)
    gap = np.inf if top == e else float((w[:, -1] - np.take_along_axis(s, order[:, top:top + 1], 1)[:, 0]).min())
    if top > 1:
        gap = min(gap, float((w[:, :-1] - w[:, 1:]).min()))
    if score == 0:
        w = np.exp(w - w[:, :1])
        w /= w.sum(1, keepdims=True)
    if renormalise:
        w = w / w.sum(1, keepdims=True)
    w = w * scale
    out, mag = np.zeros_like(x), np.zeros_like(x)
    for r in range(x.shape[0]):
        for i, k in [(i, w[r, j]) for j, i in enumerate(ids[r])] + [(e + j, 1.0) for j in range(shared)]:
            y = up_gate[i] @ x[r]
            m = np.abs(up_gate[i]) @ np.abs(x[r])
            gate = act(y[f:])
            hidden = gate * y[:f] * k
            out[r] += down[i] @ hidden
            # |act'| <= 1.13: what an error of the products may become
            mag[r] += np.abs(down[i]) @ (abs(k) * (np.abs(gate) * m[:f] + 1.13 * m[f:] * np.abs(y[:f])) + np.abs(hidden))
    return out, ids, w, mag, gap
