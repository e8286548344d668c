"""The 8-bit cache's and the draft verification's definitions in float64 (numpy), beside bounds of what rounding in 32 bits may add."""
import math

import numpy as np

from tests.state_space_plain import BF16, F16, F32, of_kept, to_kept  # noqa: F401

I8, E4M3 = 0, 1
LARGEST = {I8: 127.0, E4M3: 448.0}
NO_INDEX = 0xFFFFFFFF
HUGE = 2.0 ** 96


def _e4m3_table():
    v = np.zeros(256)
    for b in range(256):
        e, m = b >> 3 & 15, b & 7
        v[b] = (m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)) * (-1 if b & 128 else 1)
    v[[0x7F, 0xFF]] = np.nan
    return v


E4M3_VALUES = _e4m3_table()
_POSITIVE = E4M3_VALUES[:0x7F]


def stands_for(codes, code):
    return codes.view(np.int8).astype(np.float64) if code == I8 else E4M3_VALUES[codes]


def coded(x, code):
    """numbers within the codes' range to the nearest code, ties to even"""
    if code == I8:
        return np.rint(x).astype(np.int8).view(np.uint8)
    a = np.abs(x)
    hi = np.clip(np.searchsorted(_POSITIVE, a), 0, 0x7E)
    lo = np.maximum(hi - 1, 0)
    up, down = _POSITIVE[hi] - a, a - _POSITIVE[lo]
    pick = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    return (pick | np.where(np.signbit(x), 0x80, 0)).astype(np.uint8)


def scale_of(x, code):
    """the smallest power of two from 2^-100 on with |x| <= LARGEST * scale; 0 for zeros, NaN for what has none"""
    if x.size == 0 or not np.any(x):
        return 0.0
    most = np.abs(x).max()
    if not most < HUGE:
        return math.nan
    e = max(-100, math.floor(math.log2(most / LARGEST[code])) - 1)
    while LARGEST[code] * 2.0 ** e < most:
        e += 1
    return 2.0 ** e


class Cache:
    def __init__(self, blocks, heads, block, dim, code, rng=None, garbage=None):
        shape = (blocks, heads, block, dim)
        self.blocks, self.heads, self.block, self.dim, self.code = blocks, heads, block, dim, code
        rng = rng or np.random.default_rng(0)
        self.codes = [np.full(shape, garbage, np.uint8) if garbage is not None else coded(np.clip(rng.standard_normal(shape) * LARGEST[code] / 4, -LARGEST[code], LARGEST[code]), code) for _ in range(2)]
        self.scales = [np.exp2(rng.integers(-7, -3, (blocks, heads))).astype(np.float64) for _ in range(2)]
        self.weights = rng.exponential(size=(blocks, heads, block)).astype(np.float32).astype(np.float64)

    def copy(self):
        c = object.__new__(Cache)
        c.__dict__.update(self.__dict__)
        c.codes, c.scales, c.weights = [x.copy() for x in self.codes], [x.copy() for x in self.scales], self.weights.copy()
        return c

    def numbers(self, which, table, tokens):
        """[len(tokens), heads, dim], and whether each has a block"""
        table = np.asarray(table, np.int64)
        nth = tokens // self.block
        b = table[nth]
        there = b < self.blocks
        b = np.where(there, b, 0)
        with np.errstate(invalid="ignore"):
            x = stands_for(self.codes[which][b, :, tokens % self.block], self.code) * self.scales[which][b][..., None]
        return x, there

    def append(self, table, length, rows, capacity):
        """rows: keys, values [n, heads, dim] of one sequence behind its `length` tokens"""
        for which, x in enumerate(rows):
            end = min(length + len(x), capacity)
            for nth in range(length // self.block, -(-end // self.block) if end > length else length // self.block):
                b, first = table[nth], nth * self.block
                if b >= self.blocks:
                    continue
                lo, hi = max(length, first), min(end, first + self.block)
                for h in range(self.heads):
                    old = lo - first
                    was = self.scales[which][b, h] if old else 0.0
                    new = x[lo - length:hi - length, h]
                    need = scale_of(new, self.code)
                    s = math.nan if math.isnan(was) or math.isnan(need) else max(was, need)
                    at = self.codes[which][b, h]
                    if math.isnan(s) or s == 0:
                        at[old:hi - first] = 0
                    else:
                        if s > was:
                            at[:old] = coded(stands_for(at[:old], self.code) * (was / s), self.code)
                        at[old:hi - first] = coded(new / s, self.code)
                    self.scales[which][b, h] = s
                if which == 0:
                    self.weights[b, :, lo - first:hi - first] = 0
        return min(length + len(rows[0]), capacity)

    def attend(self, table, length, q, capacity, scale, window=0, first=0, cap=0.0, sinks=None, weight_rows=0, q_error=0.0, tensor=False, fast_cap=False):
        """q [rows, query heads, dim]; tensor: on tcgen05; fast_cap: of 16-bit rows. (out, bound of its error before the last rounding), and the same of what the weights of each key grow by: [tokens, heads]"""
        n, hq, d = q.shape
        per = hq // self.heads
        end = min(length + n, capacity)
        k, there = self.numbers(0, table, np.arange(end))
        v, _ = self.numbers(1, table, np.arange(end))
        out, bound = np.zeros((n, hq, d)), np.zeros((n, hq, d))
        grow, grow_bound = np.zeros((end, self.heads)), np.zeros((end, self.heads))
        j = np.arange(end)
        for t in range(n):
            p = length + t
            seen = (j <= p) & there
            if window:
                seen &= (p - j < window) | (j < first)
            js = j[seen]
            if not len(js):
                continue
            for h in range(hq):
                g = h // per
                kk, vv = k[js, g], v[js, g]
                s, mag = scale * (kk @ q[t, h]), abs(scale) * (np.abs(kk) @ np.abs(q[t, h]))
                # sums of dim products in steps of 16 that cut at the last bit, the query's parts, the factors' roundings, a difference with the largest
                err = mag * ((d / 16 + 3) * 2.0 ** -22 + q_error)
                if cap:
                    s = cap * np.tanh(s / cap)
                    err = err + (cap * 2.0 ** -21 if fast_cap else 0.0)      # 1 - 2 / (1 + e^2x): roundings of numbers of up to 2
                err = err + (np.abs(s) + np.abs(s).max()) * 2.0 ** -22
                with np.errstate(invalid="ignore"):
                    top = s.max() if sinks is None else max(s.max(), sinks[h])
                    w = np.exp(s - top)
                    total = w.sum() + (0 if sinks is None else math.exp(sinks[h] - top))
                    w = w / total
                    # a weight's own error and its sum's; a sink is rounded in units of ln 2
                    part = err + err.max() + 2.0 ** -19 + (0 if sinks is None else 2.0 ** -21 * (abs(sinks[h]) + abs(top)))
                    out[t, h] = w @ vv
                    # A small weight's second f16 part ends at the subnormal spacing: off by 2^-25 of what is at most 2^15 for the row's largest weight, 2^-40 of that one
                    bound[t, h] = (w * (part + (len(js) / 16 + 60) * 2.0 ** -23) + 2.0 ** -40 * w.max(initial=0)) @ np.abs(vv)
                    # On tcgen05 a weight is one f16 number: half a step of 11 bits, and below the normal ones half of 2^-24, lifted by 2^1 and lowered by 2^4 at most (its group's value scale over the unit)
                    bound[t, h] += ((w * 2.0 ** -12 + 2.0 ** -22 * w.max(initial=0)) @ np.abs(vv)) if tensor else 0.0
                if t >= n - min(weight_rows, n):
                    grow[js, g] += w
                    grow_bound[js, g] += w * (part + (per * n + 4) * 2.0 ** -23)
        return out, bound, grow, grow_bound

    def evict(self, table, length, budget, first, last):
        """the kept tokens of each head, [heads, budget or fewer]"""
        if length <= budget:
            return np.tile(np.arange(length), (self.heads, 1)), length
        table = np.asarray(table)
        tokens = np.arange(length)
        b, at = table[tokens // self.block], tokens % self.block
        keep = np.zeros((self.heads, budget), np.int64)
        numbers = [self.numbers(w, table, tokens) for w in range(2)]
        new = self.copy()
        for h in range(self.heads):
            w = np.where(b < self.blocks, self.weights[np.minimum(b, self.blocks - 1), h, at], np.nan)
            middle = tokens[first:length - last]
            order = sorted(middle, key=lambda j: (-w[j] if w[j] == w[j] else math.inf, j))
            # (-infinity is before NaN)
            order = [j for j in order if w[j] == w[j]] + [j for j in order if w[j] != w[j]]
            keep[h] = sorted([*range(first), *range(length - last, length), *order[:budget - first - last]])
            for nth in range(-(-budget // self.block)):
                to = table[nth]
                js = keep[h][nth * self.block:(nth + 1) * self.block]
                if to >= self.blocks:
                    continue
                for which in range(2):
                    x, there = numbers[which]
                    x = np.where(there[js][:, None], x[js, h], 0.0)
                    s = scale_of(x, self.code)
                    new.codes[which][to, h, :len(js)] = 0 if s == 0 or math.isnan(s) else coded(x / s, self.code)
                    new.scales[which][to, h] = s
                new.weights[to, h, :len(js)] = np.where(b[js] < self.blocks, self.weights[np.minimum(b[js], self.blocks - 1), h, at[js]], 0.0)
        self.codes, self.scales, self.weights = new.codes, new.scales, new.weights
        return keep, budget


def distribution(row, temperature):
    """weights that sum to 1, or None"""
    if np.isnan(row).any() or not np.isfinite(row.max()):
        return None
    w = np.exp((row - row.max()) / temperature)
    return w / w.sum()


def verify(target, draft, drafted, uniforms, temperature, draft_temperature):
    """(accepted, token behind, whether its decisions are clear) of one sequence. A probability is off by a few roundings of exponents up to 2^5 in 32 bits, some 2^-19 of itself; sums
    over the vocabulary are of 64 bits"""
    clear = True
    for k in range(len(drafted) + 1):
        row = target[k]
        if temperature == 0:
            bad = np.isnan(row).any() or not np.isfinite(row.max())
            best = NO_INDEX if bad else int(np.argmax(row))
            if k < len(drafted) and not bad and drafted[k] == best:
                continue
            return k, best, clear
        p = distribution(row, temperature)
        q = None
        if k < len(drafted):
            x = drafted[k]
            if draft is None:
                q = np.zeros(len(row))
                if x < len(row):
                    q[x] = 1
            else:
                q = distribution(draft[k], draft_temperature)
            if p is not None and q is not None and x < len(row):
                clear &= abs(uniforms[k] * q[x] - p[x]) > 1e-5 * p[x] or p[x] == 0
                if uniforms[k] * q[x] < p[x]:
                    continue
        if p is None or (k < len(drafted) and q is None):
            return k, NO_INDEX, clear
        r = p if q is None else np.maximum(p - q, 0)
        if not r.sum() > 0:
            r = p
        sums = np.cumsum(r)
        aim = uniforms[-1] * sums[-1]
        clear &= np.abs(sums - aim).min() > 1e-9 * sums[-1] or uniforms[-1] == 0
        passed = np.flatnonzero(sums > aim)
        return k, int(passed[0]) if len(passed) else int(np.flatnonzero(r > 0)[-1]), clear
