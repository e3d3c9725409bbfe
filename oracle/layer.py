"""The operators of a full layer and of a step's answer (include/aotx_layer.h) in 64 bits, from their
definitions. `far` beside a result is how far fp32 arithmetic may be from it."""
import math

import numpy as np

from oracle import hybrid as H

E32 = 2.0 ** -24        # half a step of fp32, relative


def q8_values(raw, n, k):
    """half(quant * scale) of Q8_0 rows (bytes [n][k / 32 * 34]) as float64 [n][k]."""
    b = np.ascontiguousarray(raw).reshape(n, k // 32, 34)
    scale = b[:, :, :2].copy().view(np.float16).astype(np.float32)
    with np.errstate(over="ignore", invalid="ignore"):
        w = (b[:, :, 2:].copy().view(np.int8).astype(np.float32) * scale).astype(np.float16)
    return w.astype(np.float64).reshape(n, k)


def act(x, kind):
    """(act(x), a bound of its slope)"""
    with np.errstate(over="ignore", invalid="ignore"):
        if kind == 1:
            return x / (1 + np.exp(-x)), 1.1
        if kind == 2:
            return 0.5 * x * (1 + np.vectorize(math.erf, otypes=[float])(x / math.sqrt(2))), 1.13
        if kind == 3:
            return 0.5 * x * (1 + np.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3))), 1.13
    return (np.where(x < 0, 0.0, x) if kind == 4 else x), 1.0


def linear(x, w, up=None, bias=None, up_bias=None, resid=None, kind=0):
    """(y, far): x [m][k], w and up [n][k] float64.

    A sum of k exact products is rounded k times by E32 of a partial sum, which is at most the sum of
    the terms' sizes; roundings add like a random walk, sqrt(k), and four times that is allowed.
    An activation's steps (an exponential, a quotient, products) are 16 roundings of its argument's size;
    bias, gate and residual round once each."""
    def product(w, bias):
        y, size = x @ w.T, np.abs(x) @ np.abs(w).T
        far = 4 * math.sqrt(x.shape[1]) * E32 * size
        if bias is not None:
            y = y + bias
            far = far + E32 * np.abs(y)
        return y, far

    y, far = product(w, bias)
    if kind:
        size = np.abs(y)
        y, slope = act(y, kind)
        far = slope * far + 16 * E32 * size
    if up is not None:
        u, ufar = product(up, up_bias)
        far = np.abs(u) * far + np.abs(y) * ufar + far * ufar + E32 * np.abs(y * u)
        y = y * u
    if resid is not None:
        y = y + resid
        far = far + E32 * np.abs(y)
    return y, far


def rounded(far, y, half):
    """`far` with the last rounding: 2^-11 of the value, or half a step of the subnormals."""
    return far + 2.0 ** -11 * np.abs(y) + 2.0 ** -25 if half else far


def norm_rows(x, w, eps):
    x = x.astype(np.float64)
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w


def places(slot, pos, table, layer, layers, kv_heads, d, page_bytes=2 << 20, header=256):
    """Index in the pool's halves of (slot, pos)'s K head 0, or None; table [slots][640] of byte offsets into
    the pool (below 0: no page)."""
    block_bytes = 2 * kv_heads * 16 * d * 2
    per = (page_bytes - header) // block_bytes
    block = pos // 16 * layers + layer
    if block // per >= table.shape[1] or table[slot, block // per] < 0:
        return None
    return (int(table[slot, block // per]) + header + block % per * block_bytes) // 2 + pos % 16 * d


def kv_append(qkv, heads, kv, d, rope, place, offset, pos, agent, layer, layers, table, pool, q, row_pos, row_agent):
    """Changes pool (halves), q, row_pos and row_agent in place, unrounded; returns the faults. rope: a function
    (rows, norm name, places) -> turned rows. place None: the cache positions."""
    faults, slots = 0, 64
    for i, b, e, slot in H.walk(offset, agent, slots, len(qkv)):
        if slot is None:
            q[b:e], row_pos[b:e], row_agent[b:e] = 0, 0, slots
            faults += 1
            continue
        at = int(pos[i]) + np.arange(e - b)
        row_pos[b:e], row_agent[b:e] = at & 0xFFFFFFFF, np.where(at >> 32, slots, slot)
        x = qkv[b:e].reshape(e - b, -1, d)
        where = at[:, None] if place is None else place[b:e]
        q[b:e] = rope(x[:, :heads], "q", where)
        k = rope(x[:, heads:heads + kv], "k", where)
        v = x[:, heads + kv:].astype(np.float64)
        for t in range(e - b):
            to = places(slot, int(at[t]), table, layer, layers, kv, d)
            if to is None:
                faults += 1
                continue
            for h in range(kv):
                pool[to + h * 16 * d:][:d] = k[t, h]
                pool[to + (kv + h) * 16 * d:][:d] = v[t, h]
    return faults


def adjust(row, sample=None, tokens=(), biases=(), mask=None):
    """(z, far) of one row; sample (presence, frequency, repeat, window), biases [(token, value)], mask
    a truth value a token. Six roundings of the largest value on the way."""
    z = row.astype(np.float64)
    vocab, far = len(z), np.zeros(len(z))
    if sample is not None:
        presence, frequency, repeat, window = (float(v) for v in sample)
        count, late = {}, set()
        for i, t in enumerate(tokens):
            if 0 <= t < vocab:
                count[t] = count.get(t, 0) + 1
                if i >= len(tokens) - window:
                    late.add(t)
        for t, c in count.items():
            far[t] = abs(z[t]) + abs(presence) + abs(frequency * c) if np.isfinite(z[t]) else 0
            z[t] -= presence + frequency * c
        for t in late:
            factor = 1 / repeat if z[t] > 0 else repeat
            # a value that rounding moves across zero takes the other factor
            far[t] *= max(repeat, 1 / repeat)
            z[t] *= factor
    last = {}
    for t, v in biases:
        if 0 <= t < vocab:
            last[t] = float(v)
    for t, v in last.items():
        with np.errstate(invalid="ignore"):
            z[t] += v
        far[t] += abs(v) + abs(z[t]) if np.isfinite(z[t]) else 0
    if mask is not None:
        z[~mask] = -np.inf
    return z, 6 * E32 * far
