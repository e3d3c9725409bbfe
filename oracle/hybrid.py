"""The operators of hybrid models' layers (include/aotx_hybrid.h) in 64 bits, one token after
another, straight from their definitions. Rows are packed; a sequence that names no slot, or a
slot that an earlier sequence with rows has, gets zeros and counts as a fault."""
import numpy as np


def silu(x):
    x = np.asarray(x, dtype=np.float64)
    with np.errstate(over="ignore"):
        return x / (1.0 + np.exp(-x))


def spans_of(offset, tokens):
    """(start, end) of every sequence: in bounds, none before an earlier one's last row."""
    at = np.maximum.accumulate([min(int(o), tokens) for o in offset])
    return list(zip(at[:-1].tolist(), at[1:].tolist()))


def walk(offset, agent, slots, tokens):
    """(index, start, end, slot or None) of the sequences with rows, and the refused ones."""
    taken, got = set(), []
    for i, (b, e) in enumerate(spans_of(offset, tokens)):
        if b == e:
            continue
        slot = int(agent[i])
        ok = slot < slots and slot not in taken
        taken.add(slot)
        got.append((i, b, e, slot if ok else None))
    return got


def conv(x, w, bias, offset, pos, agent, state, out):
    """out and state are changed in place; returns the faults."""
    width, faults = w.shape[1], 0
    for i, b, e, slot in walk(offset, agent, len(state), len(x)):
        if slot is None:
            out[b:e], faults = 0, faults + 1
            continue
        before = np.zeros_like(state[slot]) if pos[i] == 0 else state[slot].copy()
        full = np.concatenate([before, x[b:e].astype(np.float64)])
        for t in range(e - b):
            y = (full[t:t + width] * w.T).sum(0)
            out[b + t] = silu(y if bias is None else y + bias)
        state[slot] = full[e - b:]
    return faults


def gates(a, b, decay, dt):
    """(log decay, beta)."""
    g = np.minimum(decay * np.logaddexp(0.0, a.astype(np.float64) + dt), 0.0)
    return g, 1.0 / (1.0 + np.exp(-b.astype(np.float64)))


def rows(qkv, key_heads, heads, d, eps):
    """q', k' and v of every row and value head."""
    x = qkv.astype(np.float64)
    n, group = len(x), heads // key_heads
    q = x[:, :key_heads * d].reshape(n, key_heads, d)
    k = x[:, key_heads * d:2 * key_heads * d].reshape(n, key_heads, d)
    v = x[:, 2 * key_heads * d:(2 * key_heads + heads) * d].reshape(n, heads, d)
    q = q / np.sqrt((q * q).sum(-1, keepdims=True) + eps) / np.sqrt(d)
    k = k / np.sqrt((k * k).sum(-1, keepdims=True) + eps)
    return np.repeat(q, group, 1), np.repeat(k, group, 1), v


def delta(qkv, a, b, decay, dt, offset, pos, agent, key_heads, heads, d, eps, state, out):
    """out [rows][heads][d] and state [slots][heads][d][d] are changed in place. Returns (faults,
    the largest magnitude that a state entry or a value had, and for every output the sum of the
    sizes of the terms (q' . k'_j) exp(G - G_j) u_j of the rows j of its own 64, itself among them)."""
    q, k, v = rows(qkv, key_heads, heads, d, eps)
    g, beta = gates(a, b, decay, dt)
    faults, top, near = 0, 0.0, np.zeros(out.shape)
    for i, lo, hi, slot in walk(offset, agent, len(state), len(qkv)):
        if slot is None:
            out[lo:hi], faults = 0, faults + 1
            continue
        S = np.zeros_like(state[slot]) if pos[i] == 0 else state[slot].copy()
        top = max(top, np.abs(S).max())
        for t in range(lo, hi):
            if (t - lo) % 64 == 0:
                us, fade, first = [], np.zeros((0, heads)), t
            S = S * np.exp(g[t])[:, None, None]
            u = beta[t][:, None] * (v[t] - np.einsum("hkv,hk->hv", S, k[t]))
            S = S + k[t][:, :, None] * u[:, None, :]
            out[t] = np.einsum("hkv,hk->hv", S, q[t])
            us.append(np.abs(u))
            fade = np.concatenate([fade * np.exp(g[t]), np.ones((1, heads))])
            size = np.abs(np.einsum("hk,nhk->nh", q[t], k[first:t + 1])) * fade
            near[t] = np.einsum("nh,nhv->hv", size, np.array(us))
            top = max(top, np.abs(S).max())
        top = max(top, np.abs(v[lo:hi]).max())
        state[slot] = S
    return faults, top, near


def delta_chunked(qkv, a, b, decay, dt, key_heads, heads, d, eps, S, chunk=64):
    """One sequence in chunks (the formula of the chunked kernel); returns (out, S)."""
    q, k, v = rows(qkv, key_heads, heads, d, eps)
    g, beta = gates(a, b, decay, dt)
    out, S = np.zeros_like(v), S.copy()
    for lo in range(0, len(qkv), chunk):
        at = slice(lo, min(lo + chunk, len(qkv)))
        for h in range(heads):
            G = np.cumsum(g[at, h])
            fade = np.tril(np.exp(np.minimum(G[:, None] - G[None, :], 0.0)))
            K, Q, B = k[at, h], q[at, h], beta[at, h]
            M = np.tril(B[:, None] * (K @ K.T) * fade, -1)
            T = np.linalg.solve(np.eye(len(G)) + M, np.diag(B))
            U = T @ (v[at, h] - np.exp(G)[:, None] * (K @ S[h]))
            out[at, h] = np.exp(G)[:, None] * (Q @ S[h]) + (Q @ K.T * fade) @ U
            S[h] = np.exp(G[-1]) * S[h] + (K * np.exp(G[-1] - G)[:, None]).T @ U
    return out, S


def norm_gate(x, z, w, eps):
    """x, z [..][width]."""
    x = x.astype(np.float64)
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w * silu(z)


def axis_of(spans, order, pairs):
    if order == 0:
        return [j for j, n in enumerate(spans) for _ in range(n)]
    axes = len(spans)
    return [i % axes if i < axes * spans[i % axes] else 0 for i in range(pairs)]


def rope_axes(x, norm, eps, place, theta, rope_dim, split, spans, order, factor=None):
    """x [tokens][heads][d] fp32 -> turned rows, in 64 bits."""
    x = x.astype(np.float64)
    if norm is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * norm
    half = rope_dim // 2
    freq = float(theta) ** (-2.0 * np.arange(half) / rope_dim)
    if factor is not None:
        freq = freq / factor
    angle = place[:, axis_of(spans, order, half)].astype(np.float64) * freq
    cos, sin = np.cos(angle)[:, None], np.sin(angle)[:, None]
    low = np.arange(half) if split else 2 * np.arange(half)
    high = low + half if split else low + 1
    y = x.copy()
    y[..., low] = x[..., low] * cos - x[..., high] * sin
    y[..., high] = x[..., low] * sin + x[..., high] * cos
    return y
