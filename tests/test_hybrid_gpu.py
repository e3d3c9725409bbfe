"""The operators of hybrid models' layers on the GPU against the 64-bit oracle (oracle/hybrid.py):
lengths of zero, one and around a chunk's 64 rows, strides, slots that are missing or named twice,
rows outside the sequences, values of Inf and NaN, capture, other streams, and a layer of them.

Tolerances. A result rounded to fp16 is within 2^-11 of its value or 2^-25 of a subnormal one. An
fp32 sum of n terms of size m is off by about sqrt(n) 2^-24 m (roundings add like a random walk),
and T updates of a state add their errors the same way, so a state entry is held to
4 sqrt(d T) 2^-24 of the largest entry or value, four times what is expected; operands that are
taken as two fp16 parts are good to 2^-21, less than the sums' own errors. A delta output is S^T q'
with |q'| <= 1 / sqrt(d), so the sum of |q'| is at most 1 and the state's error bounds its own; the
factors (q' . k'_j) exp(G - G_j) of the rows of an output's own chunk are rounded to fp16 on the way,
which adds 2^-11 of the sum of those terms' sizes at most."""
import ctypes

import numpy as np
import pytest

import aotx_amd
from aotx_amd.model import normal, quantize_q8
from oracle import hybrid as H
from oracle.kvpolicy import layout_pages
from tests.gpu_util import KEEP, dev, p

pytestmark = pytest.mark.gpu

EPS = 1e-6


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


@pytest.fixture(autouse=True)
def _no_faults(lib):
    lib.aotx_model_forget()


def _up(torch, a, dtype):
    """A device tensor of `a` with its own shape."""
    t = torch.from_numpy(np.ascontiguousarray(a, dtype=dtype)).cuda()
    KEEP.append(t)
    return t


class Delta:
    """One call's inputs, on the host and the device."""

    def __init__(self, torch, seed, lens, key_heads=2, heads=4, d=128, lead=0, tail=0, pad=0, slots=8, fresh=(),
                 agent=None, scale=1.0):
        rng = np.random.default_rng(seed)
        self.eps = EPS
        self.torch, self.key_heads, self.heads, self.d, self.lens = torch, key_heads, heads, d, lens
        self.tokens = lead + sum(lens) + tail
        self.offset = lead + np.concatenate([[0], np.cumsum(lens)]).astype(np.uint32)
        self.width = (2 * key_heads + heads) * d
        self.stride, self.ab_stride = self.width + pad, heads + pad
        self.x = H.silu(rng.normal(0, 1, (self.tokens, self.stride))).astype(np.float16)
        self.x[:, 2 * key_heads * d:] *= np.float16(scale)
        self.a = rng.normal(0, 1, (self.tokens, self.ab_stride)).astype(np.float32)
        self.b = rng.normal(0, 1, (self.tokens, self.ab_stride)).astype(np.float32)
        self.decay = -rng.uniform(1, 16, heads).astype(np.float32)
        self.dt = rng.uniform(-7, -2, heads).astype(np.float32)
        n = len(lens)
        self.agent = np.array(rng.permutation(slots)[:n] if agent is None else agent, dtype=np.uint32)
        self.pos = np.array([0 if i in fresh else 10 + i for i in range(n)], dtype=np.uint32)
        self.state = rng.normal(0, 0.3 * scale, (slots, heads, d, d)).astype(np.float32)

    def want(self):
        state = self.state.astype(np.float64)
        out = np.full((self.tokens, self.heads, self.d), 7.0)
        faults, top, near = H.delta(self.x, self.a[:, :self.heads], self.b[:, :self.heads], self.decay.astype(np.float64),
                              self.dt.astype(np.float64), self.offset, self.pos, self.agent, self.key_heads, self.heads,
                              self.d, self.eps, state, out)
        self.round = 2.0 ** -11 * (np.abs(out) + near) + 2.0 ** -25      # of out and of its factors
        return out, state, faults, top

    def up(self):
        t = self.torch
        self.dev = {n: _up(t, getattr(self, n), dt) for n, dt in
                    (("x", np.float16), ("a", np.float32), ("b", np.float32), ("decay", np.float32), ("dt", np.float32),
                     ("offset", np.int32), ("pos", np.int32), ("agent", np.int32), ("state", np.float32))}
        self.dev["out"] = t.full((self.tokens, self.heads, self.d), 7.0, dtype=t.float16, device="cuda")
        return self

    def call(self, lib, step=False, stream=None, work=None):
        g = {k: p(v) for k, v in self.dev.items()}
        if step:
            rc = lib.aotx_delta_step(g["x"], self.stride, g["a"], g["b"], self.ab_stride, g["decay"], g["dt"], g["pos"],
                                     g["agent"], self.tokens, self.key_heads, self.heads, self.d, self.eps, g["state"],
                                     len(self.state), g["out"], stream)
        else:
            need = lib.aotx_delta_work(self.tokens, len(self.lens), self.heads, self.d)
            if work is None:
                work = self.torch.full((need,), 0xFF, dtype=self.torch.uint8, device="cuda")
                KEEP.append(work)
            rc = lib.aotx_delta_chunk(g["x"], self.stride, g["a"], g["b"], self.ab_stride, g["decay"], g["dt"],
                                      g["offset"], g["pos"], g["agent"], len(self.lens), self.tokens, self.key_heads,
                                      self.heads, self.d, self.eps, g["state"], len(self.state), p(work), need, g["out"], stream)
        assert rc == 0
        return self

    def got(self):
        self.torch.cuda.synchronize()
        return self.dev["out"].cpu().numpy().astype(np.float64), self.dev["state"].cpu().numpy().astype(np.float64)

    def check(self, lib):
        want, state, faults, top = self.want()
        out, S = self.got()
        far = 4 * np.sqrt(self.d * max(1, max(self.lens))) * 2.0 ** -24 * top
        assert np.abs(S - state).max() <= far, (np.abs(S - state).max(), far)
        off = np.abs(out - want) - (self.round + far)
        assert off.max() <= 0, (off.max(), far)
        assert lib.aotx_model_faulted() == faults
        # slots that no sequence with rows names, bit for bit
        named = {int(a) for a, n in zip(self.agent, self.lens) if n}
        for s in set(range(len(self.state))) - named:
            assert np.array_equal(S[s], self.state[s].astype(np.float64))
        return self


HEADS = [(2, 4, 128), (1, 1, 64), (3, 3, 128), (2, 6, 64), (16, 32, 128)]


@pytest.mark.parametrize("key_heads,heads,d", HEADS)
@pytest.mark.parametrize("tokens", [1, 5])
def test_step(torch, lib, key_heads, heads, d, tokens):
    Delta(torch, tokens, [1] * tokens, key_heads, heads, d, fresh=(1,)).up().call(lib, step=True).check(lib)


def test_step_all_slots_padded_rows(torch, lib):
    Delta(torch, 9, [1] * 64, 2, 4, 128, slots=64, pad=24, fresh=range(0, 64, 5)).up().call(lib, step=True).check(lib)


def test_step_slots_missing_and_named_twice(torch, lib):
    c = Delta(torch, 11, [1] * 6, agent=[3, 8, 3, 0, 4000000000, 0], slots=8).up().call(lib, step=True).check(lib)
    assert lib.aotx_model_faulted() == 4
    out, _ = c.got()
    assert not out[[1, 2, 4, 5]].any() and out[[0, 3]].any()


@pytest.mark.parametrize("key_heads,heads,d", HEADS)
def test_chunk_lengths(torch, lib, key_heads, heads, d):
    lens = [0, 1, 63, 64, 65, 0, 130, 17]
    Delta(torch, heads + d, lens, key_heads, heads, d, lead=3, tail=5, slots=9, fresh=(2, 6)).up().call(lib).check(lib)


@pytest.mark.parametrize("lens", [[1], [2], [16], [40], [64], [128], [1000], [700, 1], [1] * 30 + [300]])
def test_chunk_whole_calls(torch, lib, lens):
    Delta(torch, len(lens) + lens[0], lens, 1, 2, 128, slots=32, pad=8).up().call(lib).check(lib)


@pytest.mark.parametrize("key_heads,heads,d", [(16, 32, 64), (32, 32, 128)])
def test_chunk_few_rows_beside_many(torch, lib, key_heads, heads, d):
    """Sequences of few rows go row by row, the others in chunks, in one call: lengths on both
    sides of either limit, and so many heads and sequences that the higher one holds."""
    lens = [1, 12, 13, 4, 5, 0, 200, 2, 11, 64] + [1, 3, 14] * 8
    Delta(torch, heads + d, lens, key_heads, heads, d, lead=1, tail=2, slots=40, fresh=(1, 6, 9),
          agent=list(range(33)) + [5]).up().call(lib).check(lib)


@pytest.mark.parametrize("key_heads,heads,d", [(2, 4, 128), (1, 1, 64), (4, 8, 64)])
@pytest.mark.parametrize("lens,lead,tail", [([3], 0, 0), ([64], 0, 0), ([17, 0, 33, 1], 5, 8), ([1, 2, 3, 4, 5, 6], 1, 0),
                                            ([0, 31], 0, 33), ([16, 48], 0, 0)])
def test_chunk_short_calls(torch, lib, key_heads, heads, d, lens, lead, tail):
    """Up to 64 rows: one launch, whatever the sequences."""
    Delta(torch, len(lens) + heads, lens, key_heads, heads, d, lead=lead, tail=tail, pad=16, fresh=(1, 2)).up().call(
        lib).check(lib)


@pytest.mark.parametrize("heads", [32, 33])
def test_chunk_short_calls_up_to_a_workgroup_a_cu(torch, lib, heads):
    """The largest call of one launch, and one head more."""
    Delta(torch, 23, [29], heads, heads, 128).up().call(lib).check(lib)


def test_chunk_short_slots_missing_and_named_twice(torch, lib):
    Delta(torch, 24, [7, 5, 6, 0, 30, 9], agent=[3, 8, 3, 1, 1, 1], slots=8, fresh=(0,)).up().call(lib).check(lib)
    assert lib.aotx_model_faulted() == 3


@pytest.mark.parametrize("lens", [[3], [70, 1, 130]])
def test_chunk_keeps_to_its_workspace(torch, lib, lens):
    """What lies behind the workspace's stated size stays as it was, and what a workspace holds
    from before makes no difference."""
    outs = []
    for fill in (0x00, 0x7F):
        c = Delta(torch, 16, lens, 2, 4, 64).up()
        need = lib.aotx_delta_work(sum(lens), len(lens), 4, 64)
        work = torch.full((need + 4096,), fill, dtype=torch.uint8, device="cuda")
        KEEP.append(work)
        g = {k: p(v) for k, v in c.dev.items()}
        assert lib.aotx_delta_chunk(g["x"], c.stride, g["a"], g["b"], c.ab_stride, g["decay"], g["dt"], g["offset"], g["pos"],
                                    g["agent"], len(lens), c.tokens, 2, 4, 64, EPS, g["state"], 8, p(work), need, g["out"],
                                    None) == 0
        outs.append(c.got())
        assert (work[need:] == fill).all()
    assert np.array_equal(outs[0][0], outs[1][0]) and np.array_equal(outs[0][1], outs[1][1])


@pytest.mark.parametrize("heads,d,tail", [(33, 128, 37), (4, 128, 97), (2, 64, 200), (65, 64, 17)])
@pytest.mark.parametrize("rows", [0, 1, 3, 4, 5])
@pytest.mark.parametrize("agent", [2, 8])
def test_chunk_one_sequence_shorter_than_its_call(torch, lib, heads, d, tail, rows, agent):
    """A call's one sequence may have fewer rows than the call has room for: any number of them is
    taken, a fresh slot is cleared, and one that is none is told of."""
    Delta(torch, heads + rows, [rows], 1, heads, d, lead=2, tail=tail, fresh=(0,) if rows == 3 else (), agent=[agent]).up().call(
        lib).check(lib)
    assert lib.aotx_model_faulted() == (agent == 8 and rows > 0)


@pytest.mark.parametrize("heads,tokens", [(4, 200), (33, 40)])
def test_chunk_one_sequence_shrinks_in_a_graph(torch, lib, heads, tokens):
    """A call captured for a full bucket and replayed with pieces of any length, as a server does."""
    c = Delta(torch, 25, [tokens], 1, heads, 128).up()
    work = torch.empty(lib.aotx_delta_work(tokens, 1, heads, 128), dtype=torch.uint8, device="cuda")
    KEEP.append(work)
    first = {k: v.clone() for k, v in c.dev.items()}
    c.call(lib, work=work)
    side = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=side):
        c.call(lib, stream=ctypes.c_void_p(side.cuda_stream), work=work)
    for rows in (3, tokens, 1, 4, 0, 30, 3):
        for k, v in first.items():
            c.dev[k].copy_(v)
        c.dev["offset"].copy_(torch.tensor([0, rows], dtype=torch.int32))
        c.offset, c.lens = np.array([0, rows], dtype=np.uint32), [rows]
        torch.cuda.synchronize()
        g.replay()
        c.check(lib)


def _check_heads(c, lib, picks):
    """Delta.check of some heads alone, which share nothing but keys, for calls whose 64-bit walk of all
    would take too long."""
    d, kh, n = c.d, c.key_heads, len(picks)
    keys = [h // (c.heads // kh) for h in picks]
    cut = [c.x[:, j * d:(j + 1) * d] for j in keys + [kh + j for j in keys] + [2 * kh + h for h in picks]]
    some = Delta(c.torch, 0, c.lens, n, n, d, slots=1, agent=c.agent)
    some.x, some.a, some.b = np.concatenate(cut, 1), c.a[:, picks], c.b[:, picks]
    some.decay, some.dt, some.state, some.pos, some.offset, some.tokens = (c.decay[picks], c.dt[picks], c.state[:, picks], c.pos,
                                                                           c.offset, c.tokens)
    out, S = c.got()
    some.got = lambda: (out[:, picks], S[:, picks])
    some.check(lib)


@pytest.mark.parametrize("key_heads,heads,d,lens", [(2, 32, 128, [6540]), (2, 32, 128, [6500]), (4, 128, 64, [1700]),
                                                    (1, 32, 128, [4000, 2700])])
def test_chunk_workspace_past_the_caches(torch, lib, key_heads, heads, d, lens):
    """Calls whose lines are asked for two chunks before they are loaded, the last chunk whole or a part."""
    tokens, n = sum(lens), len(lens)
    assert lib.aotx_delta_work(tokens, n, heads, d) > 100 << 20
    c = Delta(torch, 38, lens, key_heads, heads, d, slots=n, fresh=(0,)).up().call(lib)
    _check_heads(c, lib, [1, heads - 1])
    for at in (64 * 3, tokens - 1):                         # and a row that is no number, early and last
        c = Delta(torch, 38, lens, key_heads, heads, d, slots=n, fresh=(0,))
        c.x[at, (2 * key_heads + 1) * d + 5] = np.inf
        base, S0 = Delta(torch, 38, lens, key_heads, heads, d, slots=n, fresh=(0,)).up().call(lib).got()
        out, S = c.up().call(lib).got()
        end = int(c.offset[np.searchsorted(c.offset, at, side="right")])
        assert not np.isfinite(out[at:end, 1, 5]).any() and np.isfinite(out[:at, 1, 5]).all()
        out[:end, 1, 5] = base[:end, 1, 5] = 0
        S[:, 1, :, 5] = S0[:, 1, :, 5] = 0
        assert np.array_equal(out, base) and np.array_equal(S, S0)


@pytest.mark.parametrize("key_heads,heads,d", [(2, 32, 64), (4, 32, 128)])
def test_chunk_few_rows_beside_a_large_call(torch, lib, key_heads, heads, d):
    """Sequences of few rows in a launch of their own: beside more than 1536 chunks and heads, and beside
    so many sequences that 12 rows are few, at lengths on both sides."""
    for lens in ([2900, 3, 1, 0, 4, 5, 300, 2], [700] * 3 + [12, 1, 13, 0, 5] * 6):
        n = len(lens)
        c = Delta(torch, n, lens, key_heads, heads, d, lead=1, tail=3, slots=40, fresh=(1, 4),
                  agent=list(range(n - 1)) + [3]).up().call(lib)
        _check_heads(c, lib, [0, 17, heads - 1])


def test_chunk_long(torch, lib):
    Delta(torch, 21, [6000], 1, 2, 64, slots=1, fresh=(0,)).up().call(lib).check(lib)


@pytest.mark.parametrize("scale", [1e-3, 200.0, 4000.0])
def test_chunk_small_and_large_values(torch, lib, scale):
    """Values from far below 1 to near the end of fp16: the state follows them."""
    Delta(torch, 5, [200, 70], 1, 2, 128, scale=scale).up().call(lib).check(lib)


@pytest.mark.parametrize("b,spread", [(-4, 1), (-6, 1), (-8, 1), (-10, 0), (-14, 0), (-18, 0), (-40, 0), (-80, 0)])
@pytest.mark.parametrize("lens,heads,d", [([64], 2, 128), ([40, 20], 4, 64), ([200, 70], 2, 128), ([330], 4, 64)])
def test_chunk_small_rates(torch, lib, b, spread, lens, heads, d):
    """Heads that write little, from a state of zeros: the state is then far below the values, and as exact
    in parts of itself. The bound is the sums' own error in parts of a head's largest entry at the end,
    which is the largest on the way but for a small factor, since what is written is alike in all rows."""
    c = Delta(torch, 33 + d, lens, 2, heads, d, fresh=range(len(lens)))
    c.b[:] = b + spread * c.b
    c.up().call(lib)
    want, state, faults, _ = c.want()
    out, S = c.got()
    for slot in c.agent:
        size = np.abs(state[slot]).max(axis=(1, 2))
        far = 4 * np.sqrt(d * max(lens)) * 2.0 ** -24 * size
        off = np.abs(S[slot] - state[slot]).max(axis=(1, 2))
        assert (off <= far).all(), (off / size, far / size)
    for i, slot in enumerate(c.agent):
        rows = slice(c.offset[i], c.offset[i + 1])
        far = 4 * np.sqrt(d * max(lens)) * 2.0 ** -24 * np.abs(state[slot]).max(axis=(1, 2))[None, :, None]
        assert (np.abs(out[rows] - want[rows]) - (c.round[rows] + far)).max() <= 0


@pytest.mark.parametrize("lens,heads", [([64], 2), ([200, 70], 2)])
def test_chunk_rates_and_values_of_many_sizes(torch, lib, lens, heads):
    """Large values at rates near zero beside small values at rates of 1/2: what a row writes is its rate
    times its value, and the column's numbers are as exact in parts of that."""
    c = Delta(torch, 34, lens, 2, heads, 128, fresh=range(len(lens)))
    small = np.random.default_rng(35).integers(0, 2, c.tokens).astype(bool)
    c.b[:] = 0
    c.b[small] = -30
    c.x[small, 4 * 128:] *= np.float16(1000)
    c.x[~small, 4 * 128:] *= np.float16(0.01)
    c.up().call(lib)
    want, state, _, _ = c.want()
    out, S = c.got()
    for i, slot in enumerate(c.agent):
        far = 4 * np.sqrt(128 * max(lens)) * 2.0 ** -24 * np.abs(state[slot]).max(axis=(1, 2))
        assert (np.abs(S[slot] - state[slot]).max(axis=(1, 2)) <= far).all()
        rows = slice(c.offset[i], c.offset[i + 1])
        assert (np.abs(out[rows] - want[rows]) - (c.round[rows] + far[None, :, None])).max() <= 0


@pytest.mark.parametrize("lens,heads,d", [([64], 2, 128), ([40, 20], 4, 64), ([200, 70], 2, 128)])
@pytest.mark.parametrize("fade", [-7.0, -14.0, -20.0])
def test_chunk_heads_that_forget_fast(torch, lib, lens, heads, d, fade):
    """Every row fades what came before by exp(fade), and every other row's values are 10^5 times the
    others': the weights of the rows before are far below 1, and as exact in parts of themselves.
    Beside its roundings (of 2^-11 of the terms' sizes) an output has the parts' errors: X, U, T and S
    2^-21 each, in parts of the same sizes, and of X and U 2^-28 of the largest rate times value, by way
    of weights whose sum is at most 2 / sqrt(d)."""
    c = Delta(torch, 37, lens, 2, heads, d)
    c.decay[:], c.dt[:], c.a[:] = fade, 0, np.log(np.e - 1)
    v = c.x[:, 4 * d:4 * d + heads * d]
    v[::2] *= np.float16(1000)
    v[1::2] *= np.float16(0.01)
    rate = 1 / (1 + np.exp(-c.b[:, :heads, None].astype(np.float64)))
    most = np.abs(rate * v.reshape(c.tokens, heads, d)).max()
    c.state[:] = 0
    c.up().call(lib)
    want, state, _, _ = c.want()
    out, S = c.got()
    far = 4 / np.sqrt(d) * 2.0 ** -28 * most
    off = np.abs(out - want) - (c.round * (1 + 2.0 ** -8) + far)
    assert off.max() <= 0, (off.max(), far)


@pytest.mark.parametrize("lens,heads,d", [([64], 2, 128), ([40, 20], 4, 64), ([200, 70], 2, 128)])
def test_chunk_keys_alike(torch, lib, lens, heads, d):
    """Keys that lean the same way, at rates near 1: each row takes most of the last one's value back. An
    output is the state's before its chunk and weights times the rows' beta (v - S^T k) of that state; the
    weights are rounded by 2^-11, and so is the output. What else there is are parts of 2^-21 of the factors
    of its products, some in a row, and the state's own roundings: 2^-18 of all terms' sizes."""
    rng = np.random.default_rng(39)
    c = Delta(torch, 39 + d, lens, 2, heads, d)
    lean = rng.normal(0, 1, 4 * d)
    c.x[:, :4 * d] = (3 * lean + rng.normal(0, 1, (c.tokens, 4 * d))).astype(np.float16)
    c.b[:] = 5 + 0.5 * c.b
    c.decay[:] = -0.05
    c.up().call(lib)
    want, state, _, top = c.want()
    out, S = c.got()
    assert np.abs(S - state).max() <= 4 * np.sqrt(d * max(lens)) * 2.0 ** -24 * top
    q, k, v = H.rows(c.x[:, :c.width], 2, heads, d, c.eps)
    g, beta = H.gates(c.a[:, :heads], c.b[:, :heads], c.decay.astype(np.float64), c.dt.astype(np.float64))
    size, far = np.zeros(out.shape), np.zeros(out.shape)
    for i in range(len(lens)):
        for h in range(heads):
            s = c.state[c.agent[i], h].astype(np.float64)
            for lo in range(c.offset[i], c.offset[i + 1], 64):
                at = slice(lo, min(lo + 64, c.offset[i + 1]))
                K, Q, B, G = k[at, h], q[at, h], beta[at, h], np.cumsum(g[at, h])
                fade = np.tril(np.exp(np.minimum(G[:, None] - G[None], 0)))
                T = np.linalg.inv(np.eye(len(G)) + np.tril(B[:, None] * (K @ K.T) * fade, -1))
                X = B[:, None] * (v[at, h] - np.exp(G)[:, None] * (K @ s))
                N, all_x = (Q @ K.T) * fade, B[:, None] * (np.abs(v[at, h]) + np.exp(G)[:, None] * (np.abs(K) @ np.abs(s)))
                size[at, h] = np.abs(N @ T) @ np.abs(X)
                far[at, h] = np.abs(N) @ np.abs(T) @ all_x + np.exp(G)[:, None] * (np.abs(Q) @ np.abs(s))
                s = np.exp(G[-1]) * s + (K * np.exp(G[-1] - G)[:, None]).T @ (T @ X)
    off = np.abs(out - want) - (2.0 ** -11 * (np.abs(out) + size) + 2.0 ** -25 + 2.0 ** -18 * far)
    assert off.max() <= 0, (off.max(), np.sqrt(((out - want) ** 2).mean() / (want ** 2).mean()))


@pytest.mark.parametrize("step", [False, True])
def test_rows_of_subnormal_values(torch, lib, step):
    """q and k whose values are all below fp16's smallest normal number are brought to length all the same."""
    c = Delta(torch, 19, [1] * 5 if step else [150, 3], 1, 2, 128)
    c.x[:, :256] = (c.x[:, :256].astype(np.float32) * 2.0 ** -18).astype(np.float16)
    c.eps = 1e-14
    c.up().call(lib, step=step).check(lib)


@pytest.mark.parametrize("values", [0.0, 2.0 ** -24, 1.0])
@pytest.mark.parametrize("state", [1e-20, 1e-9, 1e30])
def test_chunk_states_far_from_one(torch, lib, state, values):
    """The state's columns have a scale of their own: a state of any size is as exact, in parts of itself
    and of the values that join it."""
    c = Delta(torch, 18, [330], 1, 2, 128)
    c.state[:] = c.state * np.float32(state / 0.3)
    c.x[:, 2 * 128:] = np.sign(c.x[:, 2 * 128:].astype(np.float32)) * values
    c.decay[:] = -0.05
    c.up().call(lib)
    want, S, _, _ = c.want()
    out, got = c.got()
    # what a column holds at most: its state's length in the unit directions that the keys take, or the
    # sum of the values
    top = np.sqrt(128) * np.abs(c.state).max() + 330 * values
    far = 4 * np.sqrt(128 * 330) * 2.0 ** -24 * top
    assert np.abs(got - S).max() <= far, (np.abs(got - S).max(), far)
    big = np.abs(want) + c.round + far > 65504                      # no numbers of fp16
    assert (np.abs(out - want) - (c.round + far))[~big].max(initial=0) <= 0
    assert not np.isnan(out).any()


@pytest.mark.parametrize("decay,dt,b", [(0.0, 0.0, 30.0), (-1.0, -100.0, 30.0), (-16.0, 30.0, 0.0), (-1e4, 30.0, 0.0),
                                        (-1.0, -3.0, -200.0), (3.0, 0.0, 0.0)])
def test_chunk_gates_at_their_ends(torch, lib, decay, dt, b):
    """No decay, all of it, rates of 1 and 0; a decay above 0 counts as none."""
    c = Delta(torch, 6, [150], 1, 2, 128)
    c.decay[:], c.dt[:] = decay, dt
    c.b[:] = b
    c.up().call(lib).check(lib)


def test_chunk_one_key_again_and_again(torch, lib):
    """Every row has the same key: the inverse within a chunk is as far from 1 as it gets."""
    c = Delta(torch, 8, [140], 1, 1, 128)
    c.x[:, 128:256] = c.x[0, 128:256]
    c.b[:] = 4.0
    c.decay[:] = -0.01
    c.up().call(lib).check(lib)


def test_chunk_zero_rows(torch, lib):
    c = Delta(torch, 8, [80], 1, 2, 64)
    c.x[10:30] = 0
    c.up().call(lib).check(lib)


def test_chunk_equals_steps(torch, lib):
    """One slot's 70 tokens, at once and one after another."""
    c = Delta(torch, 12, [70], 2, 4, 128, slots=2, fresh=(0,)).up().call(lib).check(lib)
    whole, S = c.got()
    one = Delta(torch, 12, [70], 2, 4, 128, slots=2, fresh=(0,)).up()
    g = {k: v for k, v in one.dev.items()}
    for t in range(70):
        pos = _up(torch, [t], np.int32)
        assert lib.aotx_delta_step(p(g["x"][t]), one.stride, p(g["a"][t]), p(g["b"][t]), one.ab_stride, p(g["decay"]),
                                   p(g["dt"]), p(pos), p(g["agent"]), 1, 2, 4, 128, EPS, p(g["state"]), 2, p(g["out"][t]),
                                   None) == 0
    out, S1 = one.got()
    _, _, _, top = c.want()
    far = 8 * np.sqrt(128 * 70) * 2.0 ** -24 * top       # both sides' errors
    assert np.abs(S - S1).max() <= far
    assert (np.abs(out - whole) - (2 * c.round + far)).max() <= 0


def test_chunk_of_few_rows_is_steps_bit_by_bit(torch, lib):
    """Sequences of a few rows do what as many calls of aotx_delta_step do, in the same order: waves that
    run ahead of others leave what those still read."""
    n, rows = 64, 12
    c = Delta(torch, 17, [rows] * n, 16, 16, 128, slots=n).up()
    start = c.dev["state"].clone()
    KEEP.append(start)
    g = {k: p(v) for k, v in c.dev.items()}
    stepped = torch.zeros((rows, n, 16, 128), dtype=torch.float16, device="cuda")
    for t in range(rows):
        assert lib.aotx_delta_step(p(c.dev["x"][t]), rows * c.stride, p(c.dev["a"][t]), p(c.dev["b"][t]),
                                   rows * c.ab_stride, g["decay"], g["dt"], g["pos"], g["agent"], n, 16, 16, 128, EPS,
                                   g["state"], n, p(stepped[t]), None) == 0
    state = c.dev["state"].clone()
    for _ in range(4):
        c.dev["state"].copy_(start)
        c.call(lib)
        assert torch.equal(c.dev["out"].view(n, rows, 16, 128).transpose(0, 1), stepped)
        assert torch.equal(c.dev["state"], state)


def test_chunk_slots_missing_and_named_twice(torch, lib):
    c = Delta(torch, 13, [70, 5, 66, 0, 30, 9], agent=[3, 8, 3, 1, 1, 1], slots=8, fresh=(0,)).up().call(lib).check(lib)
    assert lib.aotx_model_faulted() == 3                 # 8 is no slot; 3 and 1 again (the empty one does not count)


@pytest.mark.parametrize("offset", [[0, 900, 1000], [50, 20, 100], [0xFFFFFFFF, 3, 0xFFFFFFF0], [100, 100, 100]])
def test_chunk_offsets_out_of_order_stay_in_bounds(torch, lib, offset):
    """Offsets past the rows end there, and a sequence that would end before it begins has none.
    What is left of the sequences has to be right."""
    c = Delta(torch, 14, [60, 40], tail=20)
    c.offset = np.array(offset, dtype=np.uint32)
    want, state, faults, top = c.want()
    c.offset = c.offset.view(np.int32)
    c.up().call(lib)
    out, S = c.got()
    far = 4 * np.sqrt(128 * 120) * 2.0 ** -24 * top + 1e-6
    assert np.abs(S - state).max() <= far and (np.abs(out - want) <= far + c.round).all()


BAD = pytest.mark.parametrize("what,bad", [("v", np.inf), ("v", np.nan), ("k", np.nan), ("k", -np.inf), ("q", np.nan),
                                         ("a", np.nan), ("b", np.nan), ("a", np.inf), ("a", -np.inf), ("b", np.inf)])


def _bad_value(torch, lib, lens, what, bad, at):
    """Row `at` of the first sequence gets a value that is no number. Rows before it, the second
    sequence, heads of other keys (or, from v, a and b, all other heads), and columns beside a bad
    value are what they are without it, bit for bit; a bad q reaches its row alone. In the column of
    a bad v the rows before it are right, but not always to the bit: a column's numbers are split
    into two parts at a scale that goes by the sizes of its values in four chunks, the replaced one
    among them, so they may round elsewhere, by 2^-21 a product, which the sums' own bound holds."""
    heads, d, n = 4, 128, lens[0]
    clean = Delta(torch, 15, lens, 2, heads, d).up().call(lib)
    base, S0 = clean.got()
    c = Delta(torch, 15, lens, 2, heads, d)
    col = {"q": 5, "k": 2 * d + 5, "v": 4 * d + d + 9}      # head 0's query, head 0's key, head 1's value 9
    if what in col:
        c.x[at, col[what]] = bad
    else:
        getattr(c, what)[at, 1] = bad                       # head 1's gate
    out, S = c.up().call(lib).got()
    hit = np.zeros(out.shape, dtype=bool)
    hit_state = np.zeros(S.shape, dtype=bool)
    slot = int(c.agent[0])
    if what == "q":
        hit[at, 0:2] = True
    elif what == "k":
        hit[at:n, 0:2] = True
        hit_state[slot, 0:2] = True
    elif what == "v":
        hit[at:n, 1, 9] = True
        hit_state[slot, 1, :, 9] = True
    else:
        hit[at:n, 1] = True
        hit_state[slot, 1] = True
    near = np.zeros(out.shape, dtype=bool)
    if what == "v":
        near[:at, 1, 9] = True
        want, _, _, top = clean.want()
        far = 4 * np.sqrt(d * n) * 2.0 ** -24 * top
        assert (np.abs(out[near] - want[near]) <= clean.round[near] + far).all()
    assert np.array_equal(out[~hit & ~near], base[~hit & ~near])
    assert np.array_equal(S[~hit_state], S0[~hit_state])
    if what not in ("a", "b") or np.isnan(bad):
        assert not np.isfinite(out[hit]).any()
        assert not np.isfinite(S[hit_state]).any()
    else:                                                   # an infinite gate is a decay or rate at its end
        want, state, _, top = c.want()
        far = 4 * np.sqrt(d * n) * 2.0 ** -24 * top
        assert np.abs(S - state).max() <= far
        assert (np.abs(out - want) - (c.round + far)).max() <= 0


@BAD
@pytest.mark.parametrize("at", [0, 37, 63, 64, 100])
def test_chunk_inf_and_nan_reach_no_earlier_row(torch, lib, what, bad, at):
    _bad_value(torch, lib, [130, 20], what, bad, at)


@BAD
@pytest.mark.parametrize("at", [0, 15, 16, 39])
def test_short_call_inf_and_nan_reach_no_earlier_row(torch, lib, what, bad, at):
    _bad_value(torch, lib, [40, 20], what, bad, at)


# ---- convolution -----------------------------------------------------------------------------

def _conv(torch, lib, seed, lens, channels, width, bias=False, lead=0, tail=0, pad=0, slots=8, fresh=(), agent=None,
          step=False):
    rng = np.random.default_rng(seed)
    tokens, n = lead + sum(lens) + tail, len(lens)
    x = rng.normal(0, 1, (tokens, channels + pad)).astype(np.float32)
    w = rng.normal(0, 0.5, (channels, width)).astype(np.float32)
    bb = rng.normal(0, 0.5, channels).astype(np.float32) if bias else None
    offset = (lead + np.concatenate([[0], np.cumsum(lens)])).astype(np.uint32)
    agent = np.array(rng.permutation(slots)[:n] if agent is None else agent, dtype=np.uint32)
    pos = np.array([0 if i in fresh else 4 + i for i in range(n)], dtype=np.uint32)
    state = rng.normal(0, 1, (slots, width - 1, channels)).astype(np.float32)
    want, S = np.full((tokens, channels), 7.0), state.astype(np.float64)
    faults = H.conv(x[:, :channels], w.astype(np.float64), bb, offset, pos, agent, S, want)
    out = torch.full((tokens, channels), 7.0, dtype=torch.float16, device="cuda")
    st = _up(torch, state, np.float32)
    rc = lib.aotx_delta_conv(p(_up(torch, x, np.float32)), channels + pad, p(_up(torch, w, np.float32)),
                             p(_up(torch, bb, np.float32)) if bias else None,
                             None if step else p(_up(torch, offset, np.int32)), p(_up(torch, pos, np.int32)),
                             p(_up(torch, agent, np.int32)), n, tokens, channels, width, p(st), slots, p(out), None)
    assert rc == 0
    torch.cuda.synchronize()
    got = out.cpu().numpy().astype(np.float64)
    # a sum of five fp32 products of size up to 3 sigma, then an exponential and a division: 16 steps
    far = 2.0 ** -11 * np.abs(want) + 2.0 ** -25 + 16 * 2.0 ** -24 * 8
    assert (np.abs(got - want) - far).max() <= 0
    assert np.array_equal(st.cpu().numpy().astype(np.float64), S)      # copies of rows
    assert lib.aotx_model_faulted() == faults
    return faults


@pytest.mark.parametrize("width", [2, 3, 4])
@pytest.mark.parametrize("channels", [4, 260, 1024, 8192])
def test_conv_lengths(torch, lib, width, channels):
    _conv(torch, lib, channels + width, [0, 1, 2, 3, 4, 15, 16, 0, 17, 70], channels, width, bias=width == 3, lead=2, tail=3,
          pad=8, slots=11, fresh=(1, 5, 8))


@pytest.mark.parametrize("lens", [[1] * 64, [14, 1, 1, 1, 30], [15, 40], [13, 2, 2, 2, 2, 2, 2, 2]])
def test_conv_sequences_around_a_run(torch, lib, lens):
    _conv(torch, lib, 5, lens, 128, 4, slots=64, fresh=(1,))


@pytest.mark.parametrize("width", [2, 3, 4])
@pytest.mark.parametrize("tokens,run", [(600, 2), (900, 3), (1300, 5), (2100, 8), (4099, 16)])
def test_conv_runs_of_rows(torch, lib, tokens, run, width):
    """A thread's run of 2 to 16 rows, sequences that begin, end and lie within one, and the last run short."""
    channels = 4096                                         # 4 workgroups a row: runs of tokens / 256 rows
    assert min(16, tokens * 4 // 1024) == run
    rng = np.random.default_rng(tokens + width)
    lens = [0, 1, run - 1, run, run + 1, 2, 3, 0, 1, 1, 4, 17, 2 * run, 1] + [int(n) for n in rng.integers(0, 2 * run, 30)]
    while sum(lens) > tokens - 40:
        lens.pop()
    lens.append(tokens - 9 - sum(lens))
    _conv(torch, lib, tokens, lens, channels, width, bias=width == 2, lead=4, tail=5, slots=60, fresh=range(0, 60, 3))


@pytest.mark.parametrize("lens,channels,width,pad", [([500, 1, 0, 3, 200, 16], 8192, 4, 0), ([700], 8200, 3, 4),
                                                     ([5400, 2, 60, 1, 17], 8192, 4, 0), ([3, 11000], 4104, 2, 4)])
def test_conv_past_the_caches(torch, lib, lens, channels, width, pad):
    """Calls whose rows go past the caches: out alone, and x too."""
    assert sum(lens) * channels * 6 > (256 << 20 if sum(lens) > 5000 else 32 << 20)
    _conv(torch, lib, 6, lens, channels, width, bias=True, lead=1, tail=2, pad=pad, slots=8, fresh=(0,))


def test_conv_refused_sequences_in_runs(torch, lib):
    """Slots that are missing or named twice where a run holds several sequences."""
    lens = [400, 3, 2, 1, 0, 250, 7, 1300, 5, 2]
    assert _conv(torch, lib, 9, lens, 4096, 4, lead=3, tail=30, agent=[2, 9, 2, 5, 5, 5, 1, 0, 0, 3], slots=8) == 4


@pytest.mark.parametrize("width", [2, 4])
def test_conv_in_a_graph(torch, lib, width):
    """A captured call of many rows, replayed with other rows, lengths and positions."""
    rng = np.random.default_rng(95)
    tokens, channels, slots = 2100, 4096, 4
    x = torch.zeros(tokens, channels, device="cuda")
    w = _up(torch, rng.normal(0, 0.5, (channels, width)), np.float32)
    offset, pos = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    agent = _up(torch, [2, 0, 3], np.int32)
    state = torch.zeros(slots, width - 1, channels, device="cuda")
    out = torch.zeros(tokens, channels, dtype=torch.float16, device="cuda")

    def call(s):
        assert lib.aotx_delta_conv(p(x), channels, p(w), None, p(offset), p(pos), p(agent), 3, tokens, channels, width,
                                   p(state), slots, p(out), s) == 0

    call(None)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        call(ctypes.c_void_p(side.cuda_stream))
    for at, begin in (([0, 5, 6, 2100], [0, 3, 9]), ([0, 1, 1, 3], [4, 0, 0]), ([20, 700, 1500, 1502], [1, 1, 0])):
        rows = rng.normal(0, 1, (tokens, channels)).astype(np.float32)
        kept = rng.normal(0, 1, (slots, width - 1, channels)).astype(np.float32)
        for t, v in ((x, rows), (state, kept)):
            t.copy_(torch.from_numpy(v))
        offset.copy_(torch.tensor(at, dtype=torch.int32))
        pos.copy_(torch.tensor(begin, dtype=torch.int32))
        out.fill_(7.0)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        got, S = out.clone(), state.clone()
        state.copy_(torch.from_numpy(kept))
        out.fill_(7.0)
        call(None)
        torch.cuda.synchronize()
        assert torch.equal(out, got) and torch.equal(state, S)
        want, S64 = np.full((tokens, channels), 7.0), kept.astype(np.float64)
        H.conv(rows, w.cpu().numpy().astype(np.float64), None, np.array(at), begin, [2, 0, 3], S64, want)
        far = 2.0 ** -11 * np.abs(want) + 2.0 ** -25 + 16 * 2.0 ** -24 * 8
        assert (np.abs(got.cpu().numpy().astype(np.float64) - want) - far).max() <= 0
        assert np.array_equal(S.cpu().numpy().astype(np.float64), S64)


@pytest.mark.parametrize("tokens", [1, 64])
def test_conv_step(torch, lib, tokens):
    _conv(torch, lib, tokens, [1] * tokens, 2048, 4, bias=True, slots=64, step=True, fresh=(2,))


def test_conv_slots_missing_and_named_twice(torch, lib):
    assert _conv(torch, lib, 8, [20, 3, 18, 0, 40, 2], 64, 4, agent=[2, 9, 2, 5, 5, 5], slots=8) == 3
    lib.aotx_model_forget()
    assert _conv(torch, lib, 8, [1, 1, 1], 64, 4, agent=[2, 2, 99], slots=8, step=True) == 2


# ---- gated norm ------------------------------------------------------------------------------

@pytest.mark.parametrize("heads,width", [(4, 64), (32, 128), (3, 8), (2, 72), (1, 256), (5, 504), (1, 512), (2, 520),
                                         (1, 4096), (1, 8192)])
@pytest.mark.parametrize("tokens,inplace", [(1, False), (7, True), (130, False)])
def test_norm_gate(torch, lib, heads, width, tokens, inplace):
    rng = np.random.default_rng(width + tokens)
    pad = 12 if tokens == 7 else 0
    x = rng.normal(0, 2, (tokens, heads, width)).astype(np.float16)
    x[0, 0] = 0
    z = rng.normal(0, 2, (tokens, heads * width + pad)).astype(np.float32)
    z[0, :3] = (1e4, -1e4, -120.0)
    w = rng.normal(1, 0.3, width).astype(np.float32)
    want = H.norm_gate(x, z[:, :heads * width].reshape(x.shape), w, EPS)
    xd = _up(torch, x, np.float16)
    out = xd if inplace else torch.full(x.shape, 7.0, dtype=torch.float16, device="cuda")
    assert lib.aotx_norm_gate(p(xd), p(_up(torch, z, np.float32)), heads * width + pad, p(_up(torch, w, np.float32)),
                              tokens, heads, width, EPS, p(out), None) == 0
    torch.cuda.synchronize()
    got = out.cpu().numpy().astype(np.float64)
    # the mean's sum, a root, a quotient, an exponential and four products: relative, 32 steps
    # of fp32 beside the last rounding
    assert (np.abs(got - want) - (2.0 ** -11 + 32 * 2.0 ** -24) * np.abs(want)).max() <= 2.0 ** -25


@pytest.mark.parametrize("tokens,heads,width", [(1 << 20, 17, 520), (1 << 20, 1040, 8)])
def test_norm_gate_more_rows_than_one_grid_row(torch, lib, tokens, heads, width):
    """Rows past 2^32 threads and outputs past 2^32 bytes: the last rows as any others."""
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("needs 80 GiB of device memory")
    rng = np.random.default_rng(3)
    x = torch.ones((tokens, heads, width), dtype=torch.float16, device="cuda")
    z = torch.zeros((tokens, heads * width), dtype=torch.float32, device="cuda")     # a gate of 0
    w = _up(torch, rng.normal(1, 0.3, width), np.float32)
    some = [0, tokens // 2 + 1, tokens - 1]
    xs, zs = rng.normal(0, 2, (3, heads, width)).astype(np.float16), rng.normal(0, 2, (3, heads * width)).astype(np.float32)
    for i, t in enumerate(some):
        x[t], z[t] = torch.from_numpy(xs[i]).cuda(), torch.from_numpy(zs[i]).cuda()
    assert lib.aotx_norm_gate(p(x), p(z), heads * width, p(w), tokens, heads, width, EPS, p(x), None) == 0
    torch.cuda.synchronize()
    want = H.norm_gate(xs, zs.reshape(xs.shape), w.cpu().numpy(), EPS)
    for i, t in enumerate(some):
        got = x[t].cpu().numpy().astype(np.float64)
        assert (np.abs(got - want[i]) - (2.0 ** -11 + 32 * 2.0 ** -24) * np.abs(want[i])).max() <= 2.0 ** -25
        x[t] = 0
    for part in x.split(1 << 16):
        assert not part.any()
    del x, z
    torch.cuda.empty_cache()


# ---- rotary turn -----------------------------------------------------------------------------

@pytest.mark.parametrize("d,rope_dim,spans,order,split,norm,factor", [
    (128, 128, (24, 20, 20), 0, True, True, False), (128, 64, (12, 10, 10), 1, True, True, False),
    (128, 128, (64,), 0, False, False, True), (64, 16, (2, 2, 2, 2), 1, False, True, False),
    (64, 64, (0, 32), 0, True, False, False), (128, 40, (7, 0, 13), 0, False, False, True),
    (64, 8, (4, 0, 0), 1, True, False, False), (128, 128, (62, 1, 1), 1, True, False, False)])
@pytest.mark.parametrize("tokens,heads,kv", [(1, 4, 1), (37, 32, 8), (3, 5, 0)])
def test_rope_axes(torch, lib, d, rope_dim, spans, order, split, norm, factor, tokens, heads, kv):
    rng = np.random.default_rng(d + rope_dim + tokens)
    width = (heads + 2 * kv) * d
    x = rng.normal(0, 1, (tokens, width + 4)).astype(np.float32)
    place = rng.integers(0, 1 << 20, (tokens, len(spans))).astype(np.uint32)
    place[0] = 0
    place[-1, -1] = 0xFFFFFFFF
    qn = rng.normal(1, 0.2, d).astype(np.float32) if norm else None
    kn = rng.normal(1, 0.2, d).astype(np.float32) if norm and tokens > 1 else None
    fac = rng.uniform(1, 8, rope_dim // 2).astype(np.float32) if factor else None
    how = aotx_amd.RopeHow(theta=1e6, eps=EPS, rope_dim=rope_dim, pairs=0 if split else 1, axes=len(spans), order=order,
                           span=(ctypes.c_uint32 * 4)(*spans))
    outs = [torch.full((tokens, n, d), 7.0, dtype=torch.float16, device="cuda") for n in (heads, max(kv, 1), max(kv, 1))]
    with_v = kv > 0 and tokens > 1

    def up(a):
        return None if a is None else p(_up(torch, a, np.float32))

    assert lib.aotx_rope_axes(up(x), width + 4, up(qn), up(kn), ctypes.byref(how), up(fac),
                              p(_up(torch, place.view(np.int32), np.int32)), tokens, heads, kv, d, p(outs[0]),
                              p(outs[1]) if kv else None, p(outs[2]) if with_v else None, None) == 0
    torch.cuda.synchronize()
    rows = x[:, :width].reshape(tokens, -1, d)
    parts = [(rows[:, :heads], qn, outs[0])]
    if kv:
        parts.append((rows[:, heads:heads + kv], kn, outs[1]))
    f64 = None if fac is None else fac.astype(np.float64)
    for part, nw, out in parts:
        want = H.rope_axes(part, nw, EPS, place, np.float32(1e6), rope_dim, split, list(spans), order, f64)
        got = out.cpu().numpy().astype(np.float64)
        # sines to 2^-22 (the fraction of a turn is rounded to 2^-25), a norm's 20 steps
        size = np.abs(want).max()
        assert (np.abs(got - want) - (2.0 ** -11 * np.abs(want) + 2.0 ** -25 + 32 * 2.0 ** -24 * size)).max() <= 0
    if with_v:
        assert np.array_equal(outs[2].cpu().numpy(), rows[:, heads + kv:].astype(np.float16))
    elif kv:
        assert (outs[2] == 7.0).all()


# ---- a layer of each kind ----------------------------------------------------------------------

class Layer:
    """A linear and a full attention layer's token mixing over Q8_0 products, on the device."""
    hidden, key_heads, heads, d, kv_heads, q_heads, width = 256, 2, 4, 64, 2, 4, 4

    def __init__(self, torch, lib, rows):
        self.torch, self.lib = torch, lib
        rng = np.random.default_rng(77)
        self.channels, self.inner = (2 * self.key_heads + self.heads) * self.d, self.heads * self.d
        self.att = (self.q_heads + 2 * self.kv_heads) * self.d
        sizes = {"mix": (self.channels, self.hidden), "gate": (self.inner, self.hidden), "ab": (2 * self.heads, self.hidden),
                 "out": (self.hidden, self.inner), "qkv": (self.att, self.hidden), "o": (self.hidden, self.q_heads * self.d)}
        self.w, self.w64 = {}, {}
        for i, (name, (n, k)) in enumerate(sizes.items()):
            blocks = quantize_q8(np.float32(0.08) * normal(900 + i, 0, n * k).reshape(n, k))
            raw = np.ascontiguousarray(blocks).view(np.uint8).reshape(n, k // 32, 34)
            scale = raw[..., :2].copy().view(np.float16).astype(np.float64)
            self.w64[name] = (raw[..., 2:].copy().view(np.int8) * scale).reshape(n, k)
            self.w[name] = (_up(torch, raw.reshape(-1), np.uint8), n, k)
        self.conv_w = rng.normal(0, 0.5, (self.channels, self.width)).astype(np.float32)
        self.decay, self.dt = -rng.uniform(1, 8, self.heads).astype(np.float32), rng.uniform(-5, -2, self.heads).astype(np.float32)
        self.norm = rng.normal(1, 0.1, self.d).astype(np.float32)
        f = np.float32
        self.dw = {n: _up(torch, getattr(self, n), f) for n in ("conv_w", "decay", "dt", "norm")}
        self.how = aotx_amd.RopeHow(theta=1e4, eps=EPS, rope_dim=32, pairs=0, axes=3, order=1, span=(ctypes.c_uint32 * 4)(6, 5, 5))
        z = dict(device="cuda")
        self.b = {"mix": torch.zeros(rows, self.channels, **z), "gate": torch.zeros(rows, self.inner, **z),
                  "ab": torch.zeros(rows, 2 * self.heads, **z), "qkv": torch.zeros(rows, self.att, **z),
                  "y": torch.zeros(rows, self.hidden, **z)}
        for n, w in (("c", self.channels), ("d", self.inner), ("n", self.inner), ("q", self.q_heads * self.d),
                     ("k", self.kv_heads * self.d), ("v", self.kv_heads * self.d), ("t", self.q_heads * self.d)):
            self.b[n] = torch.zeros(rows, w, dtype=torch.float16, **z)
        self.conv_state = torch.zeros(8, self.width - 1, self.channels, **z)
        self.state = torch.zeros(8, self.heads, self.d, self.d, **z)
        self.work = torch.zeros(int(lib.aotx_delta_work(rows, 8, self.heads, self.d)), dtype=torch.uint8, **z)

    def product(self, name, x, rows, y, s):
        w, n, k = self.w[name]
        assert self.lib.aotx_q8_gemv(p(w), n, k, p(x), rows, p(y), s) == 0

    def linear(self, x, rows, batch, s=None):
        b, lib = self.b, self.lib
        self.product("mix", x, rows, b["mix"], s)
        self.product("gate", x, rows, b["gate"], s)
        self.product("ab", x, rows, b["ab"], s)
        offset, pos, agent, seqs = batch
        assert lib.aotx_delta_conv(p(b["mix"]), self.channels, p(self.dw["conv_w"]), None, offset, pos, agent, seqs, rows,
                                   self.channels, self.width, p(self.conv_state), 8, p(b["c"]), s) == 0
        head = (p(b["c"]), self.channels, p(b["ab"]), ctypes.c_void_p(b["ab"].data_ptr() + 4 * self.heads), 2 * self.heads,
                p(self.dw["decay"]), p(self.dw["dt"]))
        if offset is None:
            assert lib.aotx_delta_step(*head, pos, agent, rows, self.key_heads, self.heads, self.d, EPS, p(self.state), 8,
                                       p(b["d"]), s) == 0
        else:
            assert lib.aotx_delta_chunk(*head, offset, pos, agent, seqs, rows, self.key_heads, self.heads, self.d, EPS,
                                        p(self.state), 8, p(self.work), self.work.numel(), p(b["d"]), s) == 0
        assert lib.aotx_norm_gate(p(b["d"]), p(b["gate"]), self.inner, p(self.dw["norm"]), rows, self.heads, self.d, EPS,
                                  p(b["n"]), s) == 0
        self.product("out", b["n"], rows, b["y"], s)
        return b["y"]

    def full(self, x, rows, place, pos, agent, s=None):
        b, lib = self.b, self.lib
        self.product("qkv", x, rows, b["qkv"], s)
        assert lib.aotx_rope_axes(p(b["qkv"]), self.att, p(self.dw["norm"]), p(self.dw["norm"]), ctypes.byref(self.how), None,
                                  place, rows, self.q_heads, self.kv_heads, self.d, p(b["q"]), p(b["k"]), p(b["v"]), s) == 0
        assert lib.aotx_kv_write(p(b["k"]), p(b["v"]), pos, agent, rows, self.kv_heads, self.d, 0, 1, s) == 0
        assert lib.aotx_attend_paged(p(b["q"]), pos, agent, rows, self.q_heads, self.kv_heads, self.d, 0, 1, p(b["t"]), s) == 0
        self.product("o", b["t"], rows, b["y"], s)
        return b["y"]


def test_linear_layer_prompt_then_tokens(torch, lib):
    """A prompt of 75 and one of 6 through a linear layer, then three single tokens each, against
    the whole sequences in 64 bits."""
    lens, more = [75, 6], 3
    rows = sum(lens)
    L = Layer(torch, lib, rows)
    rng = np.random.default_rng(78)
    xs = [rng.normal(0, 1, (n + more, L.hidden)).astype(np.float16) for n in lens]
    agent = _up(torch, [5, 2], np.int32)
    got = [[], []]
    x = _up(torch, np.concatenate([xs[0][:75], xs[1][:6]]), np.float16)
    y = L.linear(x, rows, (p(_up(torch, [0, 75, 81], np.int32)), p(_up(torch, [0, 0], np.int32)), p(agent), 2))
    torch.cuda.synchronize()
    y = y.cpu().numpy()
    got[0].append(y[:75].copy())
    got[1].append(y[75:].copy())
    for t in range(more):
        x = _up(torch, np.stack([xs[0][75 + t], xs[1][6 + t]]), np.float16)
        y = L.linear(x, 2, (None, p(_up(torch, [75 + t, 6 + t], np.int32)), p(agent), 2))
        torch.cuda.synchronize()
        for i in range(2):
            got[i].append(y[i:i + 1].cpu().numpy().copy())
    assert lib.aotx_model_faulted() == 0
    for i, xi in enumerate(xs):
        n = len(xi)
        x64 = xi.astype(np.float64)
        mix, gate, ab = (x64 @ L.w64[w].T for w in ("mix", "gate", "ab"))
        c = np.zeros((n, L.channels))
        H.conv(mix, L.conv_w.astype(np.float64), None, [0, n], [0], [0], np.zeros((1, 3, L.channels)), c)
        d = np.zeros((n, L.heads, L.d))
        H.delta(c, ab[:, :L.heads], ab[:, L.heads:], L.decay, L.dt, [0, n], [0], [0], L.key_heads, L.heads, L.d, EPS,
                np.zeros((1, L.heads, L.d, L.d)), d)
        y = H.norm_gate(d, gate.reshape(d.shape), L.norm, EPS).reshape(n, -1) @ L.w64["out"].T
        # four roundings to fp16 on the way and fp16-accurate products: the framework's 1e-2
        rms = np.sqrt((y ** 2).mean())
        err = np.abs(np.concatenate(got[i]) - y) / np.maximum(np.abs(y), rms)
        assert err.max() < 1e-2, err.max()


def test_full_layer_with_axes(torch, lib, orc):
    """Rows with three positions through the turn, the pages and paged attention: a row attends
    its own sequence's turned keys."""
    n = 40
    L = Layer(torch, lib, n)
    m = aotx_amd.KvMap()
    m.limit = 8
    assert lib.aotx_kv_open(ctypes.byref(m)) == 0
    try:
        assert lib.aotx_kv_request(3, layout_pages(n, 1, L.kv_heads, L.d)) == 1
        assert lib.aotx_kv_serve(ctypes.byref(m), None) == 1
        rng = np.random.default_rng(79)
        x = rng.normal(0, 1, (n, L.hidden)).astype(np.float16)
        place = np.stack([np.arange(n) // 4 + 100, 50 + np.arange(n) % 4, 60 + np.arange(n) // 8], 1).astype(np.int32)
        y = L.full(_up(torch, x, np.float16), n, p(_up(torch, place, np.int32)), p(_up(torch, np.arange(n), np.int32)),
                   p(_up(torch, np.full(n, 3), np.int32)))
        torch.cuda.synchronize()
        assert lib.aotx_model_faulted() == 0
        qkv = (x.astype(np.float64) @ L.w64["qkv"].T).reshape(n, -1, L.d)
        q, k = (H.rope_axes(part, L.norm, EPS, place, 1e4, 32, True, [6, 5, 5], 1)
                for part in (qkv[:, :L.q_heads], qkv[:, L.q_heads:L.q_heads + L.kv_heads]))
        v = qkv[:, L.q_heads + L.kv_heads:]
        att = np.zeros((n, L.q_heads, L.d))
        for t in range(n):
            for h in range(L.q_heads):
                s = k[:t + 1, h // 2] @ q[t, h] / np.sqrt(L.d)
                w = np.exp(s - s.max())
                att[t, h] = (w / w.sum()) @ v[:t + 1, h // 2]
        want = att.reshape(n, -1) @ L.w64["o"].T
        rms = np.sqrt((want ** 2).mean())
        err = np.abs(y.cpu().numpy() - want) / np.maximum(np.abs(want), rms)
        assert err.max() < 1e-2, err.max()
    finally:
        lib.aotx_kv_close(ctypes.byref(m))


def test_linear_layer_in_a_graph(torch, lib):
    """Two captured graphs of the layer (prompt rows and single tokens) that share every buffer,
    replayed several times in turn with eager calls of the same between them: every replay equals
    the eager result, bit for bit."""
    rows = 90
    L = Layer(torch, lib, rows)
    rng = np.random.default_rng(80)
    agent, seqs = _up(torch, [5, 2], np.int32), 2
    prompt = (p(_up(torch, [0, 70, 90], np.int32)), p(_up(torch, [0, 9], np.int32)), p(agent), seqs)
    token = (None, p(_up(torch, [70, 29], np.int32)), p(agent), seqs)
    x = _up(torch, rng.normal(0, 1, (rows, L.hidden)), np.float16)
    first = [t.clone() for t in (L.conv_state, L.state)]
    first[0].normal_(generator=torch.Generator("cuda").manual_seed(1))
    first[1].normal_(generator=torch.Generator("cuda").manual_seed(2))

    def again():
        L.conv_state.copy_(first[0])
        L.state.copy_(first[1])

    def now():
        torch.cuda.synchronize()
        return [t.clone() for t in (L.b["y"], L.state, L.conv_state)]

    side = torch.cuda.Stream()
    s = ctypes.c_void_p(side.cuda_stream)
    torch.cuda.synchronize()
    want = {}
    for name, batch, n in (("prompt", prompt, rows), ("token", token, 2)):
        again()
        torch.cuda.synchronize()
        L.linear(x, n, batch, s)
        want[name] = now()
    graphs = {}
    for name, batch, n in (("prompt", prompt, rows), ("token", token, 2)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            L.linear(x, n, batch, s)
        graphs[name] = g
    for turn in range(4):
        for name, n in (("prompt", rows), ("token", 2)):
            again()
            torch.cuda.synchronize()
            graphs[name].replay()
            got = now()
            for a, b in zip(got[1:], want[name][1:]):
                assert torch.equal(a, b), (turn, name)
            assert torch.equal(got[0][:n], want[name][0][:n]), (turn, name)
        again()
        torch.cuda.synchronize()
        L.linear(x, 2, token, s)
        assert torch.equal(now()[0][:2], want["token"][0][:2])


@pytest.mark.parametrize("lens", [[40], [5, 3, 11], [2, 1], [200, 1, 70], [700, 65]])
def test_chunk_forms_in_a_graph(torch, lib, lens):
    """Each form that a call takes (one launch, row by row, both), captured and replayed with other
    values, offsets and positions than it was captured with: as an eager call of those."""
    c, other = (Delta(torch, seed, lens, 2, 4, 128, fresh=(0,)).up() for seed in (30, 31))
    other.offset[:] = other.offset[::-1].max() - other.offset[::-1]         # the lengths in another order
    other.pos[:] = other.pos[::-1]
    other.up()
    need = lib.aotx_delta_work(c.tokens, len(lens), 4, 128)
    work = torch.empty(need, dtype=torch.uint8, device="cuda")
    KEEP.append(work)
    want = []
    for d in (c, other):
        eager = {k: v.clone() for k, v in d.dev.items()}
        d.call(lib, work=work)
        torch.cuda.synchronize()
        want.append((eager, d.dev["out"].clone(), d.dev["state"].clone()))
    side = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=side):
        c.call(lib, stream=ctypes.c_void_p(side.cuda_stream), work=work)
    for turn in range(4):
        inputs, out, state = want[turn % 2]
        for k, v in inputs.items():
            c.dev[k].copy_(v)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(c.dev["out"], out) and torch.equal(c.dev["state"], state), turn
    assert lib.aotx_model_faulted() == 0


def test_rope_axes_in_a_graph(torch, lib):
    """A captured turn, replayed with other places and rows in the same buffers: the frequencies
    are the call's, everything else is read at the replay."""
    rng = np.random.default_rng(90)
    tokens, heads, kv, d = 9, 4, 2, 64
    how = aotx_amd.RopeHow(theta=1e4, eps=EPS, rope_dim=32, pairs=1, axes=2, order=1, span=(ctypes.c_uint32 * 4)(8, 8))
    x = torch.zeros(tokens, (heads + 2 * kv) * d, device="cuda")
    place = torch.zeros(tokens, 2, dtype=torch.int32, device="cuda")
    q, k, v = (torch.zeros(tokens, n, d, dtype=torch.float16, device="cuda") for n in (heads, kv, kv))

    def call(s):
        assert lib.aotx_rope_axes(p(x), x.shape[1], None, None, ctypes.byref(how), None, p(place), tokens, heads, kv, d, p(q),
                                  p(k), p(v), s) == 0

    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        call(ctypes.c_void_p(side.cuda_stream))
    for turn in range(3):
        x.copy_(torch.from_numpy(rng.normal(0, 1, tuple(x.shape)).astype(np.float32)))
        place.copy_(torch.from_numpy(rng.integers(0, 9999, (tokens, 2)).astype(np.int32)))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (q, k, v)]
        call(None)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, (q, k, v))), turn
        assert q.abs().sum() > 0


def test_two_streams_of_their_own(torch, lib):
    """Calls on two streams at once, each with its own state and workspace."""
    calls = [Delta(torch, 30 + i, [300, 65], 2, 4, 128) for i in range(2)]
    for c in calls:
        c.up()
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    for c, st in zip(calls, streams):
        c.call(lib, stream=ctypes.c_void_p(st.cuda_stream))
    for c in calls:
        c.check(lib)
