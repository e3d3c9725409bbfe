"""The operators of hybrid models' layers without a GPU: the oracle against formulas written
another way, refused arguments, the workspace's size and the struct's layout."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

import aotx_amd
from oracle import hybrid as H

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _delta_inputs(rng, rows, key_heads, heads, d):
    x = rng.normal(0, 1, (rows, (2 * key_heads + heads) * d))
    return (H.silu(x).astype(np.float16), rng.normal(0, 1, (rows, heads)), rng.normal(0, 1, (rows, heads)),
            -rng.uniform(0.5, 8, heads), rng.normal(-3, 1, heads))


@pytest.mark.parametrize("rows", [1, 63, 64, 65, 200])
def test_oracle_chunks_equal_tokens(rows):
    """The chunked formula and the token-by-token one are the same numbers in 64 bits: their
    difference is rounding, below 1e-12 of the largest state entry for some hundred rows."""
    rng = np.random.default_rng(rows)
    x, a, b, decay, dt = _delta_inputs(rng, rows, 2, 4, 16)
    S = rng.normal(0, 0.3, (1, 4, 16, 16))
    want, W = H.delta_chunked(x, a, b, decay, dt, 2, 4, 16, 1e-6, S[0])
    out = np.zeros((rows, 4, 16))
    state = S.copy()
    faults, top, _ = H.delta(x, a, b, decay, dt, [0, rows], [5], [0], 2, 4, 16, 1e-6, state, out)
    assert faults == 0
    assert np.abs(out - want).max() < 1e-12 * top
    assert np.abs(state[0] - W).max() < 1e-12 * top


def test_oracle_delta_recalls_what_it_stored():
    """beta 1, no decay, orthogonal keys: a query with a stored key gets its value back (over
    sqrt(d), the query's scale); a second value for a key replaces the first."""
    d = 8
    x = np.zeros((3, 3 * d))
    x[0, d + 2], x[0, 2 * d:] = 1, np.arange(d)          # k = e2
    x[1, d + 5], x[1, 2 * d:] = 1, 10 + np.arange(d)     # k = e5
    x[2, d + 2], x[2, 2 * d:] = 1, 20 + np.arange(d)     # k = e2 again
    x[:, 2] = 1                                          # q = e2
    state, out = np.zeros((1, 1, d, d)), np.zeros((3, 1, d))
    H.delta(x, np.full((3, 1), -1e3), np.full((3, 1), 1e3), np.array([-1.0]), np.zeros(1), [0, 3],
            [0], [0], 1, 1, d, 0.0, state, out)
    assert np.allclose(out[:, 0] * np.sqrt(d), [np.arange(d), np.arange(d), 20 + np.arange(d)])
    assert np.allclose(state[0, 0, 5], 10 + np.arange(d))


def test_oracle_conv_pieces_equal_whole():
    rng = np.random.default_rng(3)
    x, w = rng.normal(0, 1, (9, 6)), rng.normal(0, 1, (6, 4))
    whole, part = np.zeros((9, 6)), np.zeros((9, 6))
    one, two = rng.normal(0, 1, (2, 3, 6)), None
    two = one.copy()
    H.conv(x, w, None, [0, 9], [0], [1], one, whole)
    for lo, hi in ((0, 2), (2, 3), (3, 9)):
        H.conv(x[lo:hi], w, None, [0, hi - lo], [lo], [1], two, part[lo:hi])
    assert np.allclose(whole, part) and np.array_equal(one, two)
    t, c = 5, 2
    assert np.isclose(whole[t, c], H.silu(sum(x[t - 3 + j, c] * w[c, j] for j in range(4))))


def test_oracle_rope_keeps_lengths_and_differences():
    """A turn keeps every pair's length, and with one axis the product of two turned rows goes
    by the difference of their places alone."""
    rng = np.random.default_rng(4)
    q, k = rng.normal(0, 1, (2, 1, 1, 64))
    for split in (True, False):
        def at(x, p):
            return H.rope_axes(x, None, 0.0, np.array([[p]]), 1e4, 64, split, [32], 0)[0, 0]
        assert np.isclose((at(q, 7) ** 2).sum(), (q ** 2).sum())
        assert np.isclose(at(q, 1007) @ at(k, 1000), at(q, 7) @ at(k, 0))
    assert H.axis_of([3, 3, 2], 1, 8) == [0, 1, 2, 0, 1, 2, 0, 1]
    assert H.axis_of([6, 1, 1], 1, 8) == [0, 1, 2, 0, 0, 0, 0, 0]
    assert H.axis_of([3, 3, 2], 0, 8) == [0, 0, 0, 1, 1, 1, 2, 2]


# ---- refusals: nothing is read through these addresses ---------------------------------------

A16, A4 = 4096, 4100        # an aligned address and one that is not
STEP = dict(qkv=A16, stride=512, a=A16, b=A16, ab_stride=2, decay=A16, dt=A16, pos=A16, agent=A16,
            tokens=4, key_heads=1, heads=2, head_dim=128, eps=1e-6, state=A16, slots=8, out=A16,
            stream=None)
CHUNK = dict(qkv=A16, stride=512, a=A16, b=A16, ab_stride=2, decay=A16, dt=A16, offset=A16, pos=A16,
             agent=A16, seqs=2, tokens=70, key_heads=1, heads=2, head_dim=128, eps=1e-6, state=A16,
             slots=8, work=A16, work_bytes=1 << 40, out=A16, stream=None)
CONV = dict(x=A16, stride=64, w=A16, bias=None, offset=A16, pos=A16, agent=A16, seqs=2, tokens=9,
            channels=64, width=4, state=A16, slots=8, out=A16, stream=None)
NORM = dict(x=A16, z=A16, z_stride=256, w=A16, tokens=3, heads=2, width=128, eps=1e-6, out=A16, stream=None)


def _rope(**change):
    how = dict(theta=1e4, eps=1e-6, rope_dim=64, pairs=0, axes=3, order=0, span=(12, 10, 10))
    how.update({k: v for k, v in change.items() if k in how})
    span = how.pop("span")
    how = aotx_amd.RopeHow(span=(ctypes.c_uint32 * 4)(*span), **how)
    args = dict(qkv=A16, stride=512, q_norm=None, k_norm=None, how=how, factor=None, place=A16, tokens=5,
                heads=2, kv_heads=1, head_dim=128, q=A16, k=A16, v=A16, stream=None)
    args.update({k: v for k, v in change.items() if k in args})
    return args


@pytest.mark.parametrize("change", [
    dict(qkv=None), dict(a=None), dict(b=None), dict(decay=None), dict(dt=None), dict(pos=None),
    dict(agent=None), dict(state=None), dict(out=None), dict(qkv=A4), dict(state=A4), dict(out=A4),
    dict(head_dim=96), dict(head_dim=0), dict(heads=3, key_heads=2), dict(heads=0), dict(key_heads=0),
    dict(heads=512, stride=1 << 20), dict(stride=511), dict(stride=504), dict(stride=516), dict(ab_stride=1),
    dict(eps=0.0), dict(eps=1e-31), dict(eps=float("nan")), dict(slots=0), dict(slots=65), dict(stride=(1 << 22) + 8)])
def test_delta_refusals(lib, change):
    assert lib.aotx_delta_step(*{**STEP, **change}.values()) == 1
    assert lib.aotx_delta_chunk(*{**CHUNK, **change}.values()) == 1


def test_delta_call_refusals(lib):
    assert lib.aotx_delta_step(*{**STEP, "tokens": 65}.values()) == 1
    for change in (dict(seqs=65), dict(tokens=(1 << 20) + 1), dict(offset=None), dict(work=None), dict(work=A16 + 128),
                   dict(work_bytes=lib.aotx_delta_work(70, 2, 2, 128) - 1)):
        assert lib.aotx_delta_chunk(*{**CHUNK, **change}.values()) == 1, change
    # nothing to do is no refusal
    assert lib.aotx_delta_step(*{**STEP, "tokens": 0}.values()) == 0
    assert lib.aotx_delta_chunk(*{**CHUNK, "tokens": 0}.values()) == 0
    assert lib.aotx_delta_chunk(*{**CHUNK, "seqs": 0}.values()) == 0


@pytest.mark.parametrize("change", [
    dict(x=None), dict(w=None), dict(pos=None), dict(agent=None), dict(state=None), dict(out=None), dict(x=A4),
    dict(w=A4), dict(bias=A4), dict(state=A4), dict(out=A4), dict(channels=0), dict(channels=62), dict(stride=60),
    dict(stride=66), dict(width=1), dict(width=5), dict(seqs=65), dict(slots=0), dict(slots=65),
    dict(tokens=(1 << 20) + 1), dict(offset=None), dict(channels=(1 << 20) + 4, stride=(1 << 20) + 4),
    dict(tokens=1 << 20, channels=(1 << 17) + 4, stride=(1 << 17) + 4)])
def test_conv_refusals(lib, change):
    assert lib.aotx_delta_conv(*{**CONV, **change}.values()) == 1
    assert lib.aotx_delta_conv(*{**CONV, "tokens": 0}.values()) == 0


@pytest.mark.parametrize("change", [
    dict(x=None), dict(z=None), dict(w=None), dict(out=None), dict(x=A4), dict(z=A4), dict(w=A4), dict(out=A4),
    dict(width=0), dict(width=124), dict(width=8200, z_stride=16400), dict(heads=0), dict(z_stride=252),
    dict(z_stride=258), dict(eps=-1.0), dict(eps=float("nan")), dict(tokens=(1 << 20) + 1),
    dict(heads=65537, width=8, z_stride=1 << 20)])
def test_norm_gate_refusals(lib, change):
    assert lib.aotx_norm_gate(*{**NORM, **change}.values()) == 1
    assert lib.aotx_norm_gate(*{**NORM, "tokens": 0}.values()) == 0


@pytest.mark.parametrize("change", [
    dict(qkv=None), dict(how=None), dict(place=None), dict(q=None), dict(k=None), dict(qkv=A4), dict(q=A4),
    dict(k=A4), dict(v=A4), dict(q_norm=A4), dict(k_norm=A4), dict(head_dim=96), dict(heads=0), dict(stride=508),
    dict(stride=514), dict(kv_heads=0), dict(theta=0.0), dict(theta=float("inf")), dict(theta=float("nan")),
    dict(eps=-1.0), dict(rope_dim=0), dict(rope_dim=60), dict(rope_dim=136, span=(48, 10, 10)), dict(pairs=2),
    dict(axes=0), dict(axes=5), dict(order=2), dict(span=(12, 10, 9)), dict(span=(2 ** 32 - 1, 2, 31)),
    dict(tokens=(1 << 20) + 1)])
def test_rope_axes_refusals(lib, change):
    assert lib.aotx_rope_axes(*_rope(**change).values()) == 1
    assert lib.aotx_rope_axes(*_rope(tokens=0).values()) == 0


def test_delta_work_grows_with_the_call(lib):
    w = lib.aotx_delta_work
    assert w(1, 1, 1, 64) > 0
    assert w(8192, 1, 32, 128) >= w(512, 1, 32, 128) >= w(512, 1, 2, 64)
    assert w(512, 64, 32, 128) >= w(512, 1, 32, 128)


def test_rope_how_layout(tmp_path):
    src = '#include <stdio.h>\n#include <stddef.h>\n#include "%s/include/aotx_hybrid.h"\nint main(void){printf("%%zu", sizeof(aotx_rope_how));' % ROOT
    for name, _ in aotx_amd.RopeHow._fields_:
        src += 'printf(" %%zu", offsetof(aotx_rope_how, %s));' % name
    (tmp_path / "l.c").write_text(src + "return 0;}")
    subprocess.run(["gcc", "-o", str(tmp_path / "l"), str(tmp_path / "l.c")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "l")], capture_output=True, text=True, check=True).stdout.split()]
    R = aotx_amd.RopeHow
    assert got == [ctypes.sizeof(R)] + [getattr(R, n).offset for n, _ in R._fields_]
