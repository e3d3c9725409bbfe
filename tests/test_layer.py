"""The operators of a full layer and of a step's answer without a GPU: refused arguments, the
workspace's size, the structs' layout, and the oracle against formulas written another way."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

import aotx_amd as A
from aotx_amd.model import dequant_q8, quantize_q8
from oracle import layer as O

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
# nothing is read through these: an aligned address, and ones that are not
A256, A4, A2, A1 = 4096, 4100, 4098, 4097


def test_struct_layouts_match_c(tmp_path):
    structs = {"aotx_linear_how": A.LinearHow, "aotx_adjust_how": A.AdjustHow}
    src = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{ROOT}/include/aotx_layer.h"', 'int main(void){']
    for name, s in structs.items():
        src.append(f'printf("{name} %zu\\n", sizeof({name}));')
        src += [f'printf("{name}.{f} %zu\\n", offsetof({name}, {f}));' for f, _ in s._fields_]
    src += [f'printf("{n} %llu\\n", (unsigned long long){n});' for n in
            ("AOTX_ACT_NONE", "AOTX_ACT_SILU", "AOTX_ACT_GELU", "AOTX_ACT_GELU_TANH", "AOTX_ACT_RELU", "AOTX_LINEAR_F32",
             "AOTX_LINEAR_F16", "AOTX_LINEAR_ZERO", "AOTX_LINEAR_ROWS_MAX")]
    (tmp_path / "l.c").write_text("\n".join(src + ["return 0;}"]))
    subprocess.run(["gcc", "-o", str(tmp_path / "l"), str(tmp_path / "l.c")], check=True)
    out = subprocess.run([str(tmp_path / "l")], capture_output=True, text=True, check=True).stdout
    for key, val in (line.split() for line in out.splitlines()):
        if "." in key:
            s, f = key.split(".")
            assert getattr(structs[s], f).offset == int(val), key
        else:
            assert (ctypes.sizeof(structs[key]) if key in structs else getattr(A, key)) == int(val), key


LINEAR = dict(w=A256, up=A256, bias=A256, up_bias=A256, resid=A256, n=100, k=64, ldx=64, ldy=100, ldr=100, act=1, out=0,
              packed=1)
LCALL = dict(x=A256, m=3, y=2 * A256, work=A256, work_bytes=1 << 40, stream=None)


@pytest.mark.parametrize("change", [
    dict(w=None), dict(x=None), dict(y=None), dict(work=None), dict(n=0), dict(n=(1 << 18) + 1, ldy=1 << 19, ldr=1 << 19),
    dict(k=0), dict(k=48), dict(k=33), dict(k=(1 << 18) + 32, ldx=1 << 19), dict(ldx=63), dict(ldx=56), dict(ldx=68),
    dict(ldx=(1 << 22) + 8), dict(ldy=99), dict(ldr=99), dict(ldy=(1 << 22) + 1), dict(ldr=(1 << 22) + 1), dict(act=5),
    dict(out=2), dict(packed=2), dict(up=None), dict(w=A2), dict(up=A2), dict(packed=0, w=A1), dict(packed=0, up=A1),
    dict(x=A2), dict(x=A4), dict(y=A2), dict(out=1, y=A1), dict(resid=A2), dict(bias=A2), dict(up_bias=A2), dict(work=A4),
    dict(work_bytes=0), dict(work_bytes=A.AOTX_LINEAR_ZERO - 1), dict(m=(1 << 20) + 1), dict(y=A256, out=1),
    dict(y=A256, ldr=101)])
def test_linear_refusals(lib, change):
    how = A.LinearHow(**{**LINEAR, **{k: v for k, v in change.items() if k in LINEAR}})
    call = {**LCALL, **{k: v for k, v in change.items() if k in LCALL}}
    assert lib.aotx_q8_linear(ctypes.byref(how), *call.values()) == 1
    assert lib.aotx_q8_linear(None, *LCALL.values()) == 1


def test_linear_no_rows_is_nothing(lib):
    how = A.LinearHow(**LINEAR)
    assert lib.aotx_q8_linear(ctypes.byref(how), *{**LCALL, "m": 0}.values()) == 0


def test_linear_workspace(lib):
    """0 for refused sizes, bounded for the others; a call with a byte less is refused."""
    work = lib.aotx_q8_linear_work
    for bad in ((0, 64, 1, 0), (100, 48, 1, 0), (100, 0, 1, 0), ((1 << 18) + 1, 64, 1, 0), (100, (1 << 18) + 32, 1, 0),
                (100, 64, (1 << 20) + 1, 0)):
        assert work(*bad) == 0
    assert work(100, 64, 0, 0) == A.AOTX_LINEAR_ZERO
    for n, k in ((4096, 4096), (4096, 14336), (100, 14336), (1, 32)):
        for gated in (0, 1):
            for m in (1, 8, 33, 64, 100, 512, 513, 700, 2048):
                need = work(n, k, m, gated)
                assert need >= A.AOTX_LINEAR_ZERO
                assert need < A.AOTX_LINEAR_ZERO + (1 << 30)
                how = A.LinearHow(**{**LINEAR, "n": n, "k": k, "ldx": k, "ldy": n, "ldr": n, "up": A256 if gated else None,
                                     "up_bias": None})
                assert lib.aotx_q8_linear(ctypes.byref(how), *{**LCALL, "m": m, "work_bytes": need - 1}.values()) == 1


def test_pairs_of_any_number_of_rows_are_for_the_product_with_an_epilogue_alone(lib):
    """The plans of the step and of routed experts refuse a pair whose matrices are not whole tiles of 16 rows."""
    two = (ctypes.c_void_p * 2)(A256, A256)
    args, swiglu = ctypes.create_string_buffer(4096), 3
    for name in ("_Z15aotx_rgemv_planP15aotx_rgemv_argsPKPKvPKjjjij", "_Z22aotx_rgemv_plan_routedP15aotx_rgemv_argsPKPKvPKjjjij"):
        for n, want in ((96, 0), (100, 1), (8, 1), (112, 0)):
            for m in (1, 8, 32, 64, 300):
                assert getattr(lib, name)(args, two, (ctypes.c_uint * 2)(n, n), 2, 256, swiglu, m) == want, (name, n, m)
    for n in (96, 100, 8, 112):
        assert lib.aotx_q8_linear_work(n, 256, 8, 1) >= A.AOTX_LINEAR_ZERO


NORM = dict(x=A256, stride=64, w=A256, tokens=3, width=64, eps=1e-6, out=A256, stream=None)


@pytest.mark.parametrize("change", [
    dict(x=None), dict(w=None), dict(out=None), dict(width=0), dict(width=60), dict(width=32776, stride=32776),
    dict(stride=60), dict(stride=66), dict(tokens=(1 << 20) + 1), dict(eps=-1.0), dict(eps=float("nan")), dict(x=A4),
    dict(w=A4), dict(out=A4)])
def test_norm_rows_refusals(lib, change):
    assert lib.aotx_norm_rows(*{**NORM, **change}.values()) == 1


def test_norm_rows_no_rows_is_nothing(lib):
    assert lib.aotx_norm_rows(*{**NORM, "tokens": 0}.values()) == 0


def _append(**change):
    how = dict(theta=1e4, eps=1e-6, rope_dim=64, pairs=0, axes=1, order=0, span=(32, 0, 0))
    how.update({k: v for k, v in change.items() if k in how})
    span = how.pop("span")
    how = A.RopeHow(span=(ctypes.c_uint32 * 4)(*span), **how)
    args = dict(qkv=A256, stride=512, q_norm=None, k_norm=None, how=how, factor=None, gain=1.0, place=None, offset=A256,
                pos=A256, agent=A256, seqs=2, tokens=5, heads=2, kv_heads=1, head_dim=128, layer=0, layers=2, page=A256,
                q=A256, row_pos=A256, row_agent=A256, stream=None)
    args.update({k: v for k, v in change.items() if k in args})
    return args


@pytest.mark.parametrize("change", [
    dict(qkv=None), dict(how=None), dict(pos=None), dict(agent=None), dict(page=None), dict(q=None), dict(row_pos=None),
    dict(row_agent=None), dict(head_dim=96), dict(head_dim=256, stride=4096), dict(heads=0), dict(kv_heads=0),
    dict(heads=1025, stride=1 << 18), dict(kv_heads=1025, stride=1 << 19), dict(tokens=(1 << 20) + 1), dict(stride=508),
    dict(stride=514), dict(seqs=65), dict(offset=None, seqs=2, tokens=5), dict(offset=None, seqs=65, tokens=65),
    dict(rope_dim=0, span=(0,)), dict(rope_dim=12, span=(6,)), dict(rope_dim=136, span=(68,)), dict(pairs=2), dict(axes=0),
    dict(axes=5), dict(axes=3, span=(12, 10, 10)), dict(order=2), dict(span=(31,)), dict(theta=0.0),
    dict(theta=float("inf")), dict(eps=-1.0), dict(gain=0.0), dict(gain=-1.0), dict(gain=float("inf")),
    dict(gain=float("nan")), dict(layer=2), dict(layer=0, layers=0), dict(qkv=A4), dict(q=A4), dict(q_norm=A4),
    dict(k_norm=A4), dict(heads=1, kv_heads=256, stride=(1 + 512) * 128)])
def test_append_refusals(lib, change):
    assert lib.aotx_kv_append(*_append(**change).values()) == 1


@pytest.mark.parametrize("change", [dict(tokens=0), dict(seqs=0)])
def test_append_no_rows_is_nothing(lib, change):
    assert lib.aotx_kv_append(*_append(**change).values()) == 0


ADJUST = dict(sample=A256, agent=A256, list=A256, length=A256, lists=64, list_stride=100, bias_at=A256, bias_token=A256,
              bias=A256, biases=4, mask=A256, mask_of=A256, masks=2, mask_stride=4)
ACALL = dict(logits=A256, ld=100, rows=2, vocab=100, out=2 * A256, ld_out=100, stream=None)


@pytest.mark.parametrize("change", [
    dict(logits=None), dict(out=None), dict(vocab=0), dict(vocab=(1 << 20) + 1, ld=1 << 21, ld_out=1 << 21, mask_stride=1 << 16),
    dict(rows=4097), dict(ld=99), dict(ld_out=99), dict(ld=(1 << 22) + 1), dict(ld_out=(1 << 22) + 1), dict(out=A256, ld=101),
    dict(list=None), dict(length=None), dict(list_stride=(1 << 20) + 1), dict(bias_token=None), dict(bias=None),
    dict(mask_stride=3), dict(logits=A2), dict(out=A2), dict(sample=A4), dict(agent=A2), dict(list=A2), dict(length=A2),
    dict(bias_at=A2), dict(bias_token=A2), dict(bias=A2), dict(mask=A2), dict(mask_of=A2)])
def test_adjust_refusals(lib, change):
    how = A.AdjustHow(**{**ADJUST, **{k: v for k, v in change.items() if k in ADJUST}})
    call = {**ACALL, **{k: v for k, v in change.items() if k in ACALL}}
    assert lib.aotx_logits_adjust(ctypes.byref(how), *call.values()) == 1
    assert lib.aotx_logits_adjust(None, *ACALL.values()) == 1


def test_adjust_no_rows_is_nothing(lib):
    assert lib.aotx_logits_adjust(ctypes.byref(A.AdjustHow(**ADJUST)), *{**ACALL, "rows": 0}.values()) == 0


# ---- the oracle ------------------------------------------------------------------------------

def test_oracle_values_are_the_readers():
    rng = np.random.default_rng(1)
    raw = quantize_q8(rng.normal(0, 1, (5, 96)).astype(np.float32))
    assert np.array_equal(O.q8_values(raw, 5, 96), dequant_q8(raw, 96).astype(np.float64))


def test_oracle_activations_at_known_places():
    x = np.array([-30.0, -1.0, 0.0, 1.0, 30.0])
    assert np.allclose(O.act(x, 1)[0], x / (1 + np.exp(-x)))
    assert np.allclose(O.act(x, 2)[0], [0, -0.15865525393145707, 0, 0.8413447460685429, 30])
    assert np.allclose(O.act(x, 3)[0], [0, -0.15880800939172324, 0, 0.8411919906082768, 30])
    assert np.array_equal(O.act(x, 4)[0], [0, 0, 0, 1, 30]) and O.act(x, 0)[0] is x
    # the bounds of the slopes
    y = np.linspace(-10, 10, 20001)
    for kind in range(1, 5):
        v, slope = O.act(y, kind)
        assert np.abs(np.diff(v) / np.diff(y)).max() <= slope


def test_oracle_adjust_is_the_ticks(orc):
    """The decode tick's oracle (fp32) says the same."""
    rng = np.random.default_rng(2)
    row = rng.normal(0, 3, 50).astype(np.float32)
    tokens = rng.integers(0, 12, 40).astype(np.int32)
    for presence, frequency, repeat, window in ((0.5, 0.1, 1.3, 8), (0, 0, 1.2, 64), (0.3, 0, 1, 5), (0, 0.2, 0.9, 0)):
        want = orc.pick_adjust(row.copy(), tokens, presence, frequency, repeat, window)
        z, far = O.adjust(row, [np.float32(v) for v in (presence, frequency, repeat, window)], tokens.tolist())
        assert (np.abs(z - want) <= far).all()


def test_oracle_places_are_the_layout():
    """Position by position and layer by layer, a slot's blocks fill its pages in order."""
    table = np.full((64, 640), -1, dtype=np.int64)
    table[3, :4] = [2 << 21, 0, 1 << 21, 3 << 21]
    kv, d, layers = 4, 64, 3
    per = (2097152 - 256) // (2 * kv * 16 * d * 2)
    seen = set()
    for pos in range(0, per * 4 // layers * 16, 16):
        for layer in range(layers):
            at = O.places(3, pos, table, layer, layers, kv, d)
            assert at not in seen
            seen.add(at)
            block = pos // 16 * layers + layer
            assert at * 2 == table[3, block // per] + 256 + block % per * 2 * kv * 16 * d * 2
            assert O.places(3, pos + 5, table, layer, layers, kv, d) == at + 5 * d
    assert O.places(3, per * 4 * 16, table, 0, layers, kv, d) is None and O.places(2, 0, table, 0, layers, kv, d) is None
