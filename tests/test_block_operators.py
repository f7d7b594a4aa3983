"""The 8-bit linear path, the block norms and rotary positions without a GPU:
refused arguments, empty calls, and the host-side rotary frequencies."""

import math

import numpy as np
import pytest

import sam3cpp_b200 as s3t

A = 1 << 20          # an aligned address that nothing reads: refusals come before the device is touched


@pytest.fixture(scope="module", autouse=True)
def built():
    if not s3t.LIB_PATH.exists():
        pytest.skip("libs3t.so not built")


def eight(stride=256, scale_stride=256, data=A, scale=A):
    return s3t.Matrix(data, stride, scale, scale_stride)


def refused(match):
    return pytest.raises(s3t.S3TError, match=match)


QUANTIZE = dict(type=s3t.TYPE_F16, x=A, rows=5, cols=200, x_stride=200, block_rows=1, q=eight())


@pytest.mark.parametrize("change, match", [
    (dict(type=s3t.TYPE_E4M3), "F32, F16 or BF16"),
    (dict(type=8), "F32, F16 or BF16"),
    (dict(rows=-1), "negative"),
    (dict(cols=-1), "negative"),
    (dict(block_rows=64), "block_rows"),
    (dict(x=None), "device pointer"),
    (dict(x=A + 1), "aligned"),
    (dict(x_stride=199), "x_stride"),
    (dict(q=eight(data=None)), "data and scale"),
    (dict(q=eight(scale=None)), "data and scale"),
    (dict(q=eight(data=A + 8)), "16 bytes"),
    (dict(q=eight(stride=201)), "16 bytes"),
    (dict(q=eight(stride=192)), "below its columns"),
    (dict(q=eight(scale=A + 2)), "4-byte"),
    (dict(q=eight(scale_stride=4)), "scale stride"),
    (dict(rows=300, block_rows=128, q=eight(scale_stride=2)), "scale stride"),
    (dict(q=None), "data and scale"),
])
def test_quantize_refusals(change, match):
    a = {**QUANTIZE, **change}
    with refused(match):
        s3t.quantize_fp8(0, a["type"], a["x"], a["rows"], a["cols"], a["x_stride"], a["block_rows"], a["q"])


GEMM = dict(x=eight(), w=eight(), bias=None, m=5, n=200, k=200, act=0, y_type=s3t.TYPE_F16, y=s3t.Matrix(A, 200))


@pytest.mark.parametrize("change, match", [
    (dict(m=-1), "M >= 0"),
    (dict(n=-1), "N >= 0"),
    (dict(k=0), "K >= 1"),
    (dict(m=(1 << 30) + 1, x=eight(scale_stride=1 << 31)), "2\\^30"),
    (dict(act=2), "act"),
    (dict(y_type=8), "y must be"),
    (dict(x=None), "x: "),
    (dict(w=eight(stride=192)), "w: .*below"),
    (dict(x=eight(stride=257)), "x: .*16 bytes"),
    (dict(x=eight(scale_stride=4)), "x: .*scale stride"),
    (dict(w=eight(scale_stride=1)), "w: .*scale stride"),
    (dict(bias=A + 2), "bias"),
    (dict(y=s3t.Matrix(None, 200)), "y must be"),
    (dict(y=s3t.Matrix(A + 1, 200)), "y must be"),
    (dict(y=s3t.Matrix(A, 199)), "row stride of y"),
    (dict(y=None), "y must be"),
    (dict(y_type=s3t.TYPE_E4M3), "y: an 8-bit matrix"),
    (dict(y_type=s3t.TYPE_E4M3, y=eight(scale_stride=4)), "y: .*scale stride"),
])
def test_gemm_refusals(change, match):
    a = {**GEMM, **change}
    with refused(match):
        s3t.gemm_fp8(0, a["x"], a["w"], a["bias"], a["m"], a["n"], a["k"], a["act"], a["y_type"], a["y"])


NORM = dict(rows=5, dim=200, type=s3t.TYPE_F16, resid_type=s3t.TYPE_F32, u_type=s3t.TYPE_F16, flags=s3t.NORM_POST, eps=1e-5,
            resid_scale=1.0, branch_scale=1.0, y=A, y_stride=200, gate=A, gate_stride=200, gate_rows=1, x=A, x_stride=200,
            x_out=A, x_out_stride=200, u=s3t.Matrix(A, 200))


@pytest.mark.parametrize("change, match", [
    (dict(type=s3t.TYPE_E4M3), "type must"),
    (dict(resid_type=s3t.TYPE_BF16), "resid_type"),
    (dict(rows=-1), "rows"),
    (dict(rows=1 << 31), "rows"),
    (dict(dim=0), "dim"),
    (dict(dim=16385), "dim"),
    (dict(flags=16), "flags"),
    (dict(flags=s3t.NORM_GATE_TANH | s3t.NORM_GATE_SIGMOID), "not both"),
    (dict(flags=s3t.NORM_GATE_TANH, gate=None), "gate function"),
    (dict(eps=-1e-5), "eps"),
    (dict(eps=math.nan), "eps"),
    (dict(x=None), "x must"),
    (dict(x_stride=199), "x must"),
    (dict(x=A + 2), "x must"),
    (dict(y=None), "needs y"),
    (dict(y=None, flags=0), "needs y"),
    (dict(y=A + 1), "y must"),
    (dict(gate_stride=100), "gate must"),
    (dict(gate_rows=0), "gate_rows"),
    (dict(x_out=A + 16, x_out_stride=100), "x_out"),
    (dict(x_out_stride=208), "in place"),
    (dict(x_out=None, u=s3t.Matrix()), "nothing to write"),
    (dict(pre_weight=A + 2), "weights"),
    (dict(u_type=s3t.TYPE_BF16), "u_type"),
    (dict(u=s3t.Matrix(A, 199)), "u must"),
    (dict(u_type=s3t.TYPE_E4M3), "data and scale"),
    (dict(u_type=s3t.TYPE_E4M3, u=eight(scale_stride=4)), "scale stride"),
])
def test_norm_refusals(change, match):
    with refused(match):
        s3t.norm_residual(0, s3t.NormArgs(**{**NORM, **change}))


ROTARY = dict(freq=A, rot=32, positions=A, tokens=5, type=s3t.TYPE_F16, dim=64,
              q=s3t.RotaryView(A, A, 4, 256, 64, 256, 64), k=None, flags=0)


@pytest.mark.parametrize("change, match", [
    (dict(type=s3t.TYPE_E4M3), "type must"),
    (dict(dim=1), "head_dim"),
    (dict(dim=1026), "head_dim"),
    (dict(rot=31), "rot_dim"),
    (dict(rot=0), "rot_dim"),
    (dict(rot=66), "rot_dim"),
    (dict(flags=4), "flags"),
    (dict(tokens=-1), "tokens"),
    (dict(freq=None), "freq"),
    (dict(positions=A + 4), "positions"),
    (dict(q=None), "q must"),
    (dict(q=s3t.RotaryView(A, A, 0, 256, 64, 256, 64)), "heads"),
    (dict(q=s3t.RotaryView(None, A, 4, 256, 64, 256, 64)), "device pointers"),
    (dict(q=s3t.RotaryView(A + 1, A, 4, 256, 64, 256, 64)), "aligned"),
    (dict(q=s3t.RotaryView(A, A + 16, 4, -256, 64, 256, 64)), "negative"),
    (dict(q=s3t.RotaryView(A, A + 16, 4, 256, 64, 256, 32)), "at least head_dim"),
    (dict(k=s3t.RotaryView(A, A, 4, 256, 64, 512, 64)), "in place"),
    (dict(q=s3t.RotaryView(A, A + 16, 4, 256, 64, 64, 64)), "overlap"),           # token t, head h where t + 1, h - 1 is
    (dict(q=s3t.RotaryView(A, A + 16, 4, 256, 64, 64, 128)), "overlap"),
    (dict(q=s3t.RotaryView(A, A + 16, 4, 256, 64, 192, 256)), "overlap"),         # token 4, head 0 on token 0, head 3
    (dict(q=s3t.RotaryView(A, A + 16, 2, 256, 64, 1 << 62, (1 << 62) + 63)), "overlap"),
    (dict(q=s3t.RotaryView(A, A + 16, 2, 256, 64, (1 << 61) + 63, 1 << 61)), "overlap"),
    (dict(k=s3t.RotaryView(A + 4096, A, 4, 256, 64, 256, 64)), "over one another"),
    (dict(q=s3t.RotaryView(A, A + 4096, 4, 256, 64, 256, 64), k=s3t.RotaryView(A + 4096, A + 8192, 4, 256, 64, 256, 64)),
     "over one another"),
])
def test_rotary_refusals(change, match):
    a = {**ROTARY, **change}
    with refused(match):
        s3t.rotary(0, a["freq"], a["rot"], 1.0, a["positions"], a["tokens"], a["type"], a["dim"], a["q"], a["k"], a["flags"])


def test_empty_calls_succeed_without_a_device():
    s3t.quantize_fp8(0, s3t.TYPE_F32, A, 0, 200, 200, 1, eight())
    s3t.quantize_fp8(0, s3t.TYPE_F32, A, 5, 0, 0, 128, eight())
    s3t.gemm_fp8(0, eight(), eight(), None, 0, 200, 200, 0, s3t.TYPE_F16, s3t.Matrix(A, 200))
    s3t.gemm_fp8(0, eight(), eight(), None, 5, 0, 200, 0, s3t.TYPE_F16, s3t.Matrix(A, 200))
    s3t.norm_residual(0, s3t.NormArgs(**{**NORM, "rows": 0}))
    a = ROTARY
    s3t.rotary(0, A, 32, 1.0, A, 0, a["type"], 64, a["q"])


def test_empty_calls_take_the_null_pointers_of_empty_tensors():
    none = s3t.Matrix(None, 256, None, 256)
    for kind in (s3t.TYPE_F32, s3t.TYPE_BF16):
        s3t.quantize_fp8(0, kind, None, 0, 200, 200, 1, none)
        s3t.quantize_fp8(0, kind, None, 5, 0, 0, 1, none)
    for y_type in (s3t.TYPE_F32, s3t.TYPE_E4M3):
        s3t.gemm_fp8(0, none, eight(), A, 0, 200, 200, 1, y_type, none)
        s3t.gemm_fp8(0, eight(), none, None, 5, 0, 200, 0, y_type, none)
    empty = dict(rows=0, x=None, y=None, gate=None, x_out=None, u=none)
    s3t.norm_residual(0, s3t.NormArgs(**{**NORM, **empty}))
    s3t.norm_residual(0, s3t.NormArgs(**{**NORM, **empty, "flags": s3t.NORM_POST | s3t.NORM_GATE_TANH, "u_type": s3t.TYPE_E4M3}))
    v = s3t.RotaryView(None, None, 4, 256, 64, 256, 64)
    s3t.rotary(0, A, 32, 1.0, None, 0, s3t.TYPE_F16, 64, v, v)
    # what does not depend on the pointers is refused all the same
    with refused("block_rows"):
        s3t.quantize_fp8(0, s3t.TYPE_F32, None, 0, 200, 200, 64, none)
    with refused("act"):
        s3t.gemm_fp8(0, none, eight(), None, 0, 200, 200, 7, s3t.TYPE_F32, none)
    with refused("eps"):
        s3t.norm_residual(0, s3t.NormArgs(**{**NORM, **empty, "eps": -1.0}))
    with refused("rot_dim"):
        s3t.rotary(0, A, 31, 1.0, None, 0, s3t.TYPE_F16, 64, v)


@pytest.mark.parametrize("y_type", [s3t.TYPE_F16, s3t.TYPE_E4M3])
def test_empty_products_need_no_columns(y_type):
    none = s3t.Matrix(None, 0, None, 0)
    for m, n in ((0, 200), (5, 0), (0, 0)):
        s3t.gemm_fp8(0, none, none, None, m, n, 0, 0, y_type, none)
        with refused("K >= 1"):
            s3t.gemm_fp8(0, none, none, None, m, n, -1, 0, y_type, none)


WRAP = 1 << 32       # taken modulo 2^32 each of these sizes would be an empty or a valid call


@pytest.mark.parametrize("call", [
    lambda: s3t.quantize_fp8(0, s3t.TYPE_F32, A, 0, 200, 200, WRAP + 1, eight()),
    lambda: s3t.quantize_fp8(0, WRAP, A, 0, 200, 200, 1, eight()),
    lambda: s3t.quantize_fp8(0, s3t.TYPE_F32, A, 1 << 64, 200, 200, 1, eight()),
    lambda: s3t.gemm_fp8(0, eight(), eight(), None, WRAP, 200, 200, 0, s3t.TYPE_F16, s3t.Matrix(A, 200)),
    lambda: s3t.gemm_fp8(0, eight(), eight(), None, 5, -WRAP, 200, 0, s3t.TYPE_F16, s3t.Matrix(A, 200)),
    lambda: s3t.gemm_fp8(0, eight(), eight(), None, 0, 200, WRAP + 200, 0, s3t.TYPE_F16, s3t.Matrix(A, 200)),
    lambda: s3t.norm_residual(0, s3t.NormArgs(**{**NORM, "rows": 0, "dim": WRAP + 200})),
    lambda: s3t.norm_residual(0, s3t.NormArgs(0, WRAP + 200)),
    lambda: s3t.rotary(0, A, WRAP + 32, 1.0, A, 0, s3t.TYPE_F16, 64, ROTARY["q"]),
    lambda: s3t.rotary(0, A, 32, 1.0, A, 0, s3t.TYPE_F16, WRAP + 64, ROTARY["q"]),
    lambda: s3t.rotary(0, A, 32, 1.0, A, 1 << 64, s3t.TYPE_F16, 64, ROTARY["q"]),
    lambda: s3t.rotary(0, A, 32, 1.0, A, 0, s3t.TYPE_F16, 64, s3t.RotaryView(A, A, WRAP + 4, 256, 64, 256, 64)),
    lambda: s3t.rotary_frequencies(WRAP + 64),
])
def test_sizes_do_not_wrap(call):
    with refused("does not fit"):
        call()


def test_structure_fields_hold_what_they_are_given():
    a = s3t.NormArgs(7, 1024, s3t.TYPE_BF16, u_type=s3t.TYPE_E4M3, eps=0.5)
    assert (a.rows, a.dim, a.type, a.resid_type, a.u_type, a.eps) == (7, 1024, s3t.TYPE_BF16, 0, s3t.TYPE_E4M3, 0.5)
    a.dim = 1 << 20
    assert a.dim == 1 << 20
    with refused("does not fit"):
        a.dim = -(1 << 31) - 1
    assert a.dim == 1 << 20
    assert s3t.RotaryView(heads=4).heads == 4


def test_a_call_without_a_gpu_is_an_error():
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    with pytest.raises(s3t.S3TError):
        s3t.quantize_fp8(0, s3t.TYPE_F32, A, 5, 200, 200, 1, eight())


# ------------------------------------------------------ rotary frequencies ---

def test_frequencies_unscaled_and_linear():
    f, m = s3t.rotary_frequencies(64, 10000.0)
    want = 10000.0 ** (-2 * np.arange(32) / 64)
    np.testing.assert_allclose(f, want, rtol=1e-15)
    assert m == 1.0
    f4, m = s3t.rotary_frequencies(64, 10000.0, s3t.ROTARY_LINEAR, 4.0)
    np.testing.assert_allclose(f4, want / 4, rtol=1e-15)
    assert m == 1.0


def test_frequencies_by_base_keep_the_first_and_stretch_the_last():
    f, m = s3t.rotary_frequencies(64, 10000.0, s3t.ROTARY_BASE, 8.0)
    plain, _ = s3t.rotary_frequencies(64, 10000.0)
    # base' = base * factor^(d / (d - 2)): pair 0 unchanged, the last pair divided by the factor
    assert f[0] == 1.0 and m == 1.0
    np.testing.assert_allclose(f[-1], plain[-1] / 8.0, rtol=1e-12)
    assert s3t.rotary_frequencies(2, 10000.0, s3t.ROTARY_BASE, 8.0)[0] == [1.0]


def test_frequencies_by_parts():
    original, factor = 4096.0, 16.0
    f, m = s3t.rotary_frequencies(128, 10000.0, s3t.ROTARY_BY_PARTS, factor, original, 32.0, 1.0)
    plain, _ = s3t.rotary_frequencies(128, 10000.0)
    turns = original * plain / (2 * math.pi)
    keep = np.clip((turns - 1) / 31, 0, 1)
    np.testing.assert_allclose(f, plain * keep + plain / factor * (1 - keep), rtol=1e-14)
    np.testing.assert_array_equal(f[turns >= 32], plain[turns >= 32])
    np.testing.assert_array_equal(f[turns <= 1], plain[turns <= 1] / factor)
    assert m == np.float32(0.1 * math.log(factor) + 1)
    assert s3t.rotary_frequencies(128, 10000.0, s3t.ROTARY_BY_PARTS, 1.0, original)[1] == 1.0


@pytest.mark.parametrize("args, match", [
    ((63,), "rot_dim"), ((0,), "rot_dim"), ((1026,), "rot_dim"), ((64, 0.0), "base"), ((64, 1e4, 7), "scaling"),
    ((64, 1e4, s3t.ROTARY_LINEAR, 0.5), "factor"),
    ((64, 1e4, s3t.ROTARY_BY_PARTS, 2.0, 0.0), "original_len"),
    ((64, 1e4, s3t.ROTARY_BY_PARTS, 2.0, 4096.0, 1.0, 1.0), "fast > slow"),
])
def test_frequency_refusals(args, match):
    with refused(match):
        s3t.rotary_frequencies(*args)
