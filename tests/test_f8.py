"""8-bit floats, what needs no GPU: the code table, the rounding of the test oracle, and calls that are refused on the host."""
import ctypes as C
import types

import numpy as np
import pytest

import f8_util as F
import kalosm_b200 as kb


def test_code_table():
    assert np.array_equal(kb._f8_values(np.arange(256, dtype=np.uint8)), F.VALUES.astype(np.float32), equal_nan=True)
    assert F.VALUES[0x7E] == 448 and F.VALUES[0x01] == 2.0 ** -9 and F.VALUES[0x08] == 2.0 ** -6 and F.VALUES[0x38] == 1.0 and np.isnan(F.VALUES[0x7F])


def test_rounding_of_the_oracle():
    torch = pytest.importorskip("torch")
    v = np.concatenate([np.linspace(-448, 448, 200001), np.random.default_rng(0).standard_normal(100000) * 2.0 ** -7])
    v = np.concatenate([v, [17 / 16, 19 / 16, 2.0 ** -10, 3 * 2.0 ** -10, -2.0 ** -10]]).astype(np.float32)  # ties
    assert np.array_equal(F.e4m3(v.astype(np.float64)), torch.from_numpy(v).to(torch.float8_e4m3fn).double().numpy())


def test_blocks_of_the_oracle():
    v = np.random.default_rng(1).standard_normal((5, 300))
    codes, scales = F.quantise(v)
    F.check_rows(codes, scales, v, np.abs(v) * F.U)
    assert scales.shape == (5, 3) and np.all(np.abs(F.VALUES[codes]).max(1) == 448)
    wrong = codes.copy()
    wrong[3, 200] ^= 1
    with pytest.raises(AssertionError):
        F.check_rows(wrong, scales, v, np.abs(v) * F.U)
    with pytest.raises(AssertionError):
        F.check_rows(codes, scales * np.float32(1 + 1e-6), v, np.abs(v) * F.U)
    codes, scales = F.quantise(v, 4)
    assert scales.shape == (2, 3)


def _fake():
    return types.SimpleNamespace(lib=None, h=1)


def _refused(code, call):
    with pytest.raises(kb.FusorError) as e:
        call()
    assert e.value.code == code


def test_rows_are_checked():
    dev = _fake()

    def t(shape, kind, on=dev):
        return kb.Tensor(on, shape, kind, ptr=16)

    kb.F8Rows(dev, (2, 3, 130), t((6, 144), np.uint8), t((6, 2), np.float32))
    for codes, scales in [(t((6, 130), np.uint8), t((6, 2), np.float32)), (t((6, 128), np.uint8), t((6, 2), np.float32)),
                          (t((5, 144), np.uint8), t((6, 2), np.float32)), (t((6, 144), np.int8), t((6, 2), np.float32)),
                          (t((6, 144), np.uint8), t((6, 1), np.float32)), (t((6, 144), np.uint8), t((6, 2), np.float16)),
                          (t((6, 144), np.uint8, _fake()), t((6, 2), np.float32)), (t((6, 144), np.uint8), t((6, 2), np.float32, _fake()))]:
        _refused(kb.ERR_INVALID_SHAPE, lambda: kb.F8Rows(dev, (2, 3, 130), codes, scales))
    _refused(kb.ERR_INVALID_SHAPE, lambda: kb.F8Rows(dev, ()))
    _refused(kb.ERR_INVALID_SHAPE, lambda: kb.F8Matrix.from_tensors(t((6, 144), np.int8), t((1, 2), np.float32)))
    _refused(kb.ERR_INVALID_SHAPE, lambda: kb.F8Matrix.from_tensors(t((6, 144), np.uint8), t((1, 2), np.float32), 145))
    _refused(kb.ERR_INVALID_SHAPE, lambda: kb.F8Matrix.from_tensors(t((6, 144), np.uint8), t((6, 2), np.float32), 130))


def test_operations_check_their_tensors():
    dev = _fake()
    d = kb.Device.__new__(kb.Device)
    d.lib, d.h = None, 1

    def t(shape, kind=np.float32, on=None):
        return kb.Tensor(on or d, shape, kind, ptr=16)

    def rows(shape):
        return kb.F8Rows(d, shape, t((kb._rows_of(shape), -(-shape[-1] // 16) * 16), np.uint8), t((kb._rows_of(shape), -(-shape[-1] // 128))))

    x, w = t((4, 256)), t((256,))
    _refused(kb.ERR_UNSUPPORTED_DTYPE, lambda: d.quantize_f8(t((4, 256), np.float64)))
    _refused(kb.ERR_UNSUPPORTED_DTYPE, lambda: d.quantize_f8(t((4, 256), on=dev)))
    _refused(kb.ERR_INVALID_SHAPE, lambda: d.quantize_f8(x, out=rows((4, 128))))
    _refused(kb.ERR_INVALID_SHAPE, lambda: d.quantize_f8(x, out=rows((3, 256))))
    _refused(kb.ERR_INVALID_SHAPE, lambda: d.silu_mul_f8(t((4, 255))))
    _refused(kb.ERR_INVALID_SHAPE, lambda: d.silu_mul_f8(x, t((4, 128))))
    _refused(kb.ERR_INVALID_SHAPE, lambda: d.silu_mul_f8(x, t((4, 256), np.float16)))
    _refused(kb.ERR_INVALID_SHAPE, lambda: d.rms_norm_f8(x, t((128,)), 1e-5))
    _refused(kb.ERR_INVALID_SHAPE, lambda: d.rms_norm_f8(x, w, 1e-5, residual=t((3, 256))))
    _refused(kb.ERR_INVALID_SHAPE, lambda: d.rms_norm_f8(x, w, 1e-5, residual=t((4, 256), np.float16)))
    _refused(kb.ERR_INVALID_SHAPE, lambda: d.rms_norm_f8(x, w, 1e-5, sum_out=t((2, 256))))
    _refused(kb.ERR_INVALID_SHAPE, lambda: d.rms_norm_f8(x, w, 1e-5, bias=t((255,))))
    m = types.SimpleNamespace(shape=(64, 256), h=2)
    r = rows((4, 256))
    _refused(kb.ERR_INVALID_SHAPE, lambda: rows((4, 128)).f8_mat_mul(m))
    _refused(kb.ERR_UNSUPPORTED_DTYPE, lambda: r.f8_mat_mul(m, out_type=kb.Q4_0))
    _refused(kb.ERR_INVALID_SHAPE, lambda: r.f8_mat_mul(m, out=t((4, 63))))
    _refused(kb.ERR_INVALID_SHAPE, lambda: r.f8_mat_mul(m, out_type=kb.BF16, out=t((4, 64))))
    _refused(kb.ERR_INVALID_SHAPE, lambda: r.f8_mat_mul(m, epilogue=kb.EPI_RESIDUAL, r1=t((4, 63)), out=t((4, 64))))
    _refused(kb.ERR_INVALID_SHAPE, lambda: r.f8_mat_mul(m, epilogue=kb.EPI_RESIDUAL, r1=t((4, 64)), r2=t((4, 64), np.float16), out=t((4, 64))))
    _refused(kb.ERR_INVALID_SHAPE, lambda: r.f8_mat_mul(m, epilogue=kb.EPI_BIAS, r1=t((63,)), out=t((4, 64))))


def test_no_handle_is_an_error_code():
    L, out, one = kb.load_library(), C.c_void_p(), (C.c_uint64 * 2)(1, 1)
    assert L.fb200_quantize_f8(None, 16, 16, kb.F32, 1, 16, 16, 16, 16) == kb.ERR_INVALID_ARGUMENT
    assert L.fb200_silu_mul_f8(None, 16, 16, 16, 16, kb.F32, 1, 16, 16, 16, 16) == kb.ERR_INVALID_ARGUMENT
    assert L.fb200_rms_norm_f8(None, 16, 16, None, 0, None, 0, kb.F32, 16, None, 1e-5, 1, 16, 16, 16, 16) == kb.ERR_INVALID_ARGUMENT
    assert L.fb200_f8_mat_mul(None, 16, 16, 16, 1, None, kb.F32, 16, None) == kb.ERR_INVALID_ARGUMENT
    assert L.fb200_f8matrix_from_raw_bytes(None, one, 2, 16, 1, 16, 1, C.byref(out)) == kb.ERR_INVALID_ARGUMENT
    assert L.fb200_f8matrix_from_device(None, one, 2, 16, 16, 16, C.byref(out)) == kb.ERR_INVALID_ARGUMENT
    assert L.fb200_f8matrix_free(None) == kb.OK and L.fb200_f8matrix_shape(None, None, None) == kb.ERR_INVALID_ARGUMENT
