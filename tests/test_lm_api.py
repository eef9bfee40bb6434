"""Arguments, quick returns and refusals of the language-model products
(sgblas_lm.h). No GPU needed: every call here ends before device work."""
import ctypes

import pytest

import sgblas_b200 as sg

FAKE = 0x10000
BF16, FP32 = sg.SGBLAS_TYPE_BF16, sg.SGBLAS_TYPE_FP32
BAD_TYPE = 7
OK, INVALID = sg.SGBLAS_STATUS_SUCCESS, sg.SGBLAS_STATUS_INVALID_VALUE


def n_args(**kw):
    a = dict(transa=sg.SGBLAS_OP_T, m=64, n=32, k=48, groups=4, offsets=FAKE, alpha=1.0, a=FAKE,
             lda=48, stride_a=64 * 48, b=FAKE, ldb=48, beta=0.0, c=FAKE, ctype=BF16, ldc=64)
    a.update(kw)
    return list(a.values())


def k_args(**kw):
    a = dict(m=64, n=32, k=48, groups=4, offsets=FAKE, alpha=1.0, a=FAKE, lda=64, b=FAKE, ldb=32,
             beta=0.0, c=FAKE, ctype=FP32, ldc=64, stride_c=64 * 32)
    a.update(kw)
    return list(a.values())


def q_args(**kw):
    a = dict(k=300, n=20, block_n=1, x=FAKE, xtype=BF16, ldx=300, q=FAKE, ldq=300, scale=FAKE,
             ldscale=3)
    batch = {key: kw.pop(key) for key in ("batch", "stride_x", "stride_q", "stride_scale")
             if key in kw}
    a.update(kw)
    return list(a.values()), batch


def f_args(**kw):
    a = dict(m=64, n=32, k=300, groups=4, offsets=FAKE, a=FAKE, lda=300, stride_a=64 * 300,
             scale_a=FAKE, ldsa=3, stride_sa=3, b=FAKE, ldb=300, scale_b=FAKE, ldsb=3, c=FAKE,
             ctype=BF16, ldc=64)
    a.update(kw)
    return list(a.values())


def o_args(**kw):
    a = dict(m=64, n=32, batch=2, steps=5, coefficients=(3.4445, -4.775, 2.0315), eps=1e-7,
             scale=1.0, g=FAKE, gtype=FP32, ldg=64, stride_g=64 * 32, o=FAKE, ldo=64,
             stride_o=64 * 32)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw", [
    dict(transa=2), dict(m=-1), dict(n=-1), dict(k=-1), dict(groups=-1), dict(ctype=BAD_TYPE),
    dict(lda=47), dict(transa=sg.SGBLAS_OP_N, lda=63), dict(ldb=47), dict(ldc=63), dict(alpha=None),
    dict(beta=None), dict(offsets=None), dict(a=None), dict(b=None), dict(c=None),
    dict(k=0, c=None), dict(alpha=0.0, c=None), dict(lda=0, k=0)])
def test_grouped_n_refuses(handle, kw):
    assert handle.grouped_gemm_n_status(*n_args(**kw)) == INVALID
    with pytest.raises(sg.SgblasError):
        handle.grouped_gemm_n(*n_args(**kw))


@pytest.mark.parametrize("kw", [
    dict(m=0, a=None, alpha=None), dict(n=0, offsets=None), dict(groups=0, c=None),
    dict(k=0, beta=1.0, a=None, b=None, c=None), dict(alpha=0.0, beta=1.0, a=None, c=None)])
def test_grouped_n_has_nothing_to_do(handle, kw):
    assert handle.grouped_gemm_n_status(*n_args(**kw)) == OK


@pytest.mark.parametrize("kw", [
    dict(m=-1), dict(n=-1), dict(k=-1), dict(groups=-1), dict(ctype=BAD_TYPE), dict(lda=63),
    dict(ldb=31), dict(ldc=63), dict(alpha=None), dict(beta=None), dict(offsets=None),
    dict(a=None), dict(b=None), dict(c=None), dict(k=0, c=None)])
def test_grouped_k_refuses(handle, kw):
    assert handle.grouped_gemm_k_status(*k_args(**kw)) == INVALID


@pytest.mark.parametrize("kw", [
    dict(m=0, a=None), dict(n=0, alpha=None), dict(groups=0), dict(k=0, beta=1.0, c=None)])
def test_grouped_k_has_nothing_to_do(handle, kw):
    assert handle.grouped_gemm_k_status(*k_args(**kw)) == OK


@pytest.mark.parametrize("kw", [
    dict(k=-1), dict(n=-1), dict(batch=-1), dict(block_n=64), dict(block_n=0), dict(xtype=BAD_TYPE),
    dict(ldx=299), dict(ldq=299), dict(ldscale=2), dict(x=None), dict(q=None), dict(scale=None)])
def test_quantize_refuses(handle, kw):
    args, batch = q_args(**kw)
    assert handle.quantize_fp8_status(*args, **batch) == INVALID


@pytest.mark.parametrize("kw", [dict(k=0, x=None), dict(n=0, q=None), dict(batch=0, scale=None)])
def test_quantize_has_nothing_to_do(handle, kw):
    args, batch = q_args(**kw)
    assert handle.quantize_fp8_status(*args, **batch) == OK


@pytest.mark.parametrize("kw", [
    dict(m=-1), dict(n=-1), dict(k=-1), dict(groups=-1), dict(ctype=BAD_TYPE), dict(lda=299),
    dict(ldb=299), dict(ldc=63), dict(ldsa=2), dict(ldsb=2), dict(offsets=None), dict(a=None),
    dict(b=None), dict(scale_a=None), dict(scale_b=None), dict(c=None)])
def test_grouped_fp8_refuses(handle, kw):
    assert handle.grouped_gemm_fp8_status(*f_args(**kw)) == INVALID


@pytest.mark.parametrize("kw", [dict(m=0, a=None), dict(n=0, c=None), dict(groups=0)])
def test_grouped_fp8_has_nothing_to_do(handle, kw):
    assert handle.grouped_gemm_fp8_status(*f_args(**kw)) == OK


def test_gemm_fp8_refuses(handle):
    good = [64, 32, 300, FAKE, 300, FAKE, 3, FAKE, 300, FAKE, 3, FAKE, BF16, 64]
    for at, bad in ((0, -1), (1, -1), (2, -1), (3, None), (4, 299), (5, None), (6, 2), (7, None),
                    (8, 299), (9, None), (10, 2), (11, None), (12, BAD_TYPE), (13, 63)):
        args = list(good)
        args[at] = bad
        assert handle.gemm_fp8_status(*args) == INVALID, at
    assert handle.gemm_fp8_status(*([0] + good[1:])) == OK


@pytest.mark.parametrize("kw", [
    dict(m=-1), dict(n=-1), dict(batch=-1), dict(steps=0), dict(steps=33), dict(gtype=BAD_TYPE),
    dict(ldg=63), dict(ldo=63), dict(coefficients=None), dict(g=None), dict(o=None), dict(eps=-1.0),
    dict(eps=float("nan"))])
def test_orthogonalize_refuses(handle, kw):
    assert handle.orthogonalize_status(*o_args(**kw)) == INVALID


@pytest.mark.parametrize("kw", [dict(m=0, ldg=1, ldo=1, g=None), dict(n=0, o=None),
                                dict(batch=0, coefficients=None)])
def test_orthogonalize_has_nothing_to_do(handle, kw):
    assert handle.orthogonalize_status(*o_args(**kw)) == OK


def test_too_many_groups_are_not_supported(handle):
    many = sg.SGBLAS_MAX_GROUPS + 1
    unsupported = sg.SGBLAS_STATUS_NOT_SUPPORTED
    assert handle.grouped_gemm_n_status(*n_args(groups=many)) == unsupported
    assert handle.grouped_gemm_k_status(*k_args(groups=many)) == unsupported
    assert handle.grouped_gemm_fp8_status(*f_args(groups=many)) == unsupported
    assert handle.orthogonalize_status(*o_args(batch=65536)) == unsupported


def test_null_handle():
    none = ctypes.c_void_p(None)
    uninitialized = sg.SGBLAS_STATUS_NOT_INITIALIZED
    one = ctypes.byref(ctypes.c_float(1.0))
    a = n_args()
    a[6], a[12] = one, one
    assert sg.lib.sgblasGroupedGemmN(none, *a) == uninitialized
    a = k_args()
    a[5], a[10] = one, one
    assert sg.lib.sgblasGroupedGemmK(none, *a) == uninitialized
    assert sg.lib.sgblasQuantizeFp8(none, 300, 20, 1, 1, FAKE, BF16, 300, 0, FAKE, 300, 0, FAKE, 3,
                                    0) == uninitialized
    assert sg.lib.sgblasGemmFp8(none, 64, 32, 300, FAKE, 300, FAKE, 3, FAKE, 300, FAKE, 3, FAKE,
                                BF16, 64) == uninitialized
    assert sg.lib.sgblasGroupedGemmFp8(none, *f_args()) == uninitialized
    a = o_args()
    a[4] = (ctypes.c_float * 3)(1.0, 1.0, 1.0)
    assert sg.lib.sgblasOrthogonalize(none, *a) == uninitialized
