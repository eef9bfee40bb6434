"""Arguments, quick returns and refusals of the operators around a layer's
products (sgblas_lm.h). No GPU needed: every call here ends before device work."""
import ctypes

import pytest

import sgblas_b200 as sg

FAKE = 0x10000
BF16, FP32, BYTE = sg.SGBLAS_TYPE_BF16, sg.SGBLAS_TYPE_FP32, sg.SGBLAS_TYPE_BYTE
BAD_TYPE = 7
OK, INVALID = sg.SGBLAS_STATUS_SUCCESS, sg.SGBLAS_STATUS_INVALID_VALUE
UNSUPPORTED = sg.SGBLAS_STATUS_NOT_SUPPORTED


def norm_args(**kw):
    a = dict(k=300, n=20, type=BF16, x=FAKE, ldx=300, residual=FAKE, ldr=300, weight=FAKE, eps=1e-6,
             sum=FAKE, ldsum=300, y=FAKE, ldy=300, q=FAKE, ldq=300, scale=FAKE, ldscale=3)
    a.update(kw)
    return list(a.values())


def back_args(**kw):
    a = dict(k=300, n=20, type=BF16, dy=FAKE, lddy=300, sum=FAKE, ldsum=300, weight=FAKE, eps=1e-6,
             dsum=FAKE, lddsum=300, dx=FAKE, lddx=300, beta=0.0, dweight=FAKE)
    a.update(kw)
    return list(a.values())


def sort_args(**kw):
    a = dict(n=20, top=2, groups=4, group=FAKE, offsets=FAKE, place=FAKE)
    a.update(kw)
    return list(a.values())


def move_args(**kw):
    a = dict(k=300, n=20, top=2, rows=40, place=FAKE, weights=FAKE, x=FAKE, type=BF16, ldx=300, y=FAKE,
             ldy=300)
    a.update(kw)
    return list(a.values())


def move_back_args(**kw):
    a = dict(k=300, n=20, top=2, rows=40, place=FAKE, weights=FAKE, dy=FAKE, type=BF16, lddy=300, x=FAKE,
             ldx=300, dx=FAKE, lddx=300, dweights=FAKE)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw", [
    dict(k=-1), dict(n=-1), dict(type=BAD_TYPE), dict(type=BYTE), dict(ldx=299), dict(ldr=299),
    dict(ldsum=299), dict(ldy=299), dict(ldq=299), dict(ldscale=2), dict(eps=-1e-6),
    dict(eps=float("nan")), dict(x=None), dict(y=None, q=None), dict(scale=None)])
def test_norm_refuses(handle, kw):
    assert handle.rms_norm_status(*norm_args(**kw)) == INVALID
    with pytest.raises(sg.SgblasError):
        handle.rms_norm(*norm_args(**kw))


@pytest.mark.parametrize("kw", [dict(k=0, x=None), dict(n=0, y=None, q=None)])
def test_norm_has_nothing_to_do(handle, kw):
    assert handle.rms_norm_status(*norm_args(**kw)) == OK


@pytest.mark.parametrize("kw", [
    dict(k=-1), dict(n=-1), dict(type=BAD_TYPE), dict(type=BYTE), dict(lddy=299), dict(ldsum=299),
    dict(lddsum=299), dict(lddx=299), dict(eps=-1.0), dict(eps=float("nan")), dict(beta=None),
    dict(dy=None), dict(sum=None), dict(dx=None)])
def test_norm_backward_refuses(handle, kw):
    assert handle.rms_norm_backward_status(*back_args(**kw)) == INVALID
    with pytest.raises(sg.SgblasError):
        handle.rms_norm_backward(*back_args(**kw))


@pytest.mark.parametrize("kw", [dict(k=0, dy=None), dict(n=0, beta=1.0, dx=None),
                                dict(n=0, dweight=None, beta=None)])
def test_norm_backward_has_nothing_to_do(handle, kw):
    assert handle.rms_norm_backward_status(*back_args(**kw)) == OK


@pytest.mark.parametrize("kw", [dict(n=-1), dict(top=-1), dict(groups=-1), dict(group=None),
                                dict(offsets=None), dict(place=None), dict(n=0, offsets=None)])
def test_sort_refuses(handle, kw):
    assert handle.sort_tokens_status(*sort_args(**kw)) == INVALID
    with pytest.raises(sg.SgblasError):
        handle.sort_tokens(*sort_args(**kw))


def test_sort_limits(handle):
    assert handle.sort_tokens_status(*sort_args(groups=sg.SGBLAS_MAX_GROUPS + 1)) == UNSUPPORTED
    assert handle.sort_tokens_status(*sort_args(n=(1 << 30) + 1, top=1)) == UNSUPPORTED
    assert handle.sort_tokens_status(*sort_args(n=1 << 30, top=1 << 30)) == UNSUPPORTED


MOVE_REFUSALS = [dict(k=-1), dict(n=-1), dict(top=-1), dict(rows=-1), dict(type=BAD_TYPE), dict(ldx=299),
                 dict(ldy=299), dict(place=None), dict(x=None), dict(y=None)]


@pytest.mark.parametrize("kw", MOVE_REFUSALS + [dict(type=BYTE)])
def test_scatter_refuses(handle, kw):
    assert handle.scatter_tokens_status(*move_args(**kw)) == INVALID
    with pytest.raises(sg.SgblasError):
        handle.scatter_tokens(*move_args(**kw))


@pytest.mark.parametrize("kw", [dict(k=0, x=None), dict(n=0, y=None), dict(top=0, place=None),
                                dict(rows=0, y=None), dict(type=BYTE, weights=None, n=0)])
def test_scatter_has_nothing_to_do(handle, kw):
    assert handle.scatter_tokens_status(*move_args(**kw)) == OK


@pytest.mark.parametrize("kw", MOVE_REFUSALS + [dict(type=BYTE, weights=None)])
def test_gather_refuses(handle, kw):
    assert handle.gather_tokens_status(*move_args(**kw)) == INVALID
    with pytest.raises(sg.SgblasError):
        handle.gather_tokens(*move_args(**kw))


@pytest.mark.parametrize("kw", [dict(k=0, x=None), dict(n=0, y=None)])
def test_gather_has_nothing_to_do(handle, kw):
    assert handle.gather_tokens_status(*move_args(**kw)) == OK


@pytest.mark.parametrize("kw", [
    dict(k=-1), dict(n=-1), dict(top=-1), dict(rows=-1), dict(type=BAD_TYPE), dict(type=BYTE),
    dict(lddy=299), dict(ldx=299), dict(lddx=299), dict(place=None), dict(dy=None), dict(x=None),
    dict(dx=None)])
def test_gather_backward_refuses(handle, kw):
    assert handle.gather_tokens_backward_status(*move_back_args(**kw)) == INVALID
    with pytest.raises(sg.SgblasError):
        handle.gather_tokens_backward(*move_back_args(**kw))


@pytest.mark.parametrize("kw", [dict(n=0, dy=None), dict(top=0, place=None), dict(k=0, dweights=None),
                                dict(rows=0, dweights=None, dx=None)])
def test_gather_backward_has_nothing_to_do(handle, kw):
    assert handle.gather_tokens_backward_status(*move_back_args(**kw)) == OK


def test_choices_of_a_token(handle):
    """More are not counted in 32 bits, and would never end."""
    for top in ((1 << 30) + 1, 2**31 - 1):
        assert handle.gather_tokens_status(*move_args(top=top)) == UNSUPPORTED
        assert handle.gather_tokens_backward_status(*move_back_args(top=top)) == UNSUPPORTED


def quantize4_args(**kw):
    a = dict(k=301, n=20, x=FAKE, xtype=BF16, ldx=301, q=FAKE, ldq=151, scale=FAKE, ldscale=10, batch=2)
    a.update(kw)
    return list(a.values())


def fp4_args(**kw):
    a = dict(m=64, n=32, k=301, groups=4, offsets=FAKE, a=FAKE, lda=151, stride_a=64 * 151, scale_a=FAKE, ldsa=10,
             stride_sa=640, b=FAKE, ldb=151, scale_b=FAKE, ldsb=10, c=FAKE, ctype=BF16, ldc=64)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw", [dict(k=-1), dict(n=-1), dict(batch=-1), dict(xtype=BAD_TYPE), dict(xtype=BYTE),
                                dict(ldx=300), dict(ldq=150), dict(ldscale=9), dict(x=None), dict(q=None),
                                dict(scale=None)])
def test_quantize_fp4_refuses(handle, kw):
    assert handle.quantize_fp4_status(*quantize4_args(**kw)) == INVALID
    with pytest.raises(sg.SgblasError):
        handle.quantize_fp4(*quantize4_args(**kw))


@pytest.mark.parametrize("kw", [dict(k=0, x=None), dict(n=0, q=None), dict(batch=0, scale=None)])
def test_quantize_fp4_has_nothing_to_do(handle, kw):
    assert handle.quantize_fp4_status(*quantize4_args(**kw)) == OK


def test_quantize_fp4_limit(handle):
    big = 2**31 - 1
    assert handle.quantize_fp4_status(*quantize4_args(k=64, n=big, ldx=64, ldq=32, ldscale=2, batch=1)) == UNSUPPORTED


FP4_REFUSALS = [dict(m=-1), dict(n=-1), dict(k=-1), dict(ctype=BAD_TYPE), dict(ctype=BYTE), dict(lda=150), dict(ldb=150),
                dict(ldc=63), dict(ldsa=9), dict(ldsb=9), dict(a=None), dict(b=None), dict(scale_a=None),
                dict(scale_b=None), dict(c=None)]


@pytest.mark.parametrize("kw", FP4_REFUSALS + [dict(groups=-1), dict(offsets=None)])
def test_grouped_fp4_refuses(handle, kw):
    assert handle.grouped_gemm_fp4_status(*fp4_args(**kw)) == INVALID
    with pytest.raises(sg.SgblasError):
        handle.grouped_gemm_fp4(*fp4_args(**kw))


def one_matrix(**kw):
    names = ("m", "n", "k", "groups", "offsets", "a", "lda", "stride_a", "scale_a", "ldsa", "stride_sa", "b", "ldb",
             "scale_b", "ldsb", "c", "ctype", "ldc")
    return [v for name, v in zip(names, fp4_args(**kw)) if name not in ("groups", "offsets", "stride_a", "stride_sa")]


@pytest.mark.parametrize("kw", FP4_REFUSALS)
def test_fp4_refuses(handle, kw):
    assert handle.gemm_fp4_status(*one_matrix(**kw)) == INVALID
    with pytest.raises(sg.SgblasError):
        handle.gemm_fp4(*one_matrix(**kw))


@pytest.mark.parametrize("kw", [dict(m=0, a=None, ldc=1), dict(n=0, c=None), dict(groups=0, offsets=None)])
def test_fp4_has_nothing_to_do(handle, kw):
    assert handle.grouped_gemm_fp4_status(*fp4_args(**kw)) == OK
    if "groups" not in kw:
        assert handle.gemm_fp4_status(*one_matrix(**kw)) == OK


def test_fp4_groups(handle):
    assert handle.grouped_gemm_fp4_status(*fp4_args(groups=sg.SGBLAS_MAX_GROUPS + 1)) == UNSUPPORTED


def test_bytes_are_no_type_of_products(handle):
    assert handle.quantize_fp8_status(300, 20, 1, FAKE, BYTE, 300, FAKE, 300, FAKE, 3) == INVALID
    assert handle.gemm_fp8_status(64, 32, 300, FAKE, 300, FAKE, 3, FAKE, 300, FAKE, 3, FAKE, BYTE,
                                  64) == INVALID


def test_null_handle():
    none = ctypes.c_void_p(None)
    zero = ctypes.byref(ctypes.c_float(0.0))
    back = back_args()
    back[13] = zero
    for name, args in (("sgblasRmsNorm", norm_args()), ("sgblasRmsNormBackward", back),
                       ("sgblasSortTokens", sort_args()), ("sgblasScatterTokens", move_args()),
                       ("sgblasGatherTokens", move_args()),
                       ("sgblasGatherTokensBackward", move_back_args()),
                       ("sgblasQuantizeFp4", [300, 20, 1, FAKE, BF16, 300, 0, FAKE, 150, 0, FAKE, 10, 0]),
                       ("sgblasGemmFp4", one_matrix()), ("sgblasGroupedGemmFp4", fp4_args())):
        assert getattr(sg.lib, name)(none, *args) == sg.SGBLAS_STATUS_NOT_INITIALIZED
