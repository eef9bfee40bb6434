"""The compiled caller (sgblas_b200/calls.c): the same statuses as by ctypes, and
arguments that are refused. No GPU needed."""
import ctypes

import pytest

import sgblas_b200 as sg
from tests import test_layer_api as api

_calls = pytest.importorskip("sgblas_b200._calls")
FAKE = 0x10000


def quantize4(**kw):
    k, n, x, xtype, ldx, q, ldq, scale, ldscale, batch = api.quantize4_args(**kw)
    return [k, n, batch, x, xtype, ldx, 0, q, ldq, 0, scale, ldscale, 0]


CALLS = {
    "rms_norm": ("sgblasRmsNorm", api.norm_args, [dict(k=-1), dict(ldx=299), dict(eps=-1.0), dict(n=0)]),
    "rms_norm_backward": ("sgblasRmsNormBackward", api.back_args, [dict(k=-1), dict(lddx=299), dict(beta=None), dict(k=0)]),
    "sort_tokens": ("sgblasSortTokens", api.sort_args, [dict(n=-1), dict(offsets=None), dict(groups=1025)]),
    "scatter_tokens": ("sgblasScatterTokens", api.move_args, [dict(k=-1), dict(type=api.BYTE), dict(n=0)]),
    "gather_tokens": ("sgblasGatherTokens", api.move_args, [dict(rows=-1), dict(ldy=299), dict(k=0)]),
    "gather_tokens_backward": ("sgblasGatherTokensBackward", api.move_back_args, [dict(top=-1), dict(dx=None), dict(top=0)]),
    "quantize_fp4": ("sgblasQuantizeFp4", quantize4, [dict(n=-1), dict(ldq=150), dict(batch=0)]),
    "gemm_fp4": ("sgblasGemmFp4", api.one_matrix, [dict(m=-1), dict(ldsb=9), dict(n=0)]),
    "grouped_gemm_fp4": ("sgblasGroupedGemmFp4", api.fp4_args, [dict(groups=-1), dict(offsets=None), dict(groups=1025)]),
}


def by_ctypes(symbol, handle, args):
    types = sg._SIGNATURES[symbol][1][1:]
    converted = [sg._fp(a) if t is sg._c_float_p else a for a, t in zip(args, types)]
    return getattr(sg.lib, symbol)(handle, *converted)


@pytest.mark.parametrize("name", CALLS)
def test_statuses_are_the_same(handle, name):
    symbol, make, changes = CALLS[name]
    for kw in changes:
        args = make(**kw)
        status = getattr(_calls, name)(handle._address, *args)
        assert status == by_ctypes(symbol, handle.raw, args), kw
        assert status != sg.SGBLAS_STATUS_NOT_INITIALIZED
        assert getattr(_calls, name)(None, *args) == sg.SGBLAS_STATUS_NOT_INITIALIZED


@pytest.mark.parametrize("name", CALLS)
def test_arguments_that_do_not_convert(handle, name):
    call, args = getattr(_calls, name), CALLS[name][1]()
    with pytest.raises(TypeError):
        call(handle._address, *args[:-1])
    with pytest.raises(TypeError):
        call(handle._address, *args, 0)
    for at, value in enumerate(args):
        for bad, error in (("a text", (TypeError, AttributeError)), (2**70, OverflowError)):
            if isinstance(value, float) and bad == 2**70:
                continue   # a number like any other
            wrong = list(args)
            wrong[at] = bad
            with pytest.raises(error):
                call(handle._address, *wrong)
        if isinstance(value, int) and value < 1000:   # an int: no more than 32 bits, nothing with a fraction
            for bad, error in ((2**31, OverflowError), (-2**31 - 1, OverflowError), (1.5, TypeError)):
                if bad == 2**31 and name.endswith("fp4") and sg._SIGNATURES[CALLS[name][0]][1][1:][at] is ctypes.c_longlong:
                    continue
                if sg._SIGNATURES[CALLS[name][0]][1][1:][at] is ctypes.c_longlong and bad != 1.5:
                    continue
                wrong = list(args)
                wrong[at] = bad
                with pytest.raises(error):
                    call(handle._address, *wrong)


def test_pointers_are_tensors_numbers_or_none(handle):
    class Tensor:
        def __init__(self, address):
            self.address = address

        def data_ptr(self):
            return self.address

    args = api.sort_args(n=0, group=None, place=None)
    args[4] = Tensor(0)
    assert _calls.sort_tokens(handle._address, *args) == sg.SGBLAS_STATUS_INVALID_VALUE   # offsets are needed
    norm = api.norm_args(k=0)
    norm[3] = Tensor(FAKE)
    assert _calls.rms_norm(handle._address, *norm) == sg.SGBLAS_STATUS_SUCCESS

    class Broken:
        def data_ptr(self):
            raise ValueError("freed")

    norm[3] = Broken()
    with pytest.raises(ValueError):
        _calls.rms_norm(handle._address, *norm)


def test_integers_by_index(handle):
    numpy = pytest.importorskip("numpy")
    args = api.norm_args(k=numpy.int64(0), n=numpy.int32(3), eps=numpy.float32(1e-6))
    assert _calls.rms_norm(handle._address, *args) == sg.SGBLAS_STATUS_SUCCESS


def test_bind_refuses():
    for bad, error in ((("nobody", 1), ValueError), (("rms_norm",), TypeError), ((3, 4), TypeError)):
        with pytest.raises(error):
            _calls.bind(*bad)


def test_a_closed_handle_is_refused():
    h = sg.Handle()
    h.close()
    with pytest.raises(sg.SgblasError, match="not initialized"):
        h.sort_tokens(*api.sort_args())
