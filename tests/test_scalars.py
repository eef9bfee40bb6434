"""What the Python wrappers take for alpha and beta. No GPU needed: every call
ends before device work."""
import fractions

import numpy as np
import pytest

import sgblas_b200 as sg

FAKE = 0x10000
ZEROS = [0.0, 0, -0.0, np.float32(0), np.array(0.0), np.array(0, dtype=np.int64),
         fractions.Fraction(0)]
ONES = [1.0, 1, True, np.float64(1), np.array(1.0, dtype=np.float32)]


@pytest.mark.parametrize("alpha", ZEROS, ids=repr)
@pytest.mark.parametrize("beta", ONES, ids=repr)
def test_scalars_are_whatever_converts_to_a_float(handle, alpha, beta):
    """alpha 0 and beta 1 leave C as it is, which needs no device."""
    assert handle.sgemm_status(0, 0, 8, 8, 8, alpha, None, 8, None, 8, beta, None, 8) == 0
    assert handle.grouped_gemm_n_status(sg.SGBLAS_OP_T, 8, 8, 8, 1, FAKE, alpha, None, 8, 0, None, 8,
                                        beta, None, sg.SGBLAS_TYPE_FP32, 8) == 0


@pytest.mark.parametrize("bad", ["1", 1j, 1 + 0j, [1.0], object()], ids=repr)
def test_others_are_refused(handle, bad):
    with pytest.raises(TypeError):
        handle.sgemm_status(0, 0, 8, 8, 8, bad, None, 8, None, 8, 1.0, None, 8)


def test_none_is_a_null_pointer(handle):
    assert handle.sgemm_status(0, 0, 8, 8, 8, None, FAKE, 8, FAKE, 8, 1.0, FAKE,
                               8) == sg.SGBLAS_STATUS_INVALID_VALUE
