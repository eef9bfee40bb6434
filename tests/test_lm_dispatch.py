"""Which kernels the language-model products launch, on a stand-in CUDA runtime
(no GPU): the cases that test_lm_tiles_gpu.py checks take the tiles they are
there for, so a changed rule cannot leave a kernel untested."""
import pytest

import sgblas_b200 as sg
from tests import fake_cuda
from tests.fake_cuda import FAKE
from tests.lm_cases import GRADIENTS, ORTHOGONAL, RAGGED

BF16, FP32 = sg.SGBLAS_TYPE_BF16, sg.SGBLAS_TYPE_FP32
OP_N, OP_T = sg.SGBLAS_OP_N, sg.SGBLAS_OP_T
FLAGS = {True: "true", False: "false"}


@pytest.fixture(scope="module")
def dll(tmp_path_factory):
    return fake_cuda.build(tmp_path_factory.mktemp("fake"))


@pytest.fixture()
def log(dll, monkeypatch):
    monkeypatch.setattr(sg, "lib", dll)
    dll.fakeReset()
    yield fake_cuda.Log(dll)
    dll.fakeReset()


def config(elem, ragged, width, a_mn, b_mn, pair, fp32):
    """The start of a product kernel's name: its template arguments."""
    args = f"{elem}, (Ragged){ragged}, {width}, " + ", ".join(FLAGS[v] for v in (a_mn, b_mn, pair, fp32))
    return f"void productKernel<Cfg<{args}, "


def grouped_n(trans, ctype, beta, case):
    m, k, n, groups = case["m"], case["k"], sum(case["lengths"]), len(case["lengths"])
    lda = k if trans == OP_T else m
    with sg.Handle() as h:
        h.grouped_gemm_n(trans, m, n, k, groups, FAKE, 1.0, FAKE, lda, m * k, FAKE, k, beta, FAKE,
                         ctype, m)


def grouped_fp8(ctype, case):
    m, k, n, groups = case["m"], case["k"], sum(case["lengths"]), len(case["lengths"])
    kb = -(-k // 128)
    with sg.Handle() as h:
        h.grouped_gemm_fp8(m, n, k, groups, FAKE, FAKE, k, m * k, FAKE, kb, kb * -(-m // 128), FAKE, k,
                           FAKE, kb, FAKE, ctype, m)


OUTPUTS = [(BF16, 0.0), (FP32, 0.0), (BF16, 1.0), (FP32, 0.5)]


@pytest.mark.parametrize("case", RAGGED, ids=lambda c: c["name"])
@pytest.mark.parametrize("ctype,beta", OUTPUTS)
@pytest.mark.parametrize("trans", [OP_T, OP_N])
def test_tiles_of_ragged_products(log, trans, ctype, beta, case):
    grouped_n(trans, ctype, beta, case)
    plain, width = ctype == BF16 and beta == 0.0, case["bf16"]
    kernel, _ = log.launches()[-1]
    want = (f"void thinProductKernel<ThinCfg<2, {width}, {FLAGS[trans == OP_N]}> " if width < 128
            else config(2, 0, width, trans == OP_N, False, width == 256, not plain))
    assert kernel.startswith(want), kernel


@pytest.mark.parametrize("case", RAGGED, ids=lambda c: c["name"])
@pytest.mark.parametrize("ctype", [BF16, FP32])
def test_tiles_of_ragged_products_fp8(log, ctype, case):
    grouped_fp8(ctype, case)
    kernel, _ = log.launches()[-1]
    width = case["fp8"]
    want = (f"void thinProductKernel<ThinCfg<1, {width}, false> " if width < 128
            else config(1, 0, width, False, False, False, ctype == FP32) if width == 128
            else config(1, 3, 256, False, False, True, False))
    assert kernel.startswith(want), kernel


def test_every_product_kernel_is_tested(log):
    """The cases together launch every product kernel that the library has."""
    for case in RAGGED:
        for ctype, beta in OUTPUTS:
            for trans in (OP_N, OP_T):
                grouped_n(trans, ctype, beta, case)
            grouped_fp8(ctype, case)
    with sg.Handle() as h:
        for m, n in GRADIENTS:
            for ctype, beta in OUTPUTS:
                h.grouped_gemm_k(m, n, 1500, 12, FAKE, 1.0, FAKE, m, FAKE, n, beta, FAKE, ctype, m, n * m)
        for rows, cols, batch in ORTHOGONAL:
            h.orthogonalize(cols, rows, batch, 5, (3.4445, -4.7750, 2.0315), 1e-7, 1.0, FAKE, FP32, cols,
                            rows * cols, FAKE, cols, rows * cols)
    products = {k for k in log.kernels() if "roductKernel<" in k}
    assert len(products) > 30
    assert products <= {name for name, _ in log.launches()}
