"""Which kernels the operators around a layer's products and the 4-bit products
launch, on a stand-in CUDA runtime (no GPU): the GPU tests' sizes reach every one."""
import pytest

import sgblas_b200 as sg
from tests import fake_cuda
from tests.fake_cuda import FAKE
from tests.lm_cases import RAGGED
from tests.test_fp4_gpu import DECREASING, ONE_MATRIX, PAIRS, SMALL
from tests.test_norm_gpu import RINGS
from tests.test_norm_gpu import SIZES as NORM_SIZES
from tests.test_tokens_gpu import SIZES as TOKEN_SIZES

BF16, FP32, BYTE = sg.SGBLAS_TYPE_BF16, sg.SGBLAS_TYPE_FP32, sg.SGBLAS_TYPE_BYTE


@pytest.fixture(scope="module")
def dll(tmp_path_factory):
    return fake_cuda.build(tmp_path_factory.mktemp("fake"))


@pytest.fixture()
def log(dll, monkeypatch):
    monkeypatch.setattr(sg, "lib", dll)
    dll.fakeReset()
    yield fake_cuda.Log(dll)
    dll.fakeReset()


def reached(log, part):
    every = {k for k in log.kernels() if part in k}
    launched = {name for name, _ in log.launches()}
    return every, every - launched


def fp4(h, m, n, k, groups, ctype):
    kb, ks = -(-k // 32) * 16, -(-k // 512) * 16
    h.grouped_gemm_fp4(m, n, k, groups, FAKE, FAKE, kb, m * kb, FAKE, ks, m * ks, FAKE, kb, FAKE, ks, FAKE, ctype, m)


def test_every_fp4_kernel_is_tested(log):
    with sg.Handle() as h:
        for case in RAGGED + PAIRS + SMALL:
            for ctype in (BF16, FP32):
                fp4(h, case["m"], sum(case["lengths"]), case["k"], len(case["lengths"]), ctype)
        for m, n, k in ONE_MATRIX:
            for ctype in (BF16, FP32):
                fp4(h, m, n, k, 1, ctype)
    for part, count in (("fp4TileKernel", 4), ("fp4ThinKernel", 2), ("layScalesKernel", 1)):
        every, left = reached(log, part)
        assert len(every) == count and not left, left


@pytest.mark.parametrize("case", PAIRS + [dict(m=4096, k=1542, lengths=[2500, 3700, 0, 2800]),
                                          dict(m=4001, k=1542, lengths=[2500, 3700, 0, 2800]),
                                          dict(m=4001, k=1544, lengths=[2500, 3000, 3700]),
                                          dict(m=4096, k=4608, lengths=[3500, 4000]),
                                          dict(m=4096, k=1536, lengths=[2500, 0, 4000, 3000]),
                                          dict(m=6008, k=1542, lengths=[6100])])
def test_cases_of_pairs_are_pairs(log, case):
    with sg.Handle() as h:
        fp4(h, case["m"], sum(case["lengths"]), case["k"], len(case["lengths"]), BF16)
    assert "fp4TileKernel<Fp4Cfg<192" in log.launches()[-1][0]


def test_decreasing_offsets_are_tested_on_pairs(log):
    with sg.Handle() as h:
        for ctype in (BF16, FP32):
            fp4(h, DECREASING["m"], DECREASING["n"], DECREASING["k"], DECREASING["groups"], ctype)
            assert "fp4TileKernel<Fp4Cfg<192" in log.launches()[-1][0]


@pytest.mark.parametrize("m,n,k,groups,kernel", [
    (4096, 1, 4096, 1, "fp4ThinKernel<Fp4ThinCfg<16>"), (2048, 384, 2048, 32, "fp4ThinKernel<Fp4ThinCfg<32>"),
    (1024, 256, 1024, 1, "fp4TileKernel<Fp4Cfg<128, false, false>"),
    (8192, 8192, 4096, 1, "fp4TileKernel<Fp4Cfg<192, true, false>")])
def test_fp4_widths(log, m, n, k, groups, kernel):
    with sg.Handle() as h:
        fp4(h, m, n, k, groups, BF16)
    names = [name for name, _ in log.launches()]
    assert kernel in names[-1]
    assert len(names) == (2 if "192" in kernel else 1)   # pairs: the scales are laid out first


def test_pairs_without_a_workspace_are_single_ctas(log):
    """Inside a capture the workspace is not made: the scales are staged instead."""
    with sg.Handle() as h:
        log.dll.fakeCapture(1)
        fp4(h, 8192, 8192, 4096, 1, BF16)
        assert [name for name, _ in log.launches()][-1].startswith("void fp4TileKernel<Fp4Cfg<128, false, false>")
        log.dll.fakeCapture(0)
        fp4(h, 8192, 8192, 4096, 1, BF16)
        log.dll.fakeReset()
        log.dll.fakeCapture(1)
        fp4(h, 8192, 8192, 4096, 1, BF16)
        assert "192" in log.launches()[-1][0]
        log.dll.fakeCapture(0)


@pytest.mark.parametrize("at", [2, 3])
def test_a_failed_launch_after_the_scales_is_a_use(log, at):
    """The workspace's event follows the copies and blocks of scales, also when the
    product is not launched."""
    m, n, k = 4096, 4096, 2050   # rows that TMA cannot read: one operand is copied
    args = [m, n, k, FAKE, 1040, FAKE, 80, FAKE, 1025, FAKE, 80, FAKE, BF16, m]
    with sg.Handle() as h:
        assert h.gemm_fp4_status(*args) == sg.SGBLAS_STATUS_SUCCESS
        assert len(log.launches()) == 3   # a copy, the blocks, the product
        log.dll.fakeReset()
        log.dll.fakeFailLaunch(at)
        assert h.gemm_fp4_status(*args) == sg.SGBLAS_STATUS_EXECUTION_FAILED
        assert log.lines()[-1] == "record"


@pytest.mark.parametrize("at", [1, 2])
def test_a_failed_weight_gradient_is_a_use(log, at):
    with sg.Handle() as h:
        log.dll.fakeFailLaunch(at)
        assert h.rms_norm_backward_status(256, 100, BF16, FAKE, 256, FAKE, 256, FAKE, 1e-6, FAKE, 256, FAKE, 256, 0.0,
                                          FAKE) == sg.SGBLAS_STATUS_EXECUTION_FAILED
        assert log.lines()[-1] == "record"


@pytest.mark.parametrize("type_,size", [(BF16, 2), (FP32, 4)])
def test_rings_are_tested_past_their_stages(log, type_, size):
    """Of each kernel fed by a ring a test's CTAs walk more than twice as many sets of
    columns as it has stages, and one ends in part of a set where a set has several."""
    turns, parts = {}, {}
    with sg.Handle() as h:
        for k, n in RINGS:
            for residual in (FAKE, None):   # the stages are the same without
                log.dll.fakeReset()
                h.rms_norm(k, n, type_, FAKE, k, residual, k, FAKE, 1e-6, FAKE, k, FAKE, k)
                h.rms_norm_backward(k, n, type_, FAKE, k, FAKE, k, FAKE, 1e-6, residual, k, FAKE, k, 0.0, FAKE)
                for name, grid, _, columns, smem in log.shapes():
                    if "Stream" not in name:
                        continue
                    stages = smem // ((3 if "Backward" in name else 2) * columns * k * size)
                    turns[name] = max(turns.get(name, 0), -(-n // columns) / grid / stages)
                    parts[name] = parts.get(name, False) or columns == 1 or n % columns != 0
    every = {name for name in log.kernels() if "Stream" in name and ("<float" in name) == (type_ == FP32)}
    assert len(every) == 6 and set(turns) == every
    assert min(turns.values()) > 2 and all(parts.values()), turns


@pytest.mark.parametrize("n,top,ctas", [(16, 4, 1), (1024, 2, 4), (1024, 8, 16), (65536, 8, 16)])
def test_ctas_of_a_sort(log, n, top, ctas):
    with sg.Handle() as h:
        h.sort_tokens(n, top, 64, FAKE, FAKE, FAKE)
    assert [grid for _, grid in log.launches()] == [ctas]


def test_the_longest_columns_partial_sums(log):
    """Four bytes for each of 2^31 values: their size is not counted in 32 bits."""
    k = 2**31 - 1
    with sg.Handle() as h:
        h.rms_norm_backward(k, 1, BF16, FAKE, k, FAKE, k, FAKE, 1e-6, FAKE, k, FAKE, k, 0.0, FAKE)
    sizes = [int(line.split()[2]) for line in log.lines() if line.startswith("malloc")]
    assert 2**33 <= max(sizes) < 2**34, sizes   # with room for larger calls


def test_every_norm_and_token_kernel_is_tested(log):
    with sg.Handle() as h:
        for type_ in (BF16, FP32):
            for at, ld in ((FAKE, 0), (FAKE, 8), (FAKE + 4, 3)):
                for k, n in NORM_SIZES:
                    h.rms_norm(k, n, type_, at, k + ld, at, k + ld, at, 1e-6, at, k + ld, at, k + ld)
                    h.rms_norm_backward(k, n, type_, at, k + ld, at, k + ld, at, 1e-6, at, k + ld, at, k + ld, 0.0, at)
                for k, n, top in TOKEN_SIZES:
                    h.scatter_tokens(k, n, top, n * top, at, at, at, type_, k + ld, at, k + ld)
                    h.gather_tokens(k, n, top, n * top, at, at, at, type_, k + ld, at, k + ld)
                    h.gather_tokens_backward(k, n, top, n * top, at, at, at, type_, k + ld, at, k + ld, at, k + ld, at)
        for k in (16, 37):
            h.scatter_tokens(k, 50, 3, 150, FAKE, None, FAKE, BYTE, k, FAKE, k)
        for groups in (4, 1000):
            h.sort_tokens(10, 2, groups, FAKE, FAKE, FAKE)
        for ldx in (64, 65):
            for type_ in (BF16, FP32):
                h.quantize_fp4(64, 5, FAKE, type_, ldx, FAKE, 32, FAKE, 2)
    for part, count in (("rmsNorm", 30), ("sumParts", 1), ("scatterTokens", 6), ("gatherTokens", 8), ("sortTokens", 2), ("quantizeFp4", 4)):
        every, left = reached(log, part)
        assert len(every) >= count and not left, (len(every), left)
