"""What the library does with a handle's workspace, on a stand-in CUDA runtime
(no GPU)."""
import pytest

import sgblas_b200 as sg
from tests import fake_cuda
from tests.fake_cuda import FAKE

BF16, FP32 = sg.SGBLAS_TYPE_BF16, sg.SGBLAS_TYPE_FP32


@pytest.fixture(scope="module")
def dll(tmp_path_factory):
    return fake_cuda.build(tmp_path_factory.mktemp("fake"))


@pytest.fixture()
def log(dll, monkeypatch):
    monkeypatch.setattr(sg, "lib", dll)
    dll.fakeReset()
    yield fake_cuda.Log(dll)
    dll.fakeReset()


# Calls that copy both operands into the workspace before they multiply.
def grouped_n(h):
    return h.grouped_gemm_n_status(sg.SGBLAS_OP_T, 300, 200, 77, 4, FAKE, 1.0, FAKE, 77, 300 * 77, FAKE, 77,
                                   0.0, FAKE, FP32, 300)


def grouped_k(h):
    return h.grouped_gemm_k_status(301, 203, 77, 4, FAKE, 1.0, FAKE, 301, FAKE, 203, 0.0, FAKE, FP32, 301,
                                   301 * 203)


def sgemm(h):
    return h.sgemm_status(0, 1, 2049, 2049, 1001, 1.0, FAKE, 2049, FAKE, 2049, 0.0, FAKE, 2049)


@pytest.mark.parametrize("call", [grouped_n, grouped_k, sgemm])
@pytest.mark.parametrize("at", [2, 3])
def test_copies_before_a_failed_launch_are_uses(log, call, at):
    """The workspace's event follows every launch that used it, also when a
    later one fails: the next user of the workspace waits for the copies."""
    with sg.Handle() as h:
        assert call(h) == 0
        assert len(log.launches()) == 3   # two copies, one product
        log.dll.fakeReset()
        log.dll.fakeFailLaunch(at)
        assert call(h) == sg.SGBLAS_STATUS_EXECUTION_FAILED
        assert len(log.launches()) == at - 1
        assert log.lines()[-1] == "record"


def addresses(log, what):
    return [line.split()[1] for line in log.lines() if line.startswith(what + " ")]


def larger(h):
    return h.grouped_gemm_n_status(sg.SGBLAS_OP_T, 4001, 4001, 4001, 4, FAKE, 1.0, FAKE, 4001, 4001 * 4001,
                                   FAKE, 4001, 0.0, FAKE, FP32, 4001)


def orthogonalize(h):
    return h.orthogonalize_status(64, 64, 1, 5, (3.4445, -4.7750, 2.0315), 1e-7, 1.0, FAKE, FP32, 64, 0, FAKE,
                                  64, 0)


@pytest.mark.parametrize("call", [grouped_n, sgemm, orthogonalize])
@pytest.mark.parametrize("captured", [False, True])
def test_a_workspace_in_a_graph_stays(log, captured, call):
    """A graph may be replayed after a larger call: the workspace it uses is not
    freed before the handle is destroyed. Without a capture it is."""
    with sg.Handle() as h:
        assert call(h) == 0
        first = addresses(log, "malloc")
        assert len(first) == 1
        if captured:
            log.dll.fakeCapture(1)
            assert call(h) == 0
            log.dll.fakeCapture(0)
        assert larger(h) == 0
        assert len(addresses(log, "malloc")) == 2
        assert addresses(log, "free") == ([] if captured else first)
    assert sorted(addresses(log, "free")) == sorted(addresses(log, "malloc"))
