"""The wide kernels of the language-model products where a worker takes several
tiles one after the other: ring, accumulators, scales and staging buffers go
from tile to tile. Operands are small whole numbers, so every sum is exact in
FP32 and a result is equal to the definition's, rounded once.
"""
import pytest

import sgblas_b200 as sg
from tests.lm_cases import ODD_PIECES
from tests.test_lm_products_gpu import dtype_of, generator, guards_ok, output

pytestmark = pytest.mark.gpu

BF16, FP32 = sg.SGBLAS_TYPE_BF16, sg.SGBLAS_TYPE_FP32
OP_N, OP_T = sg.SGBLAS_OP_N, sg.SGBLAS_OP_T


def whole(torch, gen, *shape):
    return torch.randint(-3, 4, shape, generator=gen, device="cuda").to(torch.bfloat16)


def ends_of(lengths, head=0):
    ends = [head]
    for n in lengths:
        ends.append(ends[-1] + n)
    return ends


def by_group(torch, x, w, ends):
    """Rows of x times the transposed w of their group, in 64 bits; zeros outside the groups."""
    y = torch.zeros(x.shape[0], w.shape[1], dtype=torch.float64, device="cuda")
    for g in range(w.shape[0]):
        y[ends[g]:ends[g + 1]] = x[ends[g]:ends[g + 1]].double() @ w[g].double().T
    return y


@pytest.mark.parametrize("ctype", [FP32, BF16])
@pytest.mark.parametrize("trans", [OP_T, OP_N])
def test_odd_pieces_of_tokens(cuda, handle, trans, ctype):
    """A tile that ends on the staging buffer that the next one begins on: their
    columns stay apart, call after call."""
    torch = cuda
    gen = generator(torch, 21)
    lengths, m, k = ODD_PIECES["lengths"], ODD_PIECES["m"], ODD_PIECES["k"]
    ends, groups = ends_of(lengths), len(lengths)
    n = ends[-1]
    x, w = whole(torch, gen, n, k), whole(torch, gen, groups, m, k)
    stored = w if trans == OP_T else w.mT.contiguous()
    lda = k if trans == OP_T else m
    offsets = torch.tensor(ends, dtype=torch.int32, device="cuda")
    want = by_group(torch, x, w, ends).to(dtype_of(torch, ctype))
    cbuf, c = output(torch, n * m, dtype_of(torch, ctype))
    for _ in range(5):
        c.fill_(float("nan"))
        handle.grouped_gemm_n(trans, m, n, k, groups, offsets, 1.0, stored, lda, m * k, x, k, 0.0, c,
                              ctype, m)
        assert torch.equal(c.view(n, m), want)
    assert guards_ok(cbuf) and sg.get_device_errors() == 0


@pytest.mark.parametrize("ctype", [FP32, BF16])
def test_odd_pieces_of_tokens_fp8(cuda, handle, ctype):
    torch = cuda
    gen = generator(torch, 22)
    lengths, m, k = ODD_PIECES["lengths"], ODD_PIECES["m"], ODD_PIECES["k"]
    ends, groups = ends_of(lengths), len(lengths)
    n = ends[-1]
    x, w = whole(torch, gen, n, k), whole(torch, gen, groups, m, k)
    xs = 2.0 ** torch.randint(-2, 3, (n, 1), generator=gen, device="cuda").float()
    ws = 2.0 ** torch.randint(-2, 3, (groups, m // 128, 1), generator=gen, device="cuda").float()
    offsets = torch.tensor(ends, dtype=torch.int32, device="cuda")
    want = by_group(torch, x * xs.to(x.dtype), w * ws.repeat_interleave(128, 1).to(w.dtype), ends)
    want = want.to(dtype_of(torch, ctype))
    q, wq = x.to(torch.float8_e4m3fn), w.to(torch.float8_e4m3fn)
    cbuf, c = output(torch, n * m, dtype_of(torch, ctype))
    for _ in range(5):
        c.fill_(float("nan"))
        handle.grouped_gemm_fp8(m, n, k, groups, offsets, wq, k, m * k, ws, 1, m // 128, q, k, xs, 1,
                                c, ctype, m)
        assert torch.equal(c.view(n, m), want)
    assert guards_ok(cbuf) and sg.get_device_errors() == 0


@pytest.mark.parametrize("ctype", [FP32, BF16])
@pytest.mark.parametrize("most", [1, 3])
def test_odd_pieces_of_gradients(cuda, handle, most, ctype):
    """64 experts of up to three tokens, some of none (nothing is waited for
    before their zeros are staged): 24 tiles each for 74 workers, the last
    columns in 7 pieces."""
    torch = cuda
    gen = generator(torch, 23 + most)
    m, n, groups = 1536, 1000, 64
    lengths = torch.randint(0, most + 1, (groups,), generator=gen, device="cuda").tolist()
    ends = ends_of(lengths, head=1)
    k = ends[-1] + 1
    a, b = whole(torch, gen, k, m), whole(torch, gen, k, n)
    a[0] = b[-1] = float("nan")   # outside the groups
    offsets = torch.tensor(ends, dtype=torch.int32, device="cuda")
    type_ = dtype_of(torch, ctype)
    want = torch.stack([(b[lo:hi].double().T @ a[lo:hi].double()).to(type_)
                        for lo, hi in zip(ends, ends[1:])])
    cbuf, c = output(torch, groups * n * m, type_)
    for _ in range(5):
        c.fill_(float("nan"))
        handle.grouped_gemm_k(m, n, k, groups, offsets, 1.0, a, m, b, n, 0.0, c, ctype, m, n * m)
        assert torch.equal(c.view(groups, n, m), want)
    assert guards_ok(cbuf) and sg.get_device_errors() == 0


@pytest.mark.parametrize("m", [1985, 1990, 1991, 1993, 1996, 1999, 2000])
@pytest.mark.parametrize("ctype", [FP32, BF16])
def test_rows_beyond_a_result_stay(cuda, handle, ctype, m):
    """Results written into the first m of 2000 rows, which may belong to
    anything: TMA writes whole units of 16 bytes."""
    torch = cuda
    gen = generator(torch, 25 + m)
    n, k, ldc = 4096, 64, 2000
    type_ = dtype_of(torch, ctype)
    x, w = whole(torch, gen, n, k), whole(torch, gen, 1, m, k)
    tokens = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    few = torch.tensor([0, 112], dtype=torch.int32, device="cuda")
    ones = torch.ones(n, device="cuda")
    q, wq = x.to(torch.float8_e4m3fn), w.to(torch.float8_e4m3fn)
    b = whole(torch, gen, k, 512)
    a = whole(torch, gen, k, ldc)   # m of its columns
    depth = torch.tensor([0, k], dtype=torch.int32, device="cuda")

    def check(rows, call, want):
        buf, c = output(torch, rows * ldc, type_)
        before = c.clone().view(rows, ldc)
        call(c)
        before[:, :m] = want.to(type_)
        assert torch.equal(c.view(rows, ldc), before) and guards_ok(buf)

    for rows, offsets in ((n, tokens), (112, few)):   # pairs of CTAs, single ones
        want = by_group(torch, x[:rows], w, [0, rows])
        check(rows, lambda c: handle.grouped_gemm_n(OP_T, m, rows, k, 1, offsets, 1.0, w, k, 0, x, k, 0.0,
                                                    c, ctype, ldc), want)
        check(rows, lambda c: handle.gemm_fp8(m, rows, k, wq, k, ones, 1, q, k, ones, 1, c, ctype, ldc),
              want)
    check(512, lambda c: handle.grouped_gemm_k(m, 512, k, 1, depth, 1.0, a, ldc, b, 512, 0.0, c, ctype, ldc,
                                               0), b.double().T @ a[:, :m].double())
