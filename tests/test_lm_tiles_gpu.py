"""Every kernel of the language-model products, most where a worker takes several
tiles one after the other: ring, accumulators, scales and staging buffers go
from tile to tile. Operands of the products are small whole numbers, so every
sum is exact in FP32 and a result is equal to the definition's, rounded once.
"""
import pytest

import sgblas_b200 as sg
from tests.lm_cases import GRADIENTS, ODD_PIECES, ORTHOGONAL, RAGGED
from tests.test_lm_products_gpu import ABC, dtype_of, generator, guards_ok, newton_schulz, output

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


# ---- every kernel --------------------------------------------------------------------

@pytest.mark.parametrize("case", RAGGED, ids=lambda c: c["name"])
@pytest.mark.parametrize("ctype,beta,pad", [(BF16, 0.0, 0), (BF16, 0.0, 8), (FP32, 0.0, 0), (FP32, 0.0, 3),
                                            (BF16, 1.0, 0), (FP32, 0.5, 1)])
@pytest.mark.parametrize("trans", [OP_T, OP_N])
def test_ragged_products(cuda, handle, trans, ctype, beta, pad, case):
    """alpha A B + beta C with tokens before and after all groups, which stay as they are."""
    torch = cuda
    lengths, m, k = case["lengths"], case["m"], case["k"]
    gen = generator(torch, 31 + k)
    ends, groups, alpha = ends_of(lengths, head=1), len(lengths), -2.0
    n = ends[-1] + 2
    x, w = whole(torch, gen, n, k), whole(torch, gen, groups, m, k)
    x[0], x[-1] = float("nan"), float("inf")
    stored = w if trans == OP_T else w.mT.contiguous()
    lda = k if trans == OP_T else m
    offsets = torch.tensor(ends, dtype=torch.int32, device="cuda")
    type_, ldc = dtype_of(torch, ctype), m + pad
    cbuf, c = output(torch, n * ldc, type_)
    c0 = whole(torch, gen, n, ldc).to(type_)
    c.copy_(c0.reshape(-1))
    want = c0.clone()
    inside = slice(1, ends[-1])
    want[inside, :m] = (alpha * by_group(torch, x, w, ends)[inside] +
                        beta * c0[inside, :m].double()).to(type_)
    handle.grouped_gemm_n(trans, m, n, k, groups, offsets, alpha, stored, lda, m * k, x, k, beta, c,
                          ctype, ldc)
    assert torch.equal(c.view(n, ldc), want)
    assert guards_ok(cbuf) and sg.get_device_errors() == 0


@pytest.mark.parametrize("case", RAGGED, ids=lambda c: c["name"])
@pytest.mark.parametrize("ctype,pad", [(BF16, 0), (BF16, 8), (BF16, 1), (FP32, 0), (FP32, 3)])
def test_ragged_products_fp8(cuda, handle, ctype, pad, case):
    """Scales are powers of two within 2^-2 .. 2^2, so the blocks' sums are exact too."""
    torch = cuda
    lengths, m, k = case["lengths"], case["m"], case["k"]
    gen = generator(torch, 41 + k)
    ends, groups = ends_of(lengths), len(lengths)
    n = ends[-1] + (groups > 1)
    kb, mb = -(-k // 128), -(-m // 128)
    lds, ldc = kb + pad, m + pad
    x, w = whole(torch, gen, n, k), whole(torch, gen, groups, m, k)
    power = lambda *s: 2.0 ** torch.randint(-2, 3, s, generator=gen, device="cuda").float()  # noqa: E731
    xs, ws = power(n, lds), power(groups, mb, lds)
    spread = lambda v: v[..., :kb].repeat_interleave(128, -1)[..., :k]  # noqa: E731
    want = by_group(torch, x.float() * spread(xs),
                    w.float() * spread(ws).repeat_interleave(128, 1)[:, :m], ends)
    type_ = dtype_of(torch, ctype)
    q, wq = x.to(torch.float8_e4m3fn), w.to(torch.float8_e4m3fn)
    cbuf, c = output(torch, n * ldc, type_)
    c0 = c.clone().view(n, ldc)
    if groups == 1:
        handle.gemm_fp8(m, n, k, wq, k, ws, lds, q, k, xs, lds, c, ctype, ldc)
    else:
        offsets = torch.tensor(ends, dtype=torch.int32, device="cuda")
        handle.grouped_gemm_fp8(m, n, k, groups, offsets, wq, k, m * k, ws, lds, mb * lds, q, k, xs, lds,
                                c, ctype, ldc)
    c0[:ends[-1], :m] = want[:ends[-1]].to(type_)
    assert torch.equal(c.view(n, ldc), c0)
    assert guards_ok(cbuf) and sg.get_device_errors() == 0


@pytest.mark.parametrize("m,n", GRADIENTS)
@pytest.mark.parametrize("ctype,beta,pad", [(FP32, 0.0, 0), (FP32, 1.0, 0), (FP32, 0.0, 1), (BF16, 0.0, 0),
                                            (BF16, 0.0, 8), (BF16, 0.5, 0)])
def test_ragged_gradients(cuda, handle, ctype, beta, pad, m, n):
    """Twelve groups, cut slices of every kind, four tiles per pair of CTAs."""
    torch = cuda
    gen = generator(torch, 51 + m)
    lengths = [1, 63, 64, 65, 0, 127, 129, 200, 31, 500, 17, 300]
    ends, groups, alpha = ends_of(lengths, head=1), len(lengths), -2.0
    k = ends[-1] + 1
    a, b = whole(torch, gen, k, m), whole(torch, gen, k, n)
    a[0], b[-1] = float("nan"), float("inf")
    offsets = torch.tensor(ends, dtype=torch.int32, device="cuda")
    type_, ldc = dtype_of(torch, ctype), m + pad
    cbuf, c = output(torch, groups * n * ldc, type_)
    c0 = whole(torch, gen, groups, n, ldc).to(type_)
    c.copy_(c0.reshape(-1))
    want = c0.clone()
    for g, (lo, hi) in enumerate(zip(ends, ends[1:])):
        want[g, :, :m] = (alpha * (b[lo:hi].double().T @ a[lo:hi].double()) +
                          beta * c0[g, :, :m].double()).to(type_)
    handle.grouped_gemm_k(m, n, k, groups, offsets, alpha, a, m, b, n, beta, c, ctype, ldc, n * ldc)
    assert torch.equal(c.view(groups, n, ldc), want)
    assert guards_ok(cbuf) and sg.get_device_errors() == 0


@pytest.mark.parametrize("rows,cols,batch", ORTHOGONAL)
def test_orthogonalize(cuda, handle, rows, cols, batch):
    """The bound of the test of the same name for smaller matrices, with the same
    inputs: BF16's rounding, and the last product's operands of 11 bits."""
    torch = cuda
    gen = generator(torch, rows)
    rank = min(rows, cols) // 8
    g = 1e-3 * (torch.randn(batch, rows, rank, generator=gen, device="cuda") @
                torch.randn(batch, rank, cols, generator=gen, device="cuda") +
                0.3 * torch.randn(batch, rows, cols, generator=gen, device="cuda"))
    buf, o = output(torch, batch * rows * cols, torch.bfloat16)
    handle.orthogonalize(cols, rows, batch, 5, ABC, 1e-7, 1.0, g, FP32, cols, rows * cols, o, cols,
                         rows * cols)
    got = o.view(batch, rows, cols).double()
    for i in range(batch):
        want = newton_schulz(g[i], 5, ABC, 1e-7, 1.0)
        rel = ((got[i] - want).norm() / want.norm()).item()
        assert rel <= 2.0 ** -9 + 2.0 ** -10, (i, rel)
    assert guards_ok(buf) and sg.get_device_errors() == 0


@pytest.mark.parametrize("type_", ["float32", "bfloat16"])
@pytest.mark.parametrize("exponent", [-149, -140, -100, -70, 60, 70, 100, 124])
def test_orthogonalize_any_magnitude(cuda, handle, exponent, type_):
    """G scaled by a power of two gives, without an eps, what G gives: the squares
    of its values lie outside FP32's range. Below 2^-126 G itself is coarser, and in
    BF16 nothing below 2^-134, so the definition takes what it holds (0 / 0 of
    nothing). The bound is that of test_orthogonalize."""
    torch = cuda
    g = torch.randn(1, 200, 300, generator=generator(torch, 61), device="cuda", dtype=torch.float64)
    g = (g * 2.0 ** exponent).to(getattr(torch, type_)).repeat(2, 1, 1)
    g[1] = 0.0
    o = torch.empty(2, 200, 300, dtype=torch.bfloat16, device="cuda")
    code = BF16 if type_ == "bfloat16" else FP32
    for eps in (0.0, 2.0 ** (exponent - 2) if exponent > 0 else 1e-7):
        handle.orthogonalize(300, 200, 2, 5, ABC, eps, 1.0, g, code, 300, 60000, o, 300, 60000)
        want = newton_schulz(g[0], 5, ABC, torch.tensor(eps, dtype=torch.float32).item(), 1.0)
        if torch.isnan(want).all():
            assert not g.any() and torch.isnan(o).all()
        elif eps == 0.0 or exponent > 0:
            assert ((o[0].double() - want).norm() / want.norm()).item() <= 2.0 ** -9 + 2.0 ** -10
        else:   # next to eps there is little left of G: an absolute 2^-37 per value of X, times 485
            assert ((o[0].double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -27).all()
        assert (o[1] == 0).all() if eps > 0.0 else torch.isnan(o[1]).all()
    assert sg.get_device_errors() == 0


@pytest.mark.parametrize("trans", [None, OP_T, OP_N])
def test_long_sums_are_not_biased(cuda, handle, trans):
    """Positive products, so that every truncation of a chain goes the same way,
    and a BF16 result: the mean over 16384 of them shows what its own rounding
    (up to 2^-8, without bias: 1.7e-3 / 128 in the mean, five times that allowed)
    hides. A chain of 4096 of k is off by 256 instructions' 2^-22 at most; its 256
    pieces are added with rounding to nearest, 2^-24 each at most.
    """
    torch = cuda
    gen = generator(torch, 71)
    k, m = 1 << 20, 128
    # Each row and column of the result of its own size, so their roundings differ.
    a, b = ((torch.rand(k, m, generator=gen, device="cuda").add_(0.5) *
             torch.exp2(torch.rand(m, generator=gen, device="cuda"))).to(torch.bfloat16)
            for _ in range(2))
    c = torch.empty(m, m, dtype=torch.bfloat16, device="cuda")
    offsets = torch.tensor([0, k if trans is None else m], dtype=torch.int32, device="cuda")
    if trans is None:      # a weight gradient of 2^20 tokens
        handle.grouped_gemm_k(m, m, k, 1, offsets, 1.0, a, m, b, m, 0.0, c, BF16, m, 0)
    else:
        tokens = b.T.contiguous()
        w, lda = (a.T.contiguous(), k) if trans == OP_T else (a, m)
        handle.grouped_gemm_n(trans, m, m, k, 1, offsets, 1.0, w, lda, 0, tokens, k, 0.0, c, BF16, m)
    want = b.double().T @ a.double()
    bias = ((c.double() - want) / want).mean().abs().item()
    assert bias <= 5 * 1.7e-3 / 128 + 256 * 2.0 ** -22 + 256 * 2.0 ** -24, bias
    assert sg.get_device_errors() == 0


def test_a_graph_outlives_a_larger_call(cuda, lib):
    """A captured call keeps the workspace it was captured with."""
    torch = cuda
    gen = generator(torch, 81)
    m, k, n = 301, 77, 200
    x, w = whole(torch, gen, n, k), whole(torch, gen, 1, m, k)
    large = torch.full((1, 5001, 5001), float("nan"), dtype=torch.bfloat16, device="cuda")
    offsets = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    y, z = torch.empty(n, m, device="cuda"), torch.empty(5001, 5001, device="cuda")
    end = torch.tensor([0, 5001], dtype=torch.int32, device="cuda")
    with lib.Handle() as h:
        call = lambda: h.grouped_gemm_n(OP_T, m, n, k, 1, offsets, 1.0, w, k, 0, x, k, 0.0, y, FP32, m)  # noqa: E731
        call()
        stream = torch.cuda.Stream()
        h.set_stream(stream)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            call()
        for _ in range(2):
            h.grouped_gemm_n(OP_T, 5001, 5001, 5001, 1, end, 1.0, large, 5001, 0, large, 5001, 0.0, z, FP32,
                             5001)
            torch.cuda.synchronize()
            y.zero_()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, (x.double() @ w[0].double().T).float())
        del graph
    assert sg.get_device_errors() == 0
