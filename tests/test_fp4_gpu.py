"""4-bit quantisation and products (MXFP4) against their definitions.

Quantisation is exact but for e2m1's own rounding: codes and bytes are compared for
equality. So are products of random codes with scales of 2^-2 to 2^2: every term is a
multiple of 2^-6, sums stay below 2^17 (the largest magnitude of a case is checked), so
FP32 holds every partial sum, and C is the exact sum, rounded once in BF16.
"""
import pytest
import torch

import sgblas_b200 as sg
from tests.layer_util import HALF, TYPES, Matrix, generator
from tests.lm_cases import RAGGED

pytestmark = pytest.mark.gpu
CODE = {"bf16": sg.SGBLAS_TYPE_BF16, "fp32": sg.SGBLAS_TYPE_FP32}
VALUES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def nearest(v):
    """Codes of the e2m1 values nearest to v (64 bits), ties to the even code."""
    grid = torch.tensor(VALUES, dtype=torch.float64, device=v.device)
    a = v.abs().clamp(max=6.0)
    hi = torch.searchsorted(grid, a).clamp(max=7)
    lo = (hi - 1).clamp(min=0)
    up, down = grid[hi] - a, a - grid[lo]
    code = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    return (code + 8 * torch.signbit(v)).to(torch.uint8)


def quantized(x):
    """The definition: codes, a byte per value, and scale bytes."""
    rows, k = x.shape
    v = torch.nn.functional.pad(x.double(), (0, -k % 32)).view(rows, -1, 32)
    top = v.abs().amax(dim=2)
    # FP32's exponent byte; 0 for zeros and subnormals.
    exponent = torch.where(top >= 2.0 ** -126, torch.frexp(top).exponent.long() + 126, torch.zeros_like(top).long())
    byte = (exponent - 2).clamp(min=0)
    codes = nearest(v * torch.exp2(127.0 - byte.double())[:, :, None]).view(rows, -1)[:, :k]
    return codes, byte.to(torch.uint8)


def packed(codes):
    rows, k = codes.shape
    c = torch.nn.functional.pad(codes, (0, k % 2))
    return c[:, 0::2] | (c[:, 1::2] << 4)


def values(codes, byte):
    table = torch.tensor(VALUES + [-v for v in VALUES], dtype=torch.float64, device=codes.device)
    return table[codes.long()] * torch.exp2(byte.double() - 127).repeat_interleave(32, dim=1)[:, :codes.shape[1]]


def check_quantize(handle, x, type_, ld=0, shift=0, ldq=None, ldscale=None, q_shift=0):
    rows, k = x.shape
    kb, ks = -(-k // 2), -(-k // 32)
    src = Matrix(rows, k, TYPES[type_], k + ld, shift, x)
    q = Matrix(rows, kb, torch.uint8, kb if ldq is None else ldq, q_shift)
    s = Matrix(rows, ks, torch.uint8, ks if ldscale is None else ldscale, q_shift)
    handle.quantize_fp4(k, rows, src, CODE[type_], src.ld, q, q.ld, s, s.ld)
    codes, byte = quantized(src.view)
    assert torch.equal(s.view, byte)
    assert torch.equal(q.view, packed(codes))
    assert not any(m.unmarked() for m in (src, q, s))


@pytest.mark.parametrize("type_", ["bf16", "fp32"])
@pytest.mark.parametrize("k,rows", [(1, 1), (2, 5), (16, 3), (17, 2), (31, 4), (32, 700), (33, 9), (63, 64), (100, 33),
                                    (1537, 20), (2048, 300), (4096, 1), (4100, 7)])
def test_quantize(cuda, handle, type_, k, rows):
    gen = generator(k + rows)
    x = torch.randn(rows, k, generator=gen, device="cuda") * torch.exp2(
        torch.randint(-20, 20, (rows, k), generator=gen, device="cuda").float() * (torch.rand(rows, 1, generator=gen, device="cuda") < 0.5))
    unit8, unit16 = -(-(-(-k // 2)) // 8) * 8, -(-(-(-k // 32)) // 16) * 16
    check_quantize(handle, x, type_)
    check_quantize(handle, x, type_, ld=-k % 8, ldq=unit8, ldscale=unit16)        # vectors
    check_quantize(handle, x, type_, ld=3, shift=1, ldq=unit8 + 1, q_shift=3)     # scalars


def test_quantize_ties_and_ends(cuda, handle):
    """Every border between values, its neighbours, both signs, from subnormals to the largest."""
    borders = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.9375], device="cuda")
    near = torch.cat([borders, torch.nextafter(borders, borders + 1), torch.nextafter(borders, borders - 1)])
    near = torch.cat([near, -near])                       # 60 values
    for power in (-149, -140, -128, -127, -126, -100, -3, 0, 1, 77, 120, 125):
        row = torch.ldexp(near, torch.tensor(power, device="cuda"))
        blocks = torch.zeros(60, 32, device="cuda")
        blocks[:, 0] = row                                # alone: the block's largest
        blocks[:, 1] = torch.ldexp(torch.tensor(4.0, device="cuda"), torch.tensor(power, device="cuda"))
        blocks[:, 2] = -0.0
        blocks[:, 3:] = row.roll(7)[:, None]
        blocks = blocks[blocks.isfinite().all(dim=1)]
        check_quantize(handle, blocks.contiguous(), "fp32")
        check_quantize(handle, blocks.to(torch.bfloat16).float().contiguous(), "bf16")


def test_quantize_nan_and_infinity(cuda, handle):
    x = torch.randn(4, 96, device="cuda")
    x[1, 40], x[2, 95], x[3, 0] = float("nan"), float("inf"), -float("inf")
    q, s = torch.zeros(4, 48, dtype=torch.uint8, device="cuda"), torch.zeros(4, 3, dtype=torch.uint8, device="cuda")
    handle.quantize_fp4(96, 4, x, CODE["fp32"], 96, q, 48, s, 3)
    assert (s == 255).tolist() == [[False] * 3, [False, True, False], [False, False, True], [True, False, False]]
    y = torch.zeros(4, 4, device="cuda")
    good_q, good_s = torch.full((4, 48), 0x22, dtype=torch.uint8, device="cuda"), torch.full((4, 3), 127, dtype=torch.uint8, device="cuda")
    handle.gemm_fp4(4, 4, 96, good_q, 48, good_s, 3, q, 48, s, 3, y, CODE["fp32"], 4)
    assert y.isnan().all(dim=1).tolist() == [False, True, True, True]   # their columns, no others
    assert bool(y[0].isfinite().all())


@pytest.mark.parametrize("type_", ["bf16", "fp32"])
def test_quantize_batch(cuda, handle, type_):
    b, rows, k = 3, 40, 200
    x = torch.randn(b, rows + 2, k + 8, device="cuda").to(TYPES[type_])
    q = torch.zeros(b, rows, 104, dtype=torch.uint8, device="cuda")
    s = torch.zeros(b, rows, 7, dtype=torch.uint8, device="cuda")
    handle.quantize_fp4(k, rows, x, CODE[type_], k + 8, q, 104, s, 7, batch=b, stride_x=(rows + 2) * (k + 8),
                        stride_q=rows * 104, stride_scale=rows * 7)
    for i in range(b):
        codes, byte = quantized(x[i, :rows, :k])
        assert torch.equal(s[i], byte) and torch.equal(q[i, :, :100], packed(codes))
    assert bool((q[:, :, 100:] == 0).all())


# ---- products ------------------------------------------------------------------------

class Operands:
    """Random codes and scales of groups' weights and of tokens, with their values."""

    def __init__(self, m, k, lengths, seed=0, ld=0, shift=0, lead=0, tail=0):
        gen = generator(seed)
        rand = lambda high, *s: torch.randint(0, high, s, generator=gen, device="cuda").to(torch.uint8)  # noqa: E731
        self.m, self.k, self.groups, self.lengths = m, k, len(lengths), lengths
        self.n = lead + sum(lengths) + tail
        kb, ks = -(-k // 2), -(-k // 32)
        up = lambda v: -(-v // 16) * 16  # noqa: E731
        self.lda, self.ldsa = (kb + ld, ks + ld) if ld else (up(kb), up(ks))
        wc, ws = rand(16, self.groups * m, k), 125 + rand(5, self.groups * m, ks)
        xc, xs = rand(16, self.n, k), 125 + rand(5, self.n, ks)
        self.a = Matrix(self.groups * m, kb, torch.uint8, self.lda, shift, packed(wc))
        self.sa = Matrix(self.groups * m, ks, torch.uint8, self.ldsa, shift, ws)
        self.b = Matrix(self.n, kb, torch.uint8, self.lda, shift, packed(xc))
        self.sb = Matrix(self.n, ks, torch.uint8, self.ldsa, shift, xs)
        self.w, self.x = values(wc, ws).view(self.groups, m, k), values(xc, xs)
        ends = [lead]
        for length in lengths:
            ends.append(ends[-1] + length)
        self.ends = ends
        self.offsets = torch.tensor(ends, dtype=torch.int32, device="cuda")

    def want(self):
        y = torch.zeros(self.n, self.m, dtype=torch.float64, device="cuda")
        for g in range(self.groups):
            lo, hi = self.ends[g], self.ends[g + 1]
            y[lo:hi] = self.x[lo:hi] @ self.w[g].mT
        assert float(y.abs().max()) < 2.0 ** 17 if y.numel() else True
        return y

    def run(self, handle, ctype, c):
        handle.grouped_gemm_fp4(self.m, self.n, self.k, self.groups, self.offsets, self.a, self.lda, self.m * self.lda,
                                self.sa, self.ldsa, self.m * self.ldsa, self.b, self.lda, self.sb, self.ldsa, c, CODE[ctype], c.ld)


def check_product(handle, ops, ctype, ldc=0, shift=0):
    c = Matrix(ops.n, ops.m, TYPES[ctype], ops.m + ldc, shift)
    before = c.view.clone()
    ops.run(handle, ctype, c)
    want = ops.want()
    lo, hi = ops.ends[0], ops.ends[-1]
    assert torch.equal(c.view[lo:hi], want[lo:hi].float().to(TYPES[ctype]))
    for part in (slice(0, lo), slice(hi, ops.n)):   # columns of no group
        assert torch.equal(c.view[part].view(torch.uint8), before[part].view(torch.uint8))
    assert not any(v.unmarked() for v in (c, ops.a, ops.b, ops.sa, ops.sb))


SMALL = [dict(m=1, k=1, lengths=[1]), dict(m=8, k=32, lengths=[3]), dict(m=128, k=256, lengths=[16]),
         dict(m=130, k=258, lengths=[5, 0, 1]), dict(m=64, k=33, lengths=[2, 7]), dict(m=200, k=511, lengths=[20, 31]),
         dict(m=127, k=513, lengths=[40]), dict(m=300, k=1000, lengths=[100, 0, 29]), dict(m=1000, k=2048, lengths=[130])]


@pytest.mark.parametrize("ctype", ["fp32", "bf16"])
@pytest.mark.parametrize("case", SMALL, ids=lambda c: f"{c['m']}x{c['k']}x{len(c['lengths'])}")
@pytest.mark.parametrize("ld,shift", [(0, 0), (3, 1)])
def test_small_products(cuda, handle, ctype, case, ld, shift):
    ops = Operands(case["m"], case["k"], case["lengths"], seed=case["k"], ld=ld, shift=shift)
    check_product(handle, ops, ctype, ldc=ld, shift=shift)


# Pairs of CTAs: tiles of 256 x 192, groups that end inside either half of one, rows and
# columns that are no multiple of anything, k from a chunk of scales to several chains.
PAIRS = [dict(name="pairs", lengths=[2999, 1, 0, 2303, 777, 3333, 193, 191, 97], m=3999, k=2120),
         dict(name="pairs, edges", lengths=[192, 384, 96, 1920, 2000, 3600, 1111, 2222], m=4112, k=4100),
         dict(name="pairs, one group", lengths=[7777], m=6001, k=1543)]


@pytest.mark.parametrize("ctype", ["fp32", "bf16"])
@pytest.mark.parametrize("case", RAGGED + PAIRS, ids=lambda c: c["name"])
def test_ragged_products(cuda, handle, ctype, case):
    check_product(handle, Operands(case["m"], case["k"], case["lengths"], seed=1), ctype)


ONE_MATRIX = [(4096, 1, 4096), (2048, 40, 4000), (4096, 600, 700), (4104, 2500, 520), (1999, 3001, 390),
              (4096, 4100, 1100), (6008, 6100, 1542)]


@pytest.mark.parametrize("ctype", ["fp32", "bf16"])
@pytest.mark.parametrize("m,n,k", ONE_MATRIX)
def test_one_matrix(cuda, handle, ctype, m, n, k):
    ops = Operands(m, k, [n], seed=n)
    c = Matrix(n, m, TYPES[ctype])
    handle.gemm_fp4(m, n, k, ops.a, ops.lda, ops.sa, ops.ldsa, ops.b, ops.lda, ops.sb, ops.ldsa, c, CODE[ctype], m)
    assert torch.equal(c.view, ops.want().float().to(TYPES[ctype]))
    assert not c.unmarked()


@pytest.mark.parametrize("lengths,sizes", [([300, 0, 40], (520, 1001)), ([3, 1, 0, 5], (520, 1001)),
                                           ([20] * 3, (520, 1001)), ([2500, 3700, 0, 2800], (4096, 4001))])
def test_columns_of_no_group_stay(cuda, handle, lengths, sizes):
    for m in sizes:
        for ctype in ("fp32", "bf16"):
            k = 300 if m < 4000 else 1542
            check_product(handle, Operands(m, k, lengths, seed=2, lead=5, tail=77), ctype)


def test_offsets_outside_count_as_the_nearer_end(cuda, handle):
    ops = Operands(256, 300, [10, 20, 30], seed=3)
    want = ops.want()
    ops.offsets.copy_(torch.tensor([-5, 10, 30, 1 << 30], dtype=torch.int32))
    c = Matrix(ops.n, 256, torch.float32)
    ops.run(handle, "fp32", c)
    assert torch.equal(c.view, want.float()) and not c.unmarked()


# Of pairs of CTAs (test_layer_dispatch.py).
DECREASING = dict(m=4096, k=1544, n=20000, groups=64)


@pytest.mark.parametrize("way", ["swinging", "backwards", "anything"])
def test_offsets_that_decrease_reach_nothing_else(cuda, handle, way):
    """They give no result, but more tiles than the host has counted: all that is written
    is the workspace and C, and the next product is right."""
    m, k, n, groups = (DECREASING[key] for key in ("m", "k", "n", "groups"))
    ops = Operands(m, k, [n // groups] * groups, seed=12, tail=n % groups)
    g = torch.arange(groups + 1, device="cuda")
    good = ops.offsets.clone()
    bad = {"swinging": g % 2 * n, "backwards": n - g * (n // groups),
           "anything": torch.randint(-2**31, 2**31 - 1, (groups + 1,), generator=generator(1), device="cuda")}[way]
    for ctype in ("bf16", "fp32"):
        c = Matrix(n, m, TYPES[ctype])
        ops.offsets.copy_(bad)
        ops.run(handle, ctype, c)
        torch.cuda.synchronize()
        assert not any(v.unmarked() for v in (c, ops.a, ops.b, ops.sa, ops.sb))
        ops.offsets.copy_(good)
        check_product(handle, ops, ctype)
    assert sg.get_device_errors() == 0


def test_neighbours_do_not_reach_a_column(cuda, handle):
    """NaN scales of one group's tokens and weights stay in that group."""
    for m, lengths in ((300, [200, 100, 300]), (300, [3, 2, 4]), (300, [8, 13, 9]), (4001, [2500, 3000, 3700])):
        ops = Operands(m, 1544, lengths, seed=4)
        want = ops.want()
        ops.sb.view[ops.ends[1]:ops.ends[2]] = 255
        ops.sa.view[m:2 * m] = 255
        c = Matrix(ops.n, m, torch.float32)
        ops.run(handle, "fp32", c)
        assert bool(c.view[ops.ends[1]:ops.ends[2]].isnan().all())
        for lo, hi in ((0, ops.ends[1]), (ops.ends[2], ops.n)):
            assert torch.equal(c.view[lo:hi], want[lo:hi].float())


def test_no_products(cuda, handle):
    """k == 0: zeros."""
    for n in (3, 500):
        c = Matrix(n, 100, torch.float32, 104)
        handle.gemm_fp4(100, n, 0, None, 1, None, 1, None, 1, None, 1, c, CODE["fp32"], 104)
        assert bool((c.view == 0).all()) and not c.unmarked()


@pytest.mark.parametrize("ctype", ["fp32", "bf16"])
@pytest.mark.parametrize("m,k,lengths", [(1024, 4096, [1]), (2048, 2048, [12] * 16), (2048, 4096, [1500, 900]),
                                         (4096, 4608, [3500, 4000])])
def test_real_values(cuda, handle, ctype, m, k, lengths):
    """Quantised activations and weights: sums of any size. An FP32 C is chained over
    32 instructions (2^-22 of the terms each, truncated) and pieces of 2048 of k (2^-24
    each, and of a split k, at most 32); a BF16 C over 64 instructions and its own half step."""
    gen = generator(k)
    n, groups = sum(lengths), len(lengths)
    x = torch.randn(n, k, generator=gen, device="cuda").to(torch.bfloat16)
    w = (torch.randn(groups, m, k, generator=gen, device="cuda") / k ** 0.5).to(torch.bfloat16)
    q = [torch.empty(n, k // 2, dtype=torch.uint8, device="cuda"), torch.empty(groups, m, k // 2, dtype=torch.uint8, device="cuda")]
    s = [torch.empty(n, k // 32, dtype=torch.uint8, device="cuda"), torch.empty(groups, m, k // 32, dtype=torch.uint8, device="cuda")]
    handle.quantize_fp4(k, n, x, CODE["bf16"], k, q[0], k // 2, s[0], k // 32)
    handle.quantize_fp4(k, m, w, CODE["bf16"], k, q[1], k // 2, s[1], k // 32, batch=groups, stride_x=m * k,
                        stride_q=m * k // 2, stride_scale=m * k // 32)
    offsets = torch.tensor([0] + torch.tensor(lengths).cumsum(0).tolist(), dtype=torch.int32, device="cuda")
    c = Matrix(n, m, TYPES[ctype])
    handle.grouped_gemm_fp4(m, n, k, groups, offsets, q[1], k // 2, m * k // 2, s[1], k // 32, m * k // 32, q[0], k // 2,
                            s[0], k // 32, c, CODE[ctype], m)
    xv, at = values(*quantized(x)), 0
    tolerance = 32 * 2.0 ** -22 + 32 * 2.0 ** -24 if ctype == "fp32" else 64 * 2.0 ** -22
    for g, length in enumerate(lengths):
        wv = values(*quantized(w[g]))
        part = xv[at:at + length]
        want, size = part @ wv.mT, part.abs() @ wv.abs().mT
        err = (c.view[at:at + length].double() - want).abs()
        assert bool((err <= tolerance * size + HALF[TYPES[ctype]] * want.abs()).all())
        at += length


@pytest.mark.parametrize("m,lengths", [(512, [3, 40, 0, 21]), (512, [1, 0, 9, 2]), (4096, [2500, 0, 4000, 3000])])
@pytest.mark.parametrize("prepared", [True, False])
def test_fp4_in_a_graph_and_on_a_stream(cuda, lib, m, lengths, prepared):
    """A captured step reads new tokens, weights and offsets on each replay, with the
    workspace for a pair's scales or without."""
    k = 1536
    ops = Operands(m, k, lengths, seed=6)
    other = Operands(m, k, lengths[1:] + lengths[:1], seed=7)
    c = Matrix(ops.n, m, torch.float32)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with lib.Handle() as h:
        h.set_stream(stream)
        if prepared:
            ops.run(h, "fp32", c)
            torch.cuda.synchronize()
            assert torch.equal(c.view, ops.want().float())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            ops.run(h, "fp32", c)
        for source in (other, ops):
            for mine, theirs in ((ops.a, source.a), (ops.b, source.b), (ops.sa, source.sa), (ops.sb, source.sb)):
                mine.view.copy_(theirs.view.clone())
            ops.offsets.copy_(source.offsets.clone())
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            if source is other:
                assert torch.equal(c.view, other.want().float())
        graph.reset()


@pytest.mark.parametrize("ctype", ["fp32", "bf16"])
def test_products_without_a_workspace_are_the_same(cuda, lib, ctype):
    """Inside a capture without a workspace large products take smaller tiles, whose sums
    are made in the same order: equal results for values of any size."""
    m, k, lengths = 4096, 4608, [3500, 4000]
    n = sum(lengths)
    gen = generator(7)
    q = [torch.randint(0, 256, (rows, k // 2), generator=gen, device="cuda").to(torch.uint8) for rows in (2 * m, n)]
    s = [torch.randint(110, 140, (rows, k // 32), generator=gen, device="cuda").to(torch.uint8) for rows in (2 * m, n)]
    offsets = torch.tensor([0, 3500, 7500], dtype=torch.int32, device="cuda")
    out = [torch.zeros(n, m, dtype=TYPES[ctype], device="cuda") for _ in range(2)]
    with lib.Handle() as h:
        run = lambda c: h.grouped_gemm_fp4(m, n, k, 2, offsets, q[0], k // 2, m * k // 2, s[0], k // 32, m * k // 32,  # noqa: E731
                                           q[1], k // 2, s[1], k // 32, c, CODE[ctype], m)
        stream = torch.cuda.Stream()
        h.set_stream(stream)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            run(out[0])
        graph.replay()
        torch.cuda.synchronize()
        run(out[1])
        torch.cuda.synchronize()
        graph.reset()
    assert torch.equal(out[0], out[1])


def test_unaligned_operands_in_a_capture_need_a_workspace(cuda, lib):
    ops = Operands(64, 77, [20], seed=8, ld=1, shift=1)
    c = Matrix(20, 64, torch.float32)
    args = [64, 20, 77, ops.a, ops.lda, ops.sa, ops.ldsa, ops.b, ops.lda, ops.sb, ops.ldsa, c, CODE["fp32"], 64]
    with lib.Handle() as h:
        stream = torch.cuda.Stream()
        h.set_stream(stream)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            assert h.gemm_fp4_status(*args) == lib.SGBLAS_STATUS_NOT_SUPPORTED
            c.fresh.zero_()   # a graph of something
        graph.reset()
        h.gemm_fp4(*args)
        torch.cuda.synchronize()
    assert torch.equal(c.view, ops.want().float())


def test_products_past_32_bits(cuda, handle):
    """Columns of C and rows of operands whose addresses do not fit 32 bits."""
    m, k, n, ld = 64, 64, 5, 1 << 30
    ops = Operands(m, k, [n], seed=9)
    b = torch.zeros(n * ld, dtype=torch.uint8, device="cuda")       # 5 GB
    b.view(n, ld)[:, :32] = ops.b.view
    sb = torch.zeros(n * ld, dtype=torch.uint8, device="cuda")
    sb.view(n, ld)[:, :2] = ops.sb.view
    c = torch.zeros(n * (ld // 2), device="cuda")                   # 10 GB
    handle.gemm_fp4(m, n, k, ops.a, ops.lda, ops.sa, ops.ldsa, b, ld, sb, ld, c, CODE["fp32"], ld // 2)
    assert torch.equal(c.view(n, ld // 2)[:, :m], ops.want().float())
