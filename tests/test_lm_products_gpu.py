"""The language-model products (sgblas_lm.h) on the GPU, against their
definitions in 64 bits.

Tolerances, per element, from the arithmetic: with mag the sum of the absolute
products, an FP32 chain of s tensor-core instructions is off by at most
s 2^-22 mag (its adder truncates; a truncation costs 2^-23, and one more bit
covers the alignment of the instruction's own products); adding p pieces in
FP32 adds p 2^-24 mag; BF16 output (8 significant bits, so half a unit in the
last place is up to 2^-8) adds 2^-8 of the result. The definition in 64 bits is
exact at this scale.
"""
import pytest

import sgblas_b200 as sg

pytestmark = pytest.mark.gpu

BF16, FP32 = sg.SGBLAS_TYPE_BF16, sg.SGBLAS_TYPE_FP32
OP_N, OP_T = sg.SGBLAS_OP_N, sg.SGBLAS_OP_T
SENTINEL = -12345.0


def dtype_of(torch, ctype):
    return torch.bfloat16 if ctype == BF16 else torch.float32


def chain_bound(k, ctype):
    """Error of a 16-bit product's sums over mag, by the length of the chains."""
    chain = min(k, 512) if ctype == FP32 else k
    return (chain / 16 + 2) * 2.0 ** -22 + (k / 512 + 2) * 2.0 ** -24


def close(got, want, mag, bound, bf16):
    err = (got.double() - want).abs()
    limit = bound * mag + (2.0 ** -8 * want.abs() if bf16 else 0.0) + 1e-30
    worst = (err / limit).max().item() if err.numel() else 0.0
    return worst <= 1.0, worst


def strided(torch, rows, cols, ld, type_, gen, offset=0):
    """rows x cols values in rows of `ld`, `offset` elements into a buffer full of NaN."""
    buf = torch.full((offset + rows * ld + 64,), float("nan"), device="cuda").to(type_)
    view = buf[offset:offset + rows * ld].view(rows, ld)[:, :cols]
    view.copy_(torch.randn(rows, cols, generator=gen, device="cuda"))
    return buf, view


def generator(torch, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return gen


def output(torch, count, type_):
    """`count` elements between two guard bands of the sentinel."""
    buf = torch.full((count + 512,), SENTINEL, device="cuda").to(type_)
    return buf, buf[256:256 + count]


def guards_ok(buf):
    s = buf.new_full((1,), SENTINEL)
    return bool((buf[:256] == s).all() and (buf[-256:] == s).all())


# ---- grouped along n --------------------------------------------------------------

LENGTHS = [
    [1], [0, 1, 0], [3, 0, 17, 1], [31, 33, 0, 64, 65], [0, 0, 0], [130, 5], [300, 0, 257, 12],
    [600, 513], [1, 255, 256, 257],
]


@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
@pytest.mark.parametrize("trans", [OP_T, OP_N])
@pytest.mark.parametrize("m,k,pad,ctype,alpha,beta", [
    (136, 200, 8, BF16, 1.0, 0.0),
    (1, 1, 0, FP32, 1.0, 0.0),
    (257, 1100, 0, FP32, -0.5, 2.0),
    (131, 77, 3, BF16, 2.0, 1.0),
    (384, 640, 8, BF16, 1.0, 0.0),
    (128, 64, 0, FP32, 0.0, 0.5),
])
def test_grouped_n(cuda, handle, lengths, trans, m, k, pad, ctype, alpha, beta):
    torch = cuda
    gen = generator(torch, 17 + len(lengths))
    groups, head, tail = len(lengths), 2, 3   # tokens before and after all groups
    n = head + sum(lengths) + tail
    offsets = torch.tensor([head] + [head + sum(lengths[:g + 1]) for g in range(groups)],
                           dtype=torch.int32, device="cuda")
    rows, cols = (m, k) if trans == OP_T else (k, m)   # weights as a row-major tensor
    lda, ldb, ldc = cols + pad, k + pad, m + pad
    wbuf, w = strided(torch, groups * rows, cols, lda, torch.bfloat16, gen, offset=pad)
    xbuf, x = strided(torch, n, k, ldb, torch.bfloat16, gen)
    x[:head] = float("nan")   # a token outside the groups takes part in nothing
    x[n - tail:] = float("inf")
    type_ = dtype_of(torch, ctype)
    cbuf, c = output(torch, n * ldc, type_)
    c0 = torch.randn(n, ldc, generator=gen, device="cuda").to(type_)
    if beta == 0.0:
        c0[:, :m] = float("nan")   # not read
    c.copy_(c0.reshape(-1))
    handle.grouped_gemm_n(trans, m, n, k, groups, offsets, alpha, w, lda, rows * lda, x, ldb, beta,
                          c, ctype, ldc)
    torch.cuda.synchronize()
    got = c.view(n, ldc)
    assert guards_ok(cbuf) and sg.get_device_errors() == 0
    assert torch.equal(got[:, m:], c0[:, m:]), "padding rows were written"
    inside = torch.zeros(n, dtype=torch.bool, device="cuda")
    for g in range(groups):
        lo, hi = int(offsets[g]), int(offsets[g + 1])
        inside[lo:hi] = True
        wg = w[g * rows:(g + 1) * rows].double()
        wg = wg if trans == OP_T else wg.T
        xg = x[lo:hi].double()
        want = alpha * (xg @ wg.T) + (beta * c0[lo:hi, :m].double() if beta != 0.0 else 0.0)
        mag = abs(alpha) * (xg.abs() @ wg.abs().T)
        if beta != 0.0:
            mag = mag + abs(beta) * c0[lo:hi, :m].double().abs()
        ok, worst = close(got[lo:hi, :m], want, mag, chain_bound(k, ctype), ctype == BF16)
        assert ok, (g, worst)
    assert torch.equal(got[~inside, :m].nan_to_num(7.0), c0[~inside, :m].nan_to_num(7.0)), \
        "a token outside the groups was written"


def test_a_nan_stays_with_its_token(cuda, handle):
    """NaN and infinities of one token reach that token's outputs only."""
    torch = cuda
    gen = generator(torch, 3)
    m, k, n = 200, 128, 90
    w = torch.randn(2, m, k, generator=gen, device="cuda").to(torch.bfloat16)
    x = torch.randn(n, k, generator=gen, device="cuda").to(torch.bfloat16)
    x[40, 5] = float("nan")
    x[41, 7] = float("inf")
    offsets = torch.tensor([0, 41, 90], dtype=torch.int32, device="cuda")
    y = torch.empty(n, m, dtype=torch.float32, device="cuda")
    handle.grouped_gemm_n(OP_T, m, n, k, 2, offsets, 1.0, w, k, m * k, x, k, 0.0, y, FP32, m)
    finite = torch.isfinite(y).all(dim=1)
    assert finite.sum().item() == n - 2 and not finite[40] and not finite[41]


def test_offsets_are_clamped(cuda, handle):
    """Offsets outside [0, n] count as the nearer end: nothing outside C is touched."""
    torch = cuda
    gen = generator(torch, 4)
    m, k, n = 64, 64, 50
    w = torch.randn(3, m, k, generator=gen, device="cuda").to(torch.bfloat16)
    x = torch.randn(n, k, generator=gen, device="cuda").to(torch.bfloat16)
    offsets = torch.tensor([-5, 20, 30, 5000], dtype=torch.int32, device="cuda")
    cbuf, y = output(torch, n * m, torch.float32)
    handle.grouped_gemm_n(OP_T, m, n, k, 3, offsets, 1.0, w, k, m * k, x, k, 0.0, y, FP32, m)
    torch.cuda.synchronize()
    assert guards_ok(cbuf)
    for g, (lo, hi) in enumerate(((0, 20), (20, 30), (30, 50))):
        want = x[lo:hi].double() @ w[g].double().T
        mag = x[lo:hi].double().abs() @ w[g].double().abs().T
        ok, worst = close(y.view(n, m)[lo:hi], want, mag, chain_bound(k, FP32), False)
        assert ok, worst


# ---- grouped along k --------------------------------------------------------------

@pytest.mark.parametrize("lengths", LENGTHS + [[64, 128, 1], [15, 16, 17, 63]], ids=str)
@pytest.mark.parametrize("m,n,pad,ctype,alpha,beta", [
    (136, 72, 8, FP32, 1.0, 0.0),
    (1, 1, 0, FP32, 1.0, 0.0),
    (300, 257, 1, FP32, 0.25, 1.0),
    (64, 520, 0, BF16, 1.0, 0.0),
    (333, 100, 0, BF16, -1.0, 0.5),
    (256, 256, 0, FP32, 0.0, 0.0),
])
def test_grouped_k(cuda, handle, lengths, m, n, pad, ctype, alpha, beta):
    torch = cuda
    gen = generator(torch, 29 + len(lengths))
    groups, head, tail = len(lengths), 1, 2
    k = head + sum(lengths) + tail
    offsets = torch.tensor([head] + [head + sum(lengths[:g + 1]) for g in range(groups)],
                           dtype=torch.int32, device="cuda")
    abuf, a = strided(torch, k, m, m + pad, torch.bfloat16, gen)
    bbuf, b = strided(torch, k, n, n + pad, torch.bfloat16, gen, offset=pad)
    a[:head] = b[k - tail:] = float("nan")   # outside the groups: part of no sum
    b[:head] = a[k - tail:] = float("inf")
    type_, ldc = dtype_of(torch, ctype), m + pad
    cbuf, c = output(torch, groups * n * ldc, type_)
    c0 = torch.randn(groups, n, ldc, generator=gen, device="cuda").to(type_)
    if beta == 0.0:
        c0[:, :, :m] = float("nan")
    c.copy_(c0.reshape(-1))
    handle.grouped_gemm_k(m, n, k, groups, offsets, alpha, a, m + pad, b, n + pad, beta, c, ctype,
                          ldc, n * ldc)
    torch.cuda.synchronize()
    got = c.view(groups, n, ldc)
    assert guards_ok(cbuf) and sg.get_device_errors() == 0
    assert torch.equal(got[:, :, m:], c0[:, :, m:]), "padding rows were written"
    for g in range(groups):
        lo, hi = int(offsets[g]), int(offsets[g + 1])
        ag, bg = a[lo:hi].double(), b[lo:hi].double()
        old = beta * c0[g, :, :m].double() if beta != 0.0 else torch.zeros((), device="cuda").double()
        want = alpha * (bg.T @ ag) + old
        mag = abs(alpha) * (bg.abs().T @ ag.abs()) + old.abs()
        ok, worst = close(got[g, :, :m], want.expand(n, m), mag.expand(n, m),
                          chain_bound(hi - lo, ctype), ctype == BF16)
        assert ok, (g, worst)


def test_a_neighbouring_groups_nan_is_not_part_of_a_sum(cuda, handle):
    torch = cuda
    gen = generator(torch, 5)
    m, n, k = 200, 300, 150
    a = torch.randn(k, m, generator=gen, device="cuda").to(torch.bfloat16)
    b = torch.randn(k, n, generator=gen, device="cuda").to(torch.bfloat16)
    a[67] = float("nan")   # the second group's first token, inside the first's last slice
    b[67] = float("nan")
    offsets = torch.tensor([0, 67, 150], dtype=torch.int32, device="cuda")
    c = torch.empty(2, n, m, device="cuda")
    handle.grouped_gemm_k(m, n, k, 2, offsets, 1.0, a, m, b, n, 0.0, c, FP32, m, n * m)
    assert torch.isfinite(c[0]).all() and torch.isnan(c[1]).all()


def test_gradients_are_the_forward_products_differences(cuda, handle):
    """L = sum(dY * Y) with small whole numbers, where every sum is exact: a
    step in one token's or one weight's value changes L by its gradient."""
    torch = cuda
    gen = generator(torch, 6)
    lengths, m, k = [5, 0, 70], 40, 48
    t = sum(lengths)
    whole = lambda *s: torch.randint(-3, 4, s, generator=gen, device="cuda").to(torch.bfloat16)  # noqa: E731
    x, w, dy = whole(t, k), whole(3, m, k), whole(t, m)
    offsets = torch.tensor([0, 5, 5, 75], dtype=torch.int32, device="cuda")

    def loss():
        y = torch.empty(t, m, device="cuda")
        handle.grouped_gemm_n(OP_T, m, t, k, 3, offsets, 1.0, w, k, m * k, x, k, 0.0, y, FP32, m)
        return (y.double() * dy.double()).sum().item()

    dx = torch.empty(t, k, device="cuda")
    dw = torch.empty(3, m, k, device="cuda")
    handle.grouped_gemm_n(OP_N, k, t, m, 3, offsets, 1.0, w, k, m * k, dy, m, 0.0, dx, FP32, k)
    handle.grouped_gemm_k(k, m, t, 3, offsets, 1.0, x, k, dy, m, 0.0, dw, FP32, k, m * k)
    for tensor, grad in ((x, dx), (w, dw)):
        flat, gflat = tensor.view(-1), grad.view(-1)
        for at in torch.randint(0, flat.numel(), (6,), generator=gen, device="cuda").tolist():
            old = flat[at].clone()
            flat[at] = old + 2
            up = loss()
            flat[at] = old - 2
            down = loss()
            flat[at] = old
            assert (up - down) / 4 == gflat[at].item()
    assert torch.equal(dw[1], torch.zeros_like(dw[1]))


# ---- e4m3 ---------------------------------------------------------------------------

def quantized(torch, x, block):
    """The definition, on the GPU in FP32: (q, scale) of row-major [rows, k]."""
    r, k = x.shape
    v = torch.nn.functional.pad(x.float(), (0, -k % 128, 0, -r % block))
    v = v.reshape(v.shape[0] // block, block, v.shape[1] // 128, 128)
    scale = v.abs().amax(dim=(1, 3)).clamp(min=2.0 ** -100) / torch.full((), 448.0, device="cuda")
    q = (v * (torch.ones((), device="cuda") / scale)[:, None, :, None]).to(torch.float8_e4m3fn)
    return q.reshape(v.shape[0] * block, -1)[:r, :k], scale


@pytest.mark.parametrize("rows,k,block", [
    (1, 1, 1), (5, 127, 1), (33, 128, 1), (7, 1537, 1), (130, 640, 1), (1, 129, 128), (300, 300, 128),
    (128, 256, 128), (257, 1536, 128)])
@pytest.mark.parametrize("type_", ["bfloat16", "float32"])
@pytest.mark.parametrize("pad", [0, 1, 16])
def test_quantize(cuda, handle, rows, k, block, type_, pad):
    torch = cuda
    gen = generator(torch, rows + k)
    type_ = getattr(torch, type_)
    xbuf, x = strided(torch, rows, k, k + pad, type_, gen)
    x *= torch.exp(4 * torch.randn(rows, 1, generator=gen, device="cuda")).to(type_)
    if rows > 4:
        x[2] = 0.0
        x[3, : min(k, 128)] = 1e-38   # blocks under the floor
    blocks, kb = -(-rows // block), -(-k // 128)
    qbuf = torch.full((rows * (k + pad) + 32,), 99, dtype=torch.uint8, device="cuda")
    q = qbuf[16:16 + rows * (k + pad)].view(rows, k + pad)
    sbuf, s = output(torch, blocks * (kb + 1), torch.float32)
    code = BF16 if type_ == torch.bfloat16 else FP32
    handle.quantize_fp8(k, rows, block, x, code, k + pad, q, k + pad, s, kb + 1)
    torch.cuda.synchronize()
    want_q, want_s = quantized(torch, x, block)
    got_s = s.view(blocks, kb + 1)
    assert torch.equal(got_s[:, :kb], want_s)
    assert torch.equal(q[:, :k].contiguous().view(torch.float8_e4m3fn).float(), want_q.float())
    assert guards_ok(sbuf) and (got_s[:, kb] == SENTINEL).all()
    assert (q[:, k:] == 99).all() and (qbuf[:16] == 99).all() and (qbuf[-16:] == 99).all()


def test_quantize_batch(cuda, handle):
    torch = cuda
    gen = generator(torch, 8)
    x = torch.randn(3, 200, 300, generator=gen, device="cuda")
    q = torch.empty(3, 200, 304, dtype=torch.uint8, device="cuda")
    s = torch.empty(3, 2, 3, device="cuda")
    handle.quantize_fp8(300, 200, 128, x, FP32, 300, q, 304, s, 3, batch=3, stride_x=200 * 300,
                        stride_q=200 * 304, stride_scale=6)
    for i in range(3):
        want_q, want_s = quantized(torch, x[i], 128)
        assert torch.equal(s[i], want_s)
        assert torch.equal(q[i, :, :300].contiguous().view(torch.float8_e4m3fn).float(),
                           want_q.float())


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("block", [1, 128])
def test_quantize_marks_what_is_not_finite(cuda, handle, bad, block):
    torch = cuda
    for type_, code in ((torch.bfloat16, BF16), (torch.float32, FP32)):
        x = torch.ones(4, 256, dtype=type_, device="cuda")
        x[1, 130] = bad
        q = torch.empty(4, 256, dtype=torch.uint8, device="cuda")
        s = torch.empty(4 if block == 1 else 1, 2, device="cuda")
        handle.quantize_fp8(256, 4, block, x, code, 256, q, 256, s, 2)
        v = q.view(torch.float8_e4m3fn).float()
        assert not torch.isfinite(s[1 if block == 1 else 0, 1]) and torch.isnan(v[1, 130])
        assert torch.isfinite(s[:, 0]).all() and (v[:, :128] == 448).all()


@pytest.mark.parametrize("lengths", [None, [1], [0, 1, 0], [3, 0, 17, 1], [31, 33, 0, 64, 65],
                                     [130, 100], [300, 0, 257, 12], [600, 513]], ids=str)
@pytest.mark.parametrize("m,k,pad,ctype", [
    (128, 128, 0, FP32), (257, 300, 4, FP32), (131, 1, 0, BF16), (520, 1100, 3, BF16),
    (64, 4000, 0, FP32), (384, 640, 16, BF16)])
def test_gemm_fp8(cuda, handle, lengths, m, k, pad, ctype):
    torch = cuda
    gen = generator(torch, 41)
    groups = 1 if lengths is None else len(lengths)
    n = 77 if lengths is None else sum(lengths) + 1
    kb, mb = -(-k // 128), -(-m // 128)
    lda, ldb, ldc, lds = k + pad, k + pad, m + pad, kb + pad
    w = (8 * torch.randn(groups, m, lda, generator=gen, device="cuda")).to(torch.float8_e4m3fn)
    x = (8 * torch.randn(n, ldb, generator=gen, device="cuda")).to(torch.float8_e4m3fn)
    ws = torch.exp(3 * torch.randn(groups, mb, lds, generator=gen, device="cuda"))
    xs = torch.exp(3 * torch.randn(n, lds, generator=gen, device="cuda"))
    xs[n // 2] = 0.0
    type_ = dtype_of(torch, ctype)
    cbuf, c = output(torch, n * ldc, type_)
    if lengths is None:
        offsets = [0, n]
        handle.gemm_fp8(m, n, k, w, lda, ws, lds, x, ldb, xs, lds, c, ctype, ldc)
    else:
        offsets = [0] + [sum(lengths[:g + 1]) for g in range(groups)]
        handle.grouped_gemm_fp8(m, n, k, groups,
                                torch.tensor(offsets, dtype=torch.int32, device="cuda"), w, lda,
                                m * lda, ws, lds, mb * lds, x, ldb, xs, lds, c, ctype, ldc)
    torch.cuda.synchronize()
    got = c.view(n, ldc)
    assert guards_ok(cbuf) and sg.get_device_errors() == 0
    assert (got[:, m:] == SENTINEL).all() and (got[offsets[-1]:] == SENTINEL).all()
    spread = lambda v, rows: v[..., :kb].double().repeat_interleave(128, -1)[..., :k]  # noqa: E731
    for g in range(groups):
        lo, hi = offsets[g], offsets[g + 1]
        wg = w[g, :, :k].double() * spread(ws[g], m).repeat_interleave(128, 0)[:m]
        xg = x[lo:hi, :k].double() * spread(xs[lo:hi], n)
        bound = (8 + 2) * 2.0 ** -22 + (kb + 2) * 2.0 ** -23   # a block, its scales, the blocks' sum
        ok, worst = close(got[lo:hi, :m], xg @ wg.T, xg.abs() @ wg.abs().T, bound, ctype == BF16)
        assert ok, (g, worst)


def test_gemm_fp8_with_nothing_to_add_writes_zeros(cuda, handle):
    torch = cuda
    y = torch.full((5, 64), 3.0, device="cuda")
    handle.gemm_fp8(64, 5, 0, None, 1, None, 1, None, 1, None, 1, y, FP32, 64)
    assert (y == 0).all()


# ---- orthogonalisation ------------------------------------------------------------------

ABC = (3.4445, -4.7750, 2.0315)


def newton_schulz(g, steps, abc, eps, scale):
    x = g.double()
    x = x / (x.square().sum().sqrt() + eps)
    wide = x if x.shape[0] <= x.shape[1] else x.T
    for _ in range(steps):
        a = wide @ wide.T
        wide = abc[0] * wide + (abc[1] * a + abc[2] * (a @ a)) @ wide
    return scale * (wide if x.shape[0] <= x.shape[1] else wide.T)


@pytest.mark.parametrize("rows,cols,batch", [
    (1, 1, 1), (1, 100, 2), (64, 64, 1), (63, 65, 3), (200, 333, 1), (333, 200, 2), (512, 128, 5),
    (129, 1030, 1), (700, 650, 1), (1300, 1280, 1)])
@pytest.mark.parametrize("type_,steps,scale,pad", [("float32", 5, 1.0, 0), ("bfloat16", 5, 0.2, 0),
                                                   ("float32", 1, -2.0, 3), ("bfloat16", 3, 1.0, 8)])
def test_orthogonalize(cuda, handle, rows, cols, batch, type_, steps, scale, pad):
    """Relative error in the Frobenius norm: BF16's rounding is 1.66e-3 there
    (2^-8 / sqrt(3) over the mean place in a binade), the last product's
    operands of 11 bits an eighth of that each, amplified by the polynomial's
    coefficients; 2^-9 + 2^-10 = 2.9e-3 holds both."""
    torch = cuda
    gen = generator(torch, rows)
    type_ = getattr(torch, type_)
    g = torch.full((batch, rows, cols + pad), float("nan"), device="cuda")
    rank = max(1, min(rows, cols) // 8)
    g[:, :, :cols] = 1e-3 * (torch.randn(batch, rows, rank, generator=gen, device="cuda") @
                             torch.randn(batch, rank, cols, generator=gen, device="cuda") +
                             0.3 * torch.randn(batch, rows, cols, generator=gen, device="cuda"))
    g = g.to(type_)
    obuf, o = output(torch, batch * rows * (cols + pad), torch.bfloat16)
    code = BF16 if type_ == torch.bfloat16 else FP32
    handle.orthogonalize(cols, rows, batch, steps, ABC, 1e-7, scale, g, code, cols + pad,
                         rows * (cols + pad), o, cols + pad, rows * (cols + pad))
    torch.cuda.synchronize()
    got = o.view(batch, rows, cols + pad)
    assert guards_ok(obuf) and sg.get_device_errors() == 0
    assert (got[:, :, cols:] == torch.tensor(SENTINEL).to(torch.bfloat16).item()).all()
    for i in range(batch):
        want = newton_schulz(g[i, :, :cols], steps, ABC, 1e-7, scale)
        rel = ((got[i, :, :cols].double() - want).norm() / want.norm()).item()
        assert rel <= 2.0 ** -9 + 2.0 ** -10, (i, rel)


@pytest.mark.parametrize("spectrum", ["equal", "decay", "one strong"])
@pytest.mark.parametrize("diagonal", [False, True])
@pytest.mark.parametrize("rows,cols,steps", [(64, 1024, 5), (1030, 129, 6), (1000, 200, 4),
                                             (1024, 2560, 5), (64, 96, 5)])
def test_orthogonalize_spectra(cuda, handle, rows, cols, steps, diagonal, spectrum):
    """Long matrices take two steps per Gram product; (64, 96) and the last steps
    do not. The bound: BF16's rounding, half a unit of 2^-8 at most and 2^-8 /
    sqrt(3) over a binade in the mean (1.4 times the test above for entries at a
    binade's low end, as a diagonal's few may be), and the last product's
    operands as there: 2^-8 holds them, and a lost digit of the small singular
    values does not fit in it."""
    torch = cuda
    gen = generator(torch, rows + cols)
    k = min(rows, cols)
    kinds = {"equal": torch.ones(k), "decay": torch.logspace(0, -4, k),
             "one strong": torch.cat([torch.ones(1), torch.full((k - 1,), 1e-3)])}
    values = kinds[spectrum].to("cuda", torch.float64)
    if diagonal:
        g = torch.zeros(rows, cols, device="cuda", dtype=torch.float64)
        g[range(k), range(k)] = values
    else:
        u, v = (torch.linalg.qr(torch.randn(d, k, generator=gen, device="cuda",
                                            dtype=torch.float64))[0] for d in (rows, cols))
        g = (u * values) @ v.T
    g = g.float().contiguous()
    o = torch.empty(rows, cols, device="cuda", dtype=torch.bfloat16)
    handle.orthogonalize(cols, rows, 1, steps, ABC, 1e-7, 1.0, g, FP32, cols, 0, o, cols, 0)
    want = newton_schulz(g, steps, ABC, 1e-7, 1.0)
    assert sg.get_device_errors() == 0
    assert ((o.double() - want).norm() / want.norm()).item() <= 2.0 ** -8


@pytest.mark.parametrize("abc", [(1.5, -0.5, 0.0), (4.0, -7.0, 3.3), (-2.0, 1.5, 0.0)])
def test_orthogonalize_coefficients(cuda, handle, abc):
    """4 * 4 is outside the pairs' range, so those steps go one by one. The
    bound: BF16's 2^-8, and 2^-11 of each operand of the last product by norms."""
    torch = cuda
    g = torch.randn(100, 1500, generator=generator(torch, 9), device="cuda")
    o = torch.empty(100, 1500, device="cuda", dtype=torch.bfloat16)
    handle.orthogonalize(1500, 100, 1, 3, abc, 0.0, 1.0, g, FP32, 1500, 0, o, 1500, 0)
    want, x = (newton_schulz(g, k, abc, 0.0, 1.0) for k in (3, 2))
    a = x @ x.T
    p = abc[0] * torch.eye(100, device="cuda", dtype=torch.float64) + abc[1] * a + abc[2] * a @ a
    operands = p.norm() * torch.linalg.matrix_norm(x, 2) + torch.linalg.matrix_norm(p, 2) * x.norm()
    assert sg.get_device_errors() == 0
    assert (o.double() - want).norm() <= 2.0 ** -8 * want.norm() + 2.0 ** -11 * operands


def test_orthogonalize_zero_and_nan(cuda, handle):
    torch = cuda
    g = torch.zeros(2, 100, 70, device="cuda")
    g[1, 3, 4] = float("nan")
    o = torch.full((2, 100, 70), 5.0, device="cuda").to(torch.bfloat16)
    handle.orthogonalize(70, 100, 2, 5, ABC, 1e-7, 1.0, g, FP32, 70, 7000, o, 70, 7000)
    assert (o[0] == 0).all() and torch.isnan(o[1]).all()


# ---- how they are called ------------------------------------------------------------------

def test_streams_graphs_and_repeats(cuda, lib):
    """On a stream of their own, captured and replayed, the results are the same bits."""
    torch = cuda
    gen = generator(torch, 9)
    m, k, lengths = 300, 260, [40, 0, 200, 9]
    n = sum(lengths)
    offsets = torch.tensor([0, 40, 40, 240, 249], dtype=torch.int32, device="cuda")
    w = torch.randn(4, m, k + 4, generator=gen, device="cuda").to(torch.bfloat16)
    x = torch.randn(n, k + 4, generator=gen, device="cuda").to(torch.bfloat16)
    g = torch.randn(2, 130, 96, generator=gen, device="cuda")
    y, dw, o = (torch.zeros(s, device="cuda", dtype=t) for s, t in (
        ((n, m), torch.float32), ((4, m, k + 4), torch.float32), ((2, 130, 96), torch.bfloat16)))
    dy = torch.randn(n, m, generator=gen, device="cuda").to(torch.bfloat16)
    with lib.Handle() as h:
        def run():
            h.grouped_gemm_n(OP_T, m, n, k, 4, offsets, 1.0, w, k + 4, m * (k + 4), x, k + 4, 0.0, y,
                             FP32, m)
            h.grouped_gemm_k(k, m, n, 4, offsets, 1.0, x, k + 4, dy, m, 0.0, dw, FP32, k + 4,
                             m * (k + 4))
            h.orthogonalize(96, 130, 2, 5, ABC, 1e-7, 1.0, g, FP32, 96, 130 * 96, o, 96, 130 * 96)

        run()
        torch.cuda.synchronize()
        first = [v.clone() for v in (y, dw, o)]
        stream = torch.cuda.Stream()
        h.set_stream(stream)
        for v in (y, dw, o):
            v.zero_()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            run()
        for _ in range(3):
            graph.replay()
        torch.cuda.synchronize()
        for got, want in zip((y, dw, o), first):
            assert torch.equal(got, want)
        del graph


def test_a_capture_never_allocates(cuda, lib):
    """A call that needs workspace no earlier call has made is refused inside a capture."""
    torch = cuda
    w = torch.zeros(2, 64, 65, dtype=torch.bfloat16, device="cuda")
    x = torch.zeros(8, 65, dtype=torch.bfloat16, device="cuda")
    y = torch.zeros(8, 64, device="cuda")
    offsets = torch.tensor([0, 4, 8], dtype=torch.int32, device="cuda")
    with lib.Handle() as h:
        stream = torch.cuda.Stream()
        h.set_stream(stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            y.add_(1.0)
            st = h.grouped_gemm_n_status(OP_T, 64, 8, 65, 2, offsets, 1.0, w, 65, 64 * 65, x, 65, 0.0,
                                         y, FP32, 64)
            so = h.orthogonalize_status(64, 64, 1, 5, ABC, 1e-7, 1.0, y, FP32, 64, 0, w, 64, 0)
        assert st == so == lib.SGBLAS_STATUS_NOT_SUPPORTED
        del graph


def test_offsets_past_32_bits(cuda, handle):
    """Weights and their gradients of more than 2^31 elements: the last expert's place."""
    torch = cuda
    gen = generator(torch, 10)
    groups, m, k, n = 33, 8192, 8192, 40
    w = torch.zeros(groups, m, k, dtype=torch.bfloat16, device="cuda")
    w[-1] = torch.randn(m, k, generator=gen, device="cuda")
    x = torch.randn(n, k, generator=gen, device="cuda").to(torch.bfloat16)
    dy = torch.randn(n, m, generator=gen, device="cuda").to(torch.bfloat16)
    offsets = torch.zeros(groups + 1, dtype=torch.int32, device="cuda")
    offsets[-1] = n
    y = torch.empty(n, m, device="cuda")
    handle.grouped_gemm_n(OP_T, m, n, k, groups, offsets, 1.0, w, k, m * k, x, k, 0.0, y, FP32, m)
    want = x.double() @ w[-1].double().T
    ok, worst = close(y, want, x.double().abs() @ w[-1].double().abs().T, chain_bound(k, FP32), False)
    assert ok, worst
    handle.grouped_gemm_k(k, m, n, groups, offsets, 1.0, x, k, dy, m, 0.0, w, BF16, k, m * k)
    want = dy.double().T @ x.double()
    ok, worst = close(w[-1], want, dy.double().abs().T @ x.double().abs(), chain_bound(n, BF16), True)
    assert ok, worst
    assert not w[:-1].any()


def test_unaligned_weights_of_empty_groups(cuda, handle):
    """Weights that TMA cannot read are copied for groups with tokens only: what an
    earlier call left in the others' copies (NaN here) reaches nothing. Products
    of small integers are exact."""
    torch = cuda
    groups, m, k, n = 4, 70, 77, 40
    gen = generator(torch, 12)
    w = torch.randint(-3, 4, (groups, m, k), generator=gen, device="cuda").to(torch.bfloat16)
    x = torch.randint(-3, 4, (n, k), generator=gen, device="cuda").to(torch.bfloat16)
    every = torch.tensor([0, 10, 20, 30, 40], dtype=torch.int32, device="cuda")
    y = torch.empty(n, m, device="cuda")
    handle.grouped_gemm_n(sg.SGBLAS_OP_T, m, n, k, groups, every, 1.0, torch.full_like(w, float("nan")),
                          k, m * k, x, k, 0.0, y, FP32, m)
    assert torch.isnan(y).all()
    for offsets in ([0, 0, 40, 40, 40], [0, 0, 13, 13, 40], [0, 40, 40, 40, 40], [0, 0, 0, 0, 40]):
        o = torch.tensor(offsets, dtype=torch.int32, device="cuda")
        y.fill_(float("nan"))
        handle.grouped_gemm_n(sg.SGBLAS_OP_T, m, n, k, groups, o, 1.0, w, k, m * k, x, k, 0.0, y, FP32, m)
        for g in range(groups):
            a, b = offsets[g], offsets[g + 1]
            assert torch.equal(y[a:b], x[a:b].float() @ w[g].float().T)
    assert sg.get_device_errors() == 0
