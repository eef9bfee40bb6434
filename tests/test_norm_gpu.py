"""sgblasRmsNorm and sgblasRmsNormBackward against their definitions in 64 bits.

Tolerances. h is equal (the same two roundings). s = (mean h^2 + eps)^-1/2: a
thread adds its values one after another, at most 160 here, then 5 shuffles, 16
warps: 200 roundings of a sum of positive terms at most, half of that in the
root, and six more roundings (the reciprocal root's is two steps): 2^-24 * 106 < 2^-17.
v adds two. So y is within half a step plus 2^-16 of v, relative; the sums of the
backward pass alike, relative to the sums of their terms' magnitudes (dw: a CTA's
columns one after another, 17 here, 32 warps of 19 rows, 32 sums: 2^-24 * 180 < 2^-16).
"""
import ctypes
import math

import pytest
import torch

import sgblas_b200 as sg
from tests.layer_util import HALF, TYPES, Matrix, generator

pytestmark = pytest.mark.gpu
CODE = {"bf16": sg.SGBLAS_TYPE_BF16, "fp32": sg.SGBLAS_TYPE_FP32}
EPS = 1e-6
SUMS = 2.0 ** -16

# k, n: a value, less than a vector, around a block, odd, every number of vectors per
# thread, longer than a CTA's registers hold; few columns, and so many that CTAs walk them.
SIZES = [(1, 1), (1, 700), (7, 5), (8, 1), (8, 2500), (127, 3), (128, 2), (129, 600), (256, 900), (333, 31), (520, 700),
         (1000, 400), (1000, 800), (1537, 333), (1537, 1300), (2048, 1), (2056, 299), (2056, 1500), (4096, 1),
         (4096, 320), (4096, 800), (4100, 7), (8192, 310), (8192, 650), (9001, 300), (10240, 600), (16384, 2),
         (16384, 600), (16392, 3), (20011, 2)]


# So many columns of whole vectors that each CTA's ring goes round more than twice, the
# last set of columns in part (test_layer_dispatch.py). The gradients of the weights are
# then sums of up to 40 columns in turn, 8 of a CTA, 19 rows of a warp, 32 warps, and s is
# off as above: 2^-24 * (99 + 106) < 2^-16.
RINGS = [(64, 100003), (504, 20001), (1000, 20001), (4096, 7001), (5120, 2001), (8200, 1501), (10240, 1501)]


def inputs(k, n, type_, ld=0, shift=0, seed=0, scale=1.0):
    gen = generator(seed)
    make = lambda f: Matrix(n, k, TYPES[type_], k + ld, shift, (f * torch.randn(n, k, generator=gen, device="cuda")))  # noqa: E731
    x, r, dy, ds = make(scale), make(4 * scale), make(0.01), make(0.02)
    w = Matrix(1, k, TYPES[type_], k, shift, 1 + 0.3 * torch.randn(1, k, generator=gen, device="cuda"))
    return x, r, dy, ds, w


def definition(h, w, eps=EPS):
    h = h.double()
    s = (h.square().mean(dim=1, keepdim=True) + eps).rsqrt()
    return s, h * s * (1.0 if w is None else w.double())


def check_y(y, v):
    err = (y.double() - v).abs()
    assert bool((err <= (HALF[y.dtype] + SUMS) * v.abs()).all())


def check_q(q, scale, v):
    n, k = v.shape
    for b in range(0, k, 128):
        part, s = v[:, b:b + 128], scale[:, b // 128].double()
        want = part.abs().amax(dim=1).clamp(min=2.0 ** -100) / 448
        assert bool(((s - want).abs() <= (SUMS + 2.0 ** -24) * want).all())
        ideal = part / s[:, None]
        got = q[:, b:b + 128].view(torch.float8_e4m3fn).double()
        # Half a step of e4m3 (of its subnormals 2^-10), and the errors of v and of the product.
        assert bool(((got - ideal).abs() <= (2.0 ** -4 + 2 * SUMS) * ideal.abs() + 2.0 ** -10).all())


@pytest.mark.parametrize("type_", ["bf16", "fp32"])
@pytest.mark.parametrize("k,n", SIZES)
@pytest.mark.parametrize("ld,shift", [(0, 0), (8, 0), (3, 1)])
def test_norm(cuda, handle, type_, k, n, ld, shift):
    x, r, _, _, w = inputs(k, n, type_, ld, shift, seed=k + n)
    t = TYPES[type_]
    blocks = -(-k // 128)
    h, y = Matrix(n, k, t, k + ld, shift), Matrix(n, k, t, k + ld, shift)
    ldq = k + ld if shift else -(-k // 16) * 16
    q, scale = Matrix(n, k, torch.uint8, ldq, shift), Matrix(n, blocks, torch.float32, blocks + ld)
    handle.rms_norm(k, n, CODE[type_], x, x.ld, r, r.ld, w, EPS, h, h.ld, y, y.ld, q, q.ld, scale, scale.ld)
    want_h = (x.view.float() + r.view.float()).to(t)
    assert torch.equal(h.view, want_h)
    _, v = definition(want_h, w.view)
    check_y(y.view, v)
    check_q(q.view, scale.view, v)
    assert not any(m.unmarked() for m in (x, r, w, h, y, q, scale))
    # Each output alone, without residual and weight, is the same kernel's.
    y2, q2, scale2 = Matrix(n, k, t, k + ld, shift), Matrix(n, k, torch.uint8, ldq, shift), Matrix(n, blocks, torch.float32)
    handle.rms_norm(k, n, CODE[type_], h, h.ld, None, 0, w, EPS, y=y2, ldy=y2.ld)
    handle.rms_norm(k, n, CODE[type_], h, h.ld, None, 0, w, EPS, q=q2, ldq=q2.ld, scale=scale2, ldscale=blocks)
    assert torch.equal(y2.view, y.view) and torch.equal(q2.view, q.view) and torch.equal(scale2.view, scale.view)
    handle.rms_norm(k, n, CODE[type_], h, h.ld, None, 0, None, EPS, y=y2, ldy=y2.ld)
    check_y(y2.view, definition(want_h, None)[1])


@pytest.mark.parametrize("type_", ["bf16", "fp32"])
@pytest.mark.parametrize("k,n", SIZES)
@pytest.mark.parametrize("ld,shift", [(0, 0), (8, 0), (3, 1)])
@pytest.mark.parametrize("past,weighted", [(True, True), (False, False)])
def test_norm_backward(cuda, handle, type_, k, n, ld, shift, past, weighted):
    x, _, dy, ds, w = inputs(k, n, type_, ld, shift, seed=2 * k + n)
    t = TYPES[type_]
    before = torch.randn(k, generator=generator(5), device="cuda")
    for beta in (0.0, 0.5):
        dx = Matrix(n, k, t, k + ld, shift)
        dw = Matrix(1, k, torch.float32, k, shift, before)
        handle.rms_norm_backward(k, n, CODE[type_], dy, dy.ld, x, x.ld, w if weighted else None, EPS,
                                 ds if past else None, ds.ld, dx, dx.ld, beta, dw)
        h, d = x.view.double(), dy.view.double()
        s, _ = definition(h, None)
        g = d * w.view.double() if weighted else d
        along = (h * g).mean(dim=1, keepdim=True)
        want = s * (g - h * s * s * along)
        size = s * (g.abs() + h.abs() * s * s * (h * g).abs().mean(dim=1, keepdim=True))
        if past:
            want, size = want + ds.view.double(), size + ds.view.double().abs()
        assert bool(((dx.view.double() - want).abs() <= HALF[t] * want.abs() + SUMS * size).all())
        terms = d * h * s
        want_w = terms.sum(dim=0) + beta * before.double()
        size_w = terms.abs().sum(dim=0) + beta * before.double().abs()
        assert bool(((dw.view[0].double() - want_w).abs() <= SUMS * size_w).all())
        assert not any(m.unmarked() for m in (x, dy, ds, w, dx, dw))


@pytest.mark.parametrize("k,n", [(5, 3), (300, 4), (9000, 2)])
def test_norm_gradients_are_the_differences(cuda, handle, k, n):
    """The gradients of sum(y c) by differences of the definition in 64 bits."""
    x, _, c, _, w = inputs(k, n, "fp32", seed=11)
    dx, dw = Matrix(n, k, torch.float32), Matrix(1, k, torch.float32)
    handle.rms_norm_backward(k, n, CODE["fp32"], c, k, x, k, w, EPS, None, k, dx, k, 0.0, dw)

    def loss(h, weight):
        return (definition(h, weight)[1] * c.view.double()).sum()

    gen = generator(3)
    for got, at in ((dx, 0), (dw, 1)):
        base = [x.view.double(), w.view.double()]
        way = torch.randn(base[at].shape, generator=gen, device="cuda", dtype=torch.float64)
        step = 1e-5
        ends = []
        for sign in (1, -1):
            moved = list(base)
            moved[at] = base[at] + sign * step * way
            ends.append(loss(*moved))
        slope = (ends[0] - ends[1]) / (2 * step)
        mine = (got.view.double() * way).sum()
        size = (got.view.double() * way).abs().sum()
        # Third differences: step^2 / 6 of derivatives of size 10 at most (s is near 1).
        assert abs((mine - slope).item()) <= (SUMS + 1e-8) * size.item() + 1e-9


def test_norm_in_place(cuda, handle):
    for k, n in ((1537, 40), (4096, 400), (20011, 2)):
        x, r, dy, ds, w = inputs(k, n, "bf16", seed=4)
        want_h, y = Matrix(n, k, torch.bfloat16), Matrix(n, k, torch.bfloat16)
        handle.rms_norm(k, n, CODE["bf16"], x, k, r, k, w, EPS, want_h, k, y, k)
        for place in (0, 1):
            ops = [Matrix(n, k, torch.bfloat16, data=x.view), Matrix(n, k, torch.bfloat16, data=r.view)]
            y2 = Matrix(n, k, torch.bfloat16)
            handle.rms_norm(k, n, CODE["bf16"], ops[0], k, ops[1], k, w, EPS, ops[place], k, y2, k)
            assert torch.equal(ops[place].view, want_h.view) and torch.equal(y2.view, y.view)
            assert torch.equal(ops[1 - place].view, (r if place == 0 else x).view)
        dx, dw, dw2 = Matrix(n, k, torch.bfloat16), Matrix(1, k, torch.float32), Matrix(1, k, torch.float32)
        handle.rms_norm_backward(k, n, CODE["bf16"], dy, k, x, k, w, EPS, ds, k, dx, k, 0.0, dw)
        for place in (0, 1):
            ops = [Matrix(n, k, torch.bfloat16, data=dy.view), Matrix(n, k, torch.bfloat16, data=ds.view)]
            handle.rms_norm_backward(k, n, CODE["bf16"], ops[0], k, x, k, w, EPS, ops[1], k, ops[place], k, 0.0, dw2)
            assert torch.equal(ops[place].view, dx.view) and torch.equal(dw2.view, dw.view)


@pytest.mark.parametrize("type_", ["bf16", "fp32"])
@pytest.mark.parametrize("k,n", RINGS)
def test_norm_of_many_columns(cuda, handle, type_, k, n):
    x, r, _, _, w = inputs(k, n, type_, seed=k)
    t, blocks = TYPES[type_], -(-k // 128)
    h, y = Matrix(n, k, t), Matrix(n, k, t)
    q, scale = Matrix(n, k, torch.uint8), Matrix(n, blocks, torch.float32)
    handle.rms_norm(k, n, CODE[type_], x, k, r, k, w, EPS, h, k, y, k, q, k, scale, blocks)
    want_h = (x.view.float() + r.view.float()).to(t)
    assert torch.equal(h.view, want_h)
    v = definition(want_h, w.view)[1]
    check_y(y.view, v)
    check_q(q.view, scale.view, v)
    assert not any(m.unmarked() for m in (x, r, w, h, y, q, scale))
    y2 = Matrix(n, k, t)
    handle.rms_norm(k, n, CODE[type_], h, k, None, 0, w, EPS, y=y2, ldy=k)   # one operand in the ring
    assert torch.equal(y2.view, y.view)
    for place in (0, 1):   # in place: columns ahead are on their way meanwhile
        ops = [Matrix(n, k, t, data=x.view), Matrix(n, k, t, data=r.view)]
        y2 = Matrix(n, k, t)
        handle.rms_norm(k, n, CODE[type_], ops[0], k, ops[1], k, w, EPS, ops[place], k, y2, k)
        assert torch.equal(ops[place].view, want_h) and torch.equal(y2.view, y.view)
        assert torch.equal(ops[1 - place].view, (r if place == 0 else x).view)


@pytest.mark.parametrize("type_", ["bf16", "fp32"])
@pytest.mark.parametrize("k,n", RINGS)
def test_norm_gradients_of_many_columns(cuda, handle, type_, k, n):
    x, _, dy, ds, w = inputs(k, n, type_, seed=k + 1)
    t = TYPES[type_]
    h, d = x.view.double(), dy.view.double()
    s, _ = definition(x.view, None)
    g = d * w.view.double()
    want = s * (g - h * s * s * (h * g).mean(dim=1, keepdim=True))
    size = s * (g.abs() + h.abs() * s * s * (h * g).abs().mean(dim=1, keepdim=True))
    terms = d * h * s
    want_w, size_w = terms.sum(dim=0), terms.abs().sum(dim=0)
    for past in (False, True):
        dx, dw = Matrix(n, k, t), Matrix(1, k, torch.float32)
        handle.rms_norm_backward(k, n, CODE[type_], dy, k, x, k, w, EPS, ds if past else None, k, dx, k, 0.0, dw)
        if past:
            want, size = want + ds.view.double(), size + ds.view.double().abs()
        assert bool(((dx.view.double() - want).abs() <= HALF[t] * want.abs() + SUMS * size).all())
        assert bool(((dw.view[0].double() - want_w).abs() <= SUMS * size_w).all())
        assert not any(m.unmarked() for m in (x, dy, ds, w, dx, dw))
    for place in (0, 1):
        ops = [Matrix(n, k, t, data=dy.view), Matrix(n, k, t, data=ds.view)]
        dw2 = Matrix(1, k, torch.float32)
        handle.rms_norm_backward(k, n, CODE[type_], ops[0], k, x, k, w, EPS, ops[1], k, ops[place], k, 0.0, dw2)
        assert torch.equal(ops[place].view, dx.view) and torch.equal(dw2.view, dw.view)


def test_norm_special_values(cuda, handle):
    """Zeros, NaN, infinities: a column's values are its own."""
    k, n = 300, 6
    for type_ in ("bf16", "fp32"):
        x, _, _, _, w = inputs(k, n, type_, seed=9)
        x.view[1] = 0.0
        x.view[2, 299] = float("nan")
        x.view[3, 0] = float("inf")
        x.view[4] *= 1e-30
        y, q, scale = Matrix(n, k, TYPES[type_]), Matrix(n, k, torch.uint8), Matrix(n, 3, torch.float32)
        handle.rms_norm(k, n, CODE[type_], x, k, None, 0, w, EPS, None, 0, y, k, q, k, scale, 3)
        assert bool((y.view[1] == 0).all()) and bool((q.view[1].view(torch.float8_e4m3fn).float() == 0).all())
        assert bool(y.view[2].isnan().all()) and bool(scale.view[2].isnan().all())
        assert bool(y.view[3, 0].isnan()) and bool((y.view[3, 1:] == 0).all())
        rows = [0, 4, 5]
        v = definition(x.view, w.view)[1]
        check_y(y.view[rows], v[rows])
        # No eps: a column of zeros is 0 / 0.
        handle.rms_norm(k, n, CODE[type_], x, k, None, 0, w, 0.0, None, 0, y, k)
        assert bool(y.view[1].isnan().all())
        check_y(y.view[[0, 5]], definition(x.view, w.view, 0.0)[1][[0, 5]])


@pytest.mark.parametrize("type_", ["bf16", "fp32"])
@pytest.mark.parametrize("k,n", [(1, 3), (300, 4), (4096, 2), (4096, 800), (20011, 2)])
def test_norm_to_the_ends_of_its_range(cuda, handle, type_, k, n):
    """Sums of h^2 up to 2^128 (the values are +-1.75 * 2^e) and means from 2^-126 on."""
    high = math.floor((127.9 - math.log2(1.75 ** 2 * k)) / 2)
    _, _, dy, _, w = inputs(k, n, type_, seed=k)
    sign = 1 - 2 * torch.randint(0, 2, (n, k), generator=generator(k), device="cuda").float()
    blocks = -(-k // 128)
    for size, eps in ((1.75 * 2.0 ** high, EPS), (2.0 ** -63, 0.0)):
        x = Matrix(n, k, TYPES[type_], data=size * sign)
        y, q, scale = Matrix(n, k, TYPES[type_]), Matrix(n, k, torch.uint8), Matrix(n, blocks, torch.float32)
        handle.rms_norm(k, n, CODE[type_], x, k, None, 0, w, eps, None, 0, y, k, q, k, scale, blocks)
        s, v = definition(x.view, w.view, eps)
        check_y(y.view, v)
        check_q(q.view, scale.view, v)
        dx, dw = Matrix(n, k, TYPES[type_]), Matrix(1, k, torch.float32)
        handle.rms_norm_backward(k, n, CODE[type_], dy, k, x, k, w, eps, None, k, dx, k, 0.0, dw)
        h, d = x.view.double(), dy.view.double()
        g = d * w.view.double()
        want = s * (g - h * s * s * (h * g).mean(dim=1, keepdim=True))
        sizes = s * (g.abs() + h.abs() * s * s * (h * g).abs().mean(dim=1, keepdim=True))
        # Past 2^126 s^2 is subnormal: 2^-22 more.
        assert bool(((dx.view.double() - want).abs() <= HALF[TYPES[type_]] * want.abs() + (SUMS + 2.0 ** -22) * sizes).all())
        terms = d * h * s
        assert bool(((dw.view[0].double() - terms.sum(dim=0)).abs() <= SUMS * terms.abs().sum(dim=0)).all())
    x = Matrix(n, k, TYPES[type_], data=1.75 * 2.0 ** (high + 2) * sign)   # sums past 2^129
    handle.rms_norm(k, n, CODE[type_], x, k, None, 0, w, EPS, None, 0, y, k)
    assert bool((y.view == 0).all())


def test_norm_backward_without_columns(cuda, handle):
    dw = torch.randn(50, device="cuda")
    want = 0.25 * dw
    handle.rms_norm_backward(50, 0, CODE["bf16"], None, 50, None, 50, None, EPS, None, 50, None, 50, 0.25, dw)
    assert torch.equal(dw, want)
    dw.fill_(float("nan"))
    handle.rms_norm_backward(50, 0, CODE["bf16"], None, 50, None, 50, None, EPS, None, 50, None, 50, 0.0, dw)
    assert bool((dw == 0).all())


def test_norm_without_weight_gradient(cuda, handle):
    x, _, dy, ds, w = inputs(1000, 500, "bf16", seed=6)
    dx, dx2, dw = Matrix(500, 1000, torch.bfloat16), Matrix(500, 1000, torch.bfloat16), Matrix(1, 1000, torch.float32)
    handle.rms_norm_backward(1000, 500, CODE["bf16"], dy, 1000, x, 1000, w, EPS, ds, 1000, dx, 1000, 0.0, dw)
    handle.rms_norm_backward(1000, 500, CODE["bf16"], dy, 1000, x, 1000, w, EPS, ds, 1000, dx2, 1000)
    assert torch.equal(dx.view, dx2.view)


def test_norm_on_streams_and_in_graphs(cuda, handle):
    k, n = 2048, 700
    x, r, dy, ds, w = inputs(k, n, "bf16", seed=8)
    out = [Matrix(n, k, torch.bfloat16) for _ in range(3)]
    dw = Matrix(1, k, torch.float32)

    def step(h):
        h.rms_norm(k, n, CODE["bf16"], x, k, r, k, w, EPS, out[0], k, out[1], k)
        h.rms_norm_backward(k, n, CODE["bf16"], out[1], k, out[0], k, w, EPS, ds, k, out[2], k, 0.0, dw)

    step(handle)
    torch.cuda.synchronize()
    want = [m.view.clone() for m in out] + [dw.view.clone()]
    stream = torch.cuda.Stream()
    handle.set_stream(stream)
    with torch.cuda.stream(stream):
        for m in out + [dw]:
            m.view.zero_()
        step(handle)
    stream.synchronize()
    assert all(torch.equal(a, m.view) for a, m in zip(want, out + [dw]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step(handle)
    x.view.mul_(-2.0)
    graph.replay()
    torch.cuda.synchronize()
    replayed = [m.view.clone() for m in out] + [dw.view.clone()]
    handle.set_stream(None)
    step(handle)
    torch.cuda.synchronize()
    assert all(torch.equal(a, m.view) for a, m in zip(replayed, out + [dw]))
    assert not torch.equal(replayed[0], want[0])
    graph.reset()


def test_weight_gradient_in_a_capture_needs_its_workspace(cuda, lib):
    x, _, dy, _, w = inputs(256, 16, "bf16", seed=1)
    dx, dw = Matrix(16, 256, torch.bfloat16), Matrix(1, 256, torch.float32)
    args = [256, 16, CODE["bf16"], dy, 256, x, 256, w, EPS, None, 256, dx, 256]
    with lib.Handle() as h:
        stream = torch.cuda.Stream()
        h.set_stream(stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            assert h.rms_norm_backward_status(*args, 0.0, dw) == lib.SGBLAS_STATUS_NOT_SUPPORTED
            assert h.rms_norm_backward_status(*args) == lib.SGBLAS_STATUS_SUCCESS
        graph.replay()
        torch.cuda.synchronize()
        graph.reset()
    assert not torch.equal(dx.view, Matrix(16, 256, torch.bfloat16).view)


def test_norm_past_32_bits(cuda, handle):
    """Columns whose places do not fit 32 bits."""
    k, n, ld = 40, 9, 1 << 28
    gen = generator(2)
    x = torch.empty(n * ld, dtype=torch.bfloat16, device="cuda")   # 4.8 GB
    rows = torch.randn(n, k, generator=gen, device="cuda").to(torch.bfloat16)
    x.view(n, ld)[:, :k] = rows
    y, want = Matrix(n, k, torch.bfloat16), Matrix(n, k, torch.bfloat16)
    handle.rms_norm(k, n, CODE["bf16"], x, ld, None, 0, None, EPS, x, ld, y, k)
    handle.rms_norm(k, n, CODE["bf16"], rows, k, None, 0, None, EPS, None, 0, want, k)
    assert torch.equal(y.view, want.view) and torch.equal(x.view(n, ld)[:, :k], rows)
    handle.rms_norm_backward(k, n, CODE["bf16"], rows, k, x, ld, None, EPS, None, 0 + k, x, ld)
    handle.rms_norm_backward(k, n, CODE["bf16"], rows, k, rows, k, None, EPS, None, k, want, k)
    assert torch.equal(x.view(n, ld)[:, :k], want.view)


@pytest.mark.parametrize("polls", [1, 100, 5000])
def test_a_warp_that_gave_up_in_part_copies_nothing(cuda, lib, polls):
    """A ring is filled by a warp whose lanes wait for themselves: after a wait that ran out
    for some of them, none fills it (and none waits for the others)."""
    gave_up = ctypes.c_int(-1)
    assert lib.get_device_errors(clear=True) == 0
    assert lib.lib.sgblasSelfTestWaitTimeout(polls, ctypes.byref(gave_up)) == 0
    assert gave_up.value == 1
    assert lib.get_device_errors(clear=True) & 1
