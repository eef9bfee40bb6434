"""Tokens sorted by expert and back, against plain forms. Sorting and copying are
compared for equality, weighted columns too (one product, one rounding)."""
import pytest
import torch

import sgblas_b200 as sg
from tests.layer_util import HALF, TYPES, Matrix, generator, marked

pytestmark = pytest.mark.gpu
CODE = {"bf16": sg.SGBLAS_TYPE_BF16, "fp32": sg.SGBLAS_TYPE_FP32}


def sorted_places(group, groups):
    """Python's own stable sort."""
    flat = group.flatten().tolist()
    order = sorted((i for i, g in enumerate(flat) if 0 <= g < groups), key=lambda i: flat[i])
    place = [-1] * len(flat)
    for at, i in enumerate(order):
        place[i] = at
    counts = [0] * groups
    for i in order:
        counts[flat[i]] += 1
    offsets = [0]
    for c in counts:
        offsets.append(offsets[-1] + c)
    return offsets, place


def check_sort(handle, group, groups):
    n, top = group.shape
    offsets = Matrix(1, groups + 1, torch.int32)
    place = Matrix(n, top, torch.int32)
    handle.sort_tokens(n, top, groups, group, offsets, place)
    want_offsets, want_place = sorted_places(group, groups)
    assert offsets.view[0].tolist() == want_offsets
    assert place.view.flatten().tolist() == want_place
    assert not offsets.unmarked() and not place.unmarked()
    return offsets.view[0], place.view


@pytest.mark.parametrize("n,top,groups", [
    (0, 2, 5), (3, 0, 4), (1, 1, 1), (5, 3, 7), (31, 1, 2), (32, 2, 1024), (100, 8, 64), (129, 1, 3),
    (1000, 8, 128), (777, 3, 1000), (300, 2, 255), (300, 2, 256), (700, 3, 1023), (4096, 4, 33), (16384, 8, 64), (50001, 5, 1024)])
def test_sort(cuda, handle, n, top, groups):
    gen = generator(n + top)
    group = torch.randint(-2, groups + 2, (n, top), generator=gen, device="cuda", dtype=torch.int32)
    check_sort(handle, group, groups)


def test_sort_of_one_group_none_and_extremes(cuda, handle):
    same = torch.full((3000, 2), 5, dtype=torch.int32, device="cuda")   # the same group twice for a token
    check_sort(handle, same, 6)
    check_sort(handle, same, 5)   # nobody has one
    check_sort(handle, same, 0)
    wild = torch.tensor([[2**31 - 1, -2**31], [0, 3], [4, -1]], dtype=torch.int32, device="cuda")
    check_sort(handle, wild, 4)


def moved(n, top, groups, seed, dead=0.1):
    gen = generator(seed)
    group = torch.randint(0, groups, (n, top), generator=gen, device="cuda", dtype=torch.int32)
    group[torch.rand(n, top, generator=gen, device="cuda") < dead] = -1
    _, place = sorted_places(group, groups)
    weight = torch.randn(n, top, generator=gen, device="cuda")
    return torch.tensor(place, dtype=torch.int32, device="cuda").view(n, top), weight, gen


SIZES = [(1, 1, 1), (7, 3, 2), (64, 40, 2), (127, 9, 3), (128, 5, 8), (300, 33, 5), (1000, 257, 4), (1537, 301, 3),
         (2048, 16, 4), (2048, 600, 8), (5000, 21, 7), (9001, 3, 6)]


@pytest.mark.parametrize("type_", ["bf16", "fp32"])
@pytest.mark.parametrize("k,n,top", SIZES)
@pytest.mark.parametrize("ld,shift", [(0, 0), (8, 0), (3, 1)])
def test_scatter_and_its_gradient(cuda, handle, type_, k, n, top, ld, shift):
    t = TYPES[type_]
    place, weight, gen = moved(n, top, 11, k + n)
    rows = n * top
    x = Matrix(n, k, t, k + ld, shift, torch.randn(n, k, generator=gen, device="cuda"))
    live = int((place >= 0).sum())
    for w in (None, weight):
        y = Matrix(rows, k, t, k + ld, shift)
        handle.scatter_tokens(k, n, top, rows, place, w, x, CODE[type_], x.ld, y, y.ld)
        token, choice = torch.nonzero(place >= 0, as_tuple=True)
        want = x.view[token] if w is None else (w[token, choice, None] * x.view[token].float()).to(t)
        assert torch.equal(y.view[place[token, choice].long()], want)
        assert bool((y.view[live:] == marked(t)).all())   # rows behind the last are as they were
        assert not y.unmarked() and not x.unmarked()
    # Its gradient adds a token's rows (weights NULL).
    dy = Matrix(rows, k, t, k + ld, shift, torch.randn(rows, k, generator=gen, device="cuda"))
    dy.view[live:] = float("nan")
    dx = Matrix(n, k, t, k + ld, shift)
    handle.gather_tokens(k, n, top, rows, place, None, dy, CODE[type_], dy.ld, dx, dx.ld)
    want = torch.zeros(n, k, dtype=torch.float64, device="cuda").index_add_(0, token, dy.view[place[token, choice].long()].double())
    size = torch.zeros(n, k, dtype=torch.float64, device="cuda").index_add_(0, token, dy.view[place[token, choice].long()].double().abs())
    assert bool(((dx.view.double() - want).abs() <= HALF[t] * want.abs() + top * 2.0 ** -24 * size).all())


@pytest.mark.parametrize("type_", ["bf16", "fp32"])
@pytest.mark.parametrize("k,n,top", SIZES)
@pytest.mark.parametrize("ld,shift", [(0, 0), (8, 0), (3, 1)])
def test_gather_and_its_gradients(cuda, handle, type_, k, n, top, ld, shift):
    t = TYPES[type_]
    place, weight, gen = moved(n, top, 11, k + 2 * n)
    rows = n * top
    live = int((place >= 0).sum())
    weight[place < 0] = float("nan")   # adds nothing, whatever it is
    x = Matrix(rows, k, t, k + ld, shift, torch.randn(rows, k, generator=gen, device="cuda"))
    x.view[live:] = float("nan")
    y = Matrix(n, k, t, k + ld, shift)
    handle.gather_tokens(k, n, top, rows, place, weight, x, CODE[type_], x.ld, y, y.ld)
    token, choice = torch.nonzero(place >= 0, as_tuple=True)
    at = place[token, choice].long()
    terms = weight[token, choice, None].double() * x.view[at].double()
    want = torch.zeros(n, k, dtype=torch.float64, device="cuda").index_add_(0, token, terms)
    size = torch.zeros(n, k, dtype=torch.float64, device="cuda").index_add_(0, token, terms.abs())
    assert bool(((y.view.double() - want).abs() <= HALF[t] * want.abs() + top * 2.0 ** -24 * size).all())
    assert not y.unmarked() and not x.unmarked()

    dy = Matrix(n, k, t, k + ld, shift, torch.randn(n, k, generator=gen, device="cuda"))
    dx, dw = Matrix(rows, k, t, k + ld, shift), Matrix(n, top, torch.float32)
    handle.gather_tokens_backward(k, n, top, rows, place, weight, dy, CODE[type_], dy.ld, x, x.ld, dx, dx.ld, dw)
    assert torch.equal(dx.view[at], (weight[token, choice, None] * dy.view[token].float()).to(t))
    assert bool((dx.view[live:] == marked(t)).all())
    terms = dy.view[token].double() * x.view[at].double()
    # A thread adds up to 40 * 8 values of a column of 9001, then 5 shuffles and 8 warps.
    err = (dw.view[token, choice].double() - terms.sum(dim=1)).abs()
    assert bool((err <= 340 * 2.0 ** -24 * terms.abs().sum(dim=1)).all())
    assert bool((dw.view[place < 0] == 0).all())
    assert not any(m.unmarked() for m in (dy, dx, dw, x))
    # Without the weights' gradient x is not read, and dx is the same.
    dx2 = Matrix(rows, k, t, k + ld, shift)
    handle.gather_tokens_backward(k, n, top, rows, place, weight, dy, CODE[type_], dy.ld, None, 0, dx2, dx2.ld)
    assert torch.equal(dx2.view[at], dx.view[at])
    dx3 = Matrix(rows, k, t, k + ld, shift)   # nor without weights
    handle.gather_tokens_backward(k, n, top, rows, place, None, dy, CODE[type_], dy.ld, x, x.ld, dx3, dx3.ld, dw)
    assert torch.equal(dx3.view[at], dy.view[token])


@pytest.mark.parametrize("k,ld,shift", [(1, 0, 0), (16, 0, 0), (37, 3, 1), (100, 12, 0), (4096, 0, 0)])
def test_scatter_of_bytes(cuda, handle, k, ld, shift):
    place, _, gen = moved(50, 3, 8, k)
    x = Matrix(50, k, torch.uint8, k + ld, shift, torch.randint(0, 256, (50, k), generator=gen, device="cuda"))
    y = Matrix(150, k, torch.uint8, k + ld, shift)
    handle.scatter_tokens(k, 50, 3, 150, place, None, x, sg.SGBLAS_TYPE_BYTE, x.ld, y, y.ld)
    token, choice = torch.nonzero(place >= 0, as_tuple=True)
    assert torch.equal(y.view[place[token, choice].long()], x.view[token])
    assert not y.unmarked()


def test_places_outside_are_none(cuda, handle):
    """Whatever a place holds, nothing outside the rows is read or written."""
    place = torch.tensor([[0, 3], [4, -1], [-2**31, 2**31 - 1], [1, 2]], dtype=torch.int32, device="cuda")
    x = Matrix(4, 64, torch.float32, data=torch.arange(256.0).view(4, 64).cuda())
    y = Matrix(3, 64, torch.float32)
    handle.scatter_tokens(64, 4, 2, 3, place, None, x, CODE["fp32"], 64, y, 64)
    assert torch.equal(y.view, x.view[[0, 3, 3]]) and not y.unmarked()
    back = Matrix(4, 64, torch.float32)
    handle.gather_tokens(64, 4, 2, 3, place, None, y, CODE["fp32"], 64, back, 64)
    assert torch.equal(back.view[0], x.view[0]) and torch.equal(back.view[3], 2 * x.view[3])
    assert bool((back.view[1:3] == 0).all())
    dx, dw = Matrix(3, 64, torch.float32), Matrix(4, 2, torch.float32)
    handle.gather_tokens_backward(64, 4, 2, 3, place, None, x, CODE["fp32"], 64, y, 64, dx, 64, dw)
    assert torch.equal(dx.view, y.view) and not dx.unmarked()
    assert (dw.view != 0).tolist() == [[True, False], [False, False], [False, False], [True, True]]
    # No rows, no choices: zeros.
    handle.gather_tokens(64, 4, 2, 0, place, None, None, CODE["fp32"], 64, back, 64)
    assert bool((back.view == 0).all())
    back.view.fill_(1.0)
    handle.gather_tokens(64, 4, 0, 3, None, None, y, CODE["fp32"], 64, back, 64)
    assert bool((back.view == 0).all())
    dw.view.fill_(1.0)
    handle.gather_tokens_backward(64, 4, 2, 0, place, None, None, CODE["fp32"], 64, None, 64, None, 64, dw)
    assert bool((dw.view == 0).all())
    dw.view.fill_(1.0)
    handle.gather_tokens_backward(0, 4, 2, 3, place, None, x, CODE["fp32"], 64, y, 64, dx, 64, dw)
    assert bool((dw.view == 0).all())


def test_gather_of_shared_places(cuda, handle):
    """Choices may share a place when columns are read."""
    place = torch.zeros(70, 3, dtype=torch.int32, device="cuda")
    x = Matrix(1, 200, torch.float32, data=torch.randn(1, 200, device="cuda"))
    y = Matrix(70, 200, torch.float32)
    weight = torch.tensor([0.5, 0.25, 0.25], device="cuda").expand(70, 3).contiguous()
    handle.gather_tokens(200, 70, 3, 1, place, weight, x, CODE["fp32"], 200, y, 200)
    assert torch.equal(y.view, x.view.expand(70, 200))


def test_gather_gradients_are_the_differences(cuda, handle):
    k, n, top = 37, 6, 3
    place, weight, gen = moved(n, top, 4, 1)
    rows = n * top
    x = torch.randn(rows, k, generator=gen, device="cuda")
    c = torch.randn(n, k, generator=gen, device="cuda")
    dx, dw = torch.zeros(rows, k, device="cuda"), torch.zeros(n, top, device="cuda")
    handle.gather_tokens_backward(k, n, top, rows, place, weight, c, CODE["fp32"], k, x, k, dx, k, dw)

    def loss(x, weight):   # bilinear: differences are exact but for 64-bit roundings
        total = 0.0
        for t in range(n):
            for j in range(top):
                if place[t, j] >= 0:
                    total = total + weight[t, j] * (x[place[t, j].long()] * c[t].double()).sum()
        return total

    for at, (got, base) in enumerate(((dx, x.double()), (dw, weight.double()))):
        way = torch.randn(base.shape, generator=gen, device="cuda", dtype=torch.float64)
        ends = [loss(*((base + s * way, weight.double()) if at == 0 else (x.double(), base + s * way))) for s in (0.5, -0.5)]
        mine, size = (got.double() * way).sum(), (got.double() * way).abs().sum()
        assert abs((ends[0] - ends[1] - mine).item()) <= 2.0 ** -18 * size.item()


def test_tokens_in_a_graph_and_on_streams(cuda, lib):
    """A captured step takes new experts on each replay, without the host."""
    n, top, groups, k = 300, 2, 16, 512
    rows = n * top
    gen = generator(12)
    group = torch.empty(n, top, dtype=torch.int32, device="cuda")
    x = torch.randn(n, k, generator=gen, device="cuda")
    weight = torch.rand(n, top, generator=gen, device="cuda")
    offsets = torch.empty(groups + 1, dtype=torch.int32, device="cuda")
    place = torch.empty(n, top, dtype=torch.int32, device="cuda")
    y, back = torch.zeros(rows, k, device="cuda"), torch.empty(n, k, device="cuda")
    stream = torch.cuda.Stream()
    with lib.Handle() as h:
        h.set_stream(stream)
        group.fill_(3)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            h.sort_tokens(n, top, groups, group, offsets, place)
            h.scatter_tokens(k, n, top, rows, place, None, x, CODE["fp32"], k, y, k)
            h.gather_tokens(k, n, top, rows, place, weight, y, CODE["fp32"], k, back, k)
        for seed in range(3):
            group.copy_(torch.randint(0, groups, (n, top), generator=gen, device="cuda", dtype=torch.int32))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            want_offsets, want_place = sorted_places(group, groups)
            assert offsets.tolist() == want_offsets and place.flatten().tolist() == want_place
            want = x.double() * weight.double().sum(dim=1, keepdim=True)
            assert bool(((back.double() - want).abs() <= 4 * 2.0 ** -24 * want.abs()).all())
        graph.reset()


def test_tokens_past_32_bits(cuda, handle):
    """Places whose addresses do not fit 32 bits."""
    k, ld, rows = 48, 1 << 23, 300
    y = torch.zeros(rows * ld, dtype=torch.bfloat16, device="cuda")   # 5 GB
    place = torch.tensor([[299], [0], [257], [256]], dtype=torch.int32, device="cuda")
    x = torch.randn(4, k, device="cuda").to(torch.bfloat16)
    handle.scatter_tokens(k, 4, 1, rows, place, None, x, CODE["bf16"], k, y, ld)
    assert torch.equal(y.view(rows, ld)[[299, 0, 257, 256], :k], x)
    back = torch.empty(4, k, dtype=torch.bfloat16, device="cuda")
    handle.gather_tokens(k, 4, 1, rows, place, None, y, CODE["bf16"], ld, back, k)
    assert torch.equal(back, x)
    dx, dw = torch.zeros(rows, k, dtype=torch.bfloat16, device="cuda"), torch.empty(4, 1, device="cuda")
    handle.gather_tokens_backward(k, 4, 1, rows, place, None, x, CODE["bf16"], k, y, ld, dx, k, dw)
    assert torch.equal(dx[[299, 0, 257, 256]], x)
    y.zero_()
    handle.gather_tokens_backward(k, 4, 1, rows, place, None, x, CODE["bf16"], k, None, k, y, ld)
    assert torch.equal(y.view(rows, ld)[[299, 0, 257, 256], :k], x)
    want = x.double().square().sum(dim=1)
    assert bool(((dw[:, 0].double() - want).abs() <= 40 * 2.0 ** -24 * want).all())
