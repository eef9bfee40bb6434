"""The operators together, as a layer is trained and served: norm and residual, tokens
to their experts, grouped products, and back; against torch's gradients in 64 bits."""
import importlib.util
import pathlib

import pytest
import torch

import sgblas_b200 as sg
from tests.layer_util import generator

pytestmark = pytest.mark.gpu
BF16, FP32, BYTE = sg.SGBLAS_TYPE_BF16, sg.SGBLAS_TYPE_FP32, sg.SGBLAS_TYPE_BYTE
EPS = 1e-6


def made(n, k, hidden, experts, seed):
    gen = generator(seed)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    x, r = rand(n, k).to(torch.bfloat16), (2 * rand(n, k)).to(torch.bfloat16)
    w = (1 + 0.2 * rand(k)).to(torch.bfloat16)
    w1, w2 = (rand(experts, hidden, k) / k ** 0.5).to(torch.bfloat16), (rand(experts, k, hidden) / hidden ** 0.5).to(torch.bfloat16)
    group = torch.rand(n, experts, generator=gen, device="cuda").argsort(dim=1)[:, :2].to(torch.int32).contiguous()
    group[n - n // 8:] = -1   # padding
    gate = torch.softmax(rand(n, 2), dim=1)
    return x, r, w, w1, w2, group, gate, (0.1 * rand(n, k)).to(torch.bfloat16)


class Layer:
    """out = sum over a token's experts of gate * W2 relu(W1 norm(x + r)), and its gradients."""

    def __init__(self, h, x, r, w, w1, w2, group, gate):
        self.h, self.r, self.w, self.w1, self.w2, self.group, self.gate = h, r, w, w1, w2, group, gate
        self.n, self.k = x.shape
        self.experts, self.hidden = w1.shape[:2]
        self.top, self.rows = group.shape[1], group.numel()
        new = lambda *s, t=torch.bfloat16: torch.zeros(s, dtype=t, device="cuda")  # noqa: E731
        self.new, self.x = new, x
        self.sum, self.y = new(self.n, self.k), new(self.n, self.k)
        self.offsets, self.place = new(self.experts + 1, t=torch.int32), new(self.n, self.top, t=torch.int32)
        self.xs, self.a, self.b = new(self.rows, self.k), new(self.rows, self.hidden), new(self.rows, self.k)
        self.out = new(self.n, self.k)
        self.relu = new(self.rows, self.hidden)
        # Gradients.
        self.db, self.dact, self.dxs = new(self.rows, self.k), new(self.rows, self.hidden), new(self.rows, self.k)
        self.dgate, self.dy, self.dx = new(self.n, self.top, t=torch.float32), new(self.n, self.k), new(self.n, self.k)
        self.dw1, self.dw2 = new(*w1.shape, t=torch.float32), new(*w2.shape, t=torch.float32)
        self.dw = new(self.k, t=torch.float32)

    def forward(self):
        h, k, f = self.h, self.k, self.hidden
        h.rms_norm(k, self.n, BF16, self.x, k, self.r, k, self.w, EPS, self.sum, k, self.y, k)
        h.sort_tokens(self.n, self.top, self.experts, self.group, self.offsets, self.place)
        h.scatter_tokens(k, self.n, self.top, self.rows, self.place, None, self.y, BF16, k, self.xs, k)
        h.grouped_gemm_n(sg.SGBLAS_OP_T, f, self.rows, k, self.experts, self.offsets, 1.0, self.w1, k, f * k, self.xs, k,
                         0.0, self.a, BF16, f)
        torch.clamp(self.a, min=0, out=self.relu)
        h.grouped_gemm_n(sg.SGBLAS_OP_T, k, self.rows, f, self.experts, self.offsets, 1.0, self.w2, f, f * k, self.relu, f,
                         0.0, self.b, BF16, k)
        h.gather_tokens(k, self.n, self.top, self.rows, self.place, self.gate, self.b, BF16, k, self.out, k)

    def backward(self, dout):
        h, k, f = self.h, self.k, self.hidden
        h.gather_tokens_backward(k, self.n, self.top, self.rows, self.place, self.gate, dout, BF16, k, self.b, k, self.db,
                                 k, self.dgate)
        h.grouped_gemm_k(f, k, self.rows, self.experts, self.offsets, 1.0, self.relu, f, self.db, k, 0.0, self.dw2, FP32, f, f * k)
        h.grouped_gemm_n(sg.SGBLAS_OP_N, f, self.rows, k, self.experts, self.offsets, 1.0, self.w2, f, f * k, self.db, k,
                         0.0, self.dact, BF16, f)
        self.dact.mul_(self.relu > 0)
        h.grouped_gemm_k(k, f, self.rows, self.experts, self.offsets, 1.0, self.xs, k, self.dact, f, 0.0, self.dw1, FP32, k, f * k)
        h.grouped_gemm_n(sg.SGBLAS_OP_N, k, self.rows, f, self.experts, self.offsets, 1.0, self.w1, k, f * k, self.dact, f,
                         0.0, self.dxs, BF16, k)
        h.gather_tokens(k, self.n, self.top, self.rows, self.place, None, self.dxs, BF16, k, self.dy, k)
        # The residual goes on to the layer's output, so its gradient joins.
        h.rms_norm_backward(k, self.n, BF16, self.dy, k, self.sum, k, self.w, EPS, dout, k, self.dx, k, 0.0, self.dw)


def reference(x, r, w, w1, w2, group, gate, dout, layer):
    """The same in 64 bits, with h held in BF16 and the layer's own signs of the relu's
    inputs (one that turns within its error of zero would change a gradient by all of
    itself: 2^-10 of them, 2^-5 in norm); its gradients by torch."""
    sign = (layer.relu > 0).double()
    h = (x.float() + r.float()).to(torch.bfloat16).double().requires_grad_()
    p = [v.double().requires_grad_() for v in (w, w1, w2, gate)]
    y = h * (h.square().mean(dim=1, keepdim=True) + EPS).rsqrt() * p[0]
    out = torch.zeros_like(h)
    for e in range(w1.shape[0]):
        token, choice = torch.nonzero(group == e, as_tuple=True)
        part = ((y[token] @ p[1][e].mT) * sign[layer.place[token, choice].long()]) @ p[2][e].mT
        out = out.index_add(0, token, p[3][token, choice, None] * part)
    (out + h).backward(dout.double())
    return [out.detach(), h.grad] + [v.grad for v in p]


@pytest.mark.parametrize("n,k,hidden,experts", [(9, 64, 96, 3), (300, 256, 320, 5), (1000, 520, 264, 7), (64, 130, 70, 4)])
def test_a_trained_layer(cuda, handle, n, k, hidden, experts):
    """Every BF16 value on the way is off by 2^-8 at most, and its errors pass through
    products of random weights like its values: at most one such step for each rounding
    between the inputs and a result, in norm (up to eight)."""
    made_ = made(n, k, hidden, experts, n)
    dout = made_[-1]
    layer = Layer(handle, *made_[:-1])
    layer.forward()
    layer.backward(dout)
    want = reference(*made_, layer)
    got = [layer.out, layer.dx, layer.dw, layer.dw1, layer.dw2, layer.dgate]
    roundings = [4, 8, 8, 7, 5, 5]
    for name, g, v, steps in zip(("out", "dx", "dw", "dw1", "dw2", "dgate"), got, want, roundings):
        assert ((g.double() - v).norm() / v.norm()).item() <= steps * 2.0 ** -8, name
    live = int(layer.offsets[-1])
    assert live == 2 * (n - n // 8)
    for rows in (layer.xs, layer.b, layer.db, layer.dxs):   # behind the last token
        assert bool((rows[live:] == 0).all())
    assert bool((layer.out[n - n // 8:] == 0).all()) and bool((layer.dgate[n - n // 8:] == 0).all())


def test_a_layer_in_a_graph_takes_new_tokens(cuda, lib):
    """Captured once, replayed on other tokens and other experts: the host is not asked."""
    with lib.Handle() as h:
        made_ = made(400, 256, 320, 6, 1)
        other = made(400, 256, 320, 6, 2)
        layer = Layer(h, *made_[:-1])
        dout = made_[-1]
        stream = torch.cuda.Stream()
        h.set_stream(stream)
        with torch.cuda.stream(stream):
            layer.forward()
            layer.backward(dout)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            layer.forward()
            layer.backward(dout)
        for mine, theirs in zip(made_, other):
            mine.copy_(theirs)
        layer.xs.zero_(), layer.b.zero_(), layer.db.zero_(), layer.dxs.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [v.clone() for v in (layer.out, layer.dx, layer.dw, layer.dw1, layer.dw2, layer.dgate)]
        with torch.cuda.stream(stream):
            layer.forward()
            layer.backward(dout)
        torch.cuda.synchronize()
        for a, b in zip(got, (layer.out, layer.dx, layer.dw, layer.dw1, layer.dw2, layer.dgate)):
            assert torch.equal(a, b)
        want = reference(*other, layer)
        assert ((got[0].double() - want[0]).norm() / want[0].norm()).item() <= 4 * 2.0 ** -8
        graph.reset()


def padded(k, unit):
    return -(-k // unit) * unit


@pytest.mark.parametrize("n,k,m,experts", [(5, 256, 130, 4), (200, 1000, 512, 8), (3000, 512, 384, 4)])
def test_a_layer_served_in_4_bits(cuda, handle, n, k, m, experts):
    """Tokens quantised once and moved as bytes give what moved and then quantised
    tokens give, bit for bit."""
    gen = generator(n)
    x = torch.randn(n, k, generator=gen, device="cuda").to(torch.bfloat16)
    w = (torch.randn(experts, m, k, generator=gen, device="cuda") / k ** 0.5).to(torch.bfloat16)
    group = torch.randint(-1, experts, (n, 2), generator=gen, device="cuda", dtype=torch.int32)
    rows, ldq, lds = 2 * n, padded(-(-k // 2), 16), padded(-(-k // 32), 16)
    new = lambda *s: torch.zeros(s, dtype=torch.uint8, device="cuda")  # noqa: E731
    offsets, place = torch.zeros(experts + 1, dtype=torch.int32, device="cuda"), torch.zeros(n, 2, dtype=torch.int32, device="cuda")
    handle.sort_tokens(n, 2, experts, group, offsets, place)
    wq, ws = new(experts, m, ldq), new(experts, m, lds)
    handle.quantize_fp4(k, m, w, BF16, k, wq, ldq, ws, lds, batch=experts, stride_x=m * k, stride_q=m * ldq, stride_scale=m * lds)
    results = []
    for first in (True, False):
        xq, xs = new(rows, ldq), new(rows, lds)
        if first:
            q, s = new(n, ldq), new(n, lds)
            handle.quantize_fp4(k, n, x, BF16, k, q, ldq, s, lds)
            handle.scatter_tokens(ldq, n, 2, rows, place, None, q, BYTE, ldq, xq, ldq)
            handle.scatter_tokens(lds, n, 2, rows, place, None, s, BYTE, lds, xs, lds)
        else:
            moved = torch.zeros(rows, k, dtype=torch.bfloat16, device="cuda")
            handle.scatter_tokens(k, n, 2, rows, place, None, x, BF16, k, moved, k)
            handle.quantize_fp4(k, rows, moved, BF16, k, xq, ldq, xs, lds)
        y = torch.zeros(rows, m, device="cuda")
        handle.grouped_gemm_fp4(m, rows, k, experts, offsets, wq, ldq, m * ldq, ws, lds, m * lds, xq, ldq, xs, lds, y, FP32, m)
        out = torch.zeros(n, m, device="cuda")
        handle.gather_tokens(m, n, 2, rows, place, None, y, FP32, m, out, m)
        results.append(out)
    assert torch.equal(*results)
    full = torch.zeros(n, m, dtype=torch.float64, device="cuda")
    for e in range(experts):
        token, _ = torch.nonzero(group == e, as_tuple=True)
        full.index_add_(0, token, x[token].double() @ w[e].double().mT)
    # A value of e2m1 with a power of two for its block is off by 2^-2 of itself at most
    # (and of the block's values below the grid, less than that of the block's norm): two
    # operands, errors that add up like independent ones.
    assert ((results[0].double() - full).norm() / full.norm()).item() < 2 * 0.25 / 3 ** 0.5


def test_a_layer_served_in_8_bits(cuda, handle):
    """The norm's e4m3 values and scales, moved to their experts, are what the 8-bit
    product takes."""
    n, k, m, experts = 300, 640, 256, 5
    x, r, w, w1, _, group, gate, _ = made(n, k, m, experts, 3)
    kb, rows = 5, 2 * n
    q, s = torch.zeros(n, k, dtype=torch.uint8, device="cuda"), torch.zeros(n, kb, device="cuda")
    h, y = torch.empty_like(x), torch.empty_like(x)
    handle.rms_norm(k, n, BF16, x, k, r, k, w, EPS, h, k, y, k, q, k, s, kb)
    offsets, place = torch.zeros(experts + 1, dtype=torch.int32, device="cuda"), torch.zeros(n, 2, dtype=torch.int32, device="cuda")
    handle.sort_tokens(n, 2, experts, group, offsets, place)
    xq, xs = torch.zeros(rows, k, dtype=torch.uint8, device="cuda"), torch.zeros(rows, kb, device="cuda")
    handle.scatter_tokens(k, n, 2, rows, place, None, q, BYTE, k, xq, k)
    handle.scatter_tokens(kb, n, 2, rows, place, None, s, FP32, kb, xs, kb)
    wq, ws = torch.zeros(experts, m, k, dtype=torch.uint8, device="cuda"), torch.zeros(experts, 2, kb, device="cuda")
    handle.quantize_fp8(k, m, 128, w1, BF16, k, wq, k, ws, kb, batch=experts, stride_x=m * k, stride_q=m * k, stride_scale=2 * kb)
    b = torch.zeros(rows, m, device="cuda")
    handle.grouped_gemm_fp8(m, rows, k, experts, offsets, wq, k, m * k, ws, kb, 2 * kb, xq, k, xs, kb, b, FP32, m)
    out = torch.zeros(n, m, device="cuda")
    handle.gather_tokens(m, n, 2, rows, place, gate, b, FP32, m, out, m)
    full = torch.zeros(n, m, dtype=torch.float64, device="cuda")
    for e in range(experts):
        token, choice = torch.nonzero(group == e, as_tuple=True)
        full.index_add_(0, token, gate[token, choice, None].double() * (y[token].double() @ w1[e].double().mT))
    # Each operand's values are off by 2^-4 at most, and y itself is rounded to BF16.
    assert ((out.double() - full).norm() / full.norm()).item() < 2 * 2.0 ** -4 / 3 ** 0.5


def test_the_example_serves_in_4_bits(cuda):
    path = pathlib.Path(__file__).resolve().parent.parent / "examples" / "moe_layer.py"
    spec = importlib.util.spec_from_file_location("moe_layer", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    losses, deviation = example.main(300, 256, 512, 6, steps=3, quiet=True)
    assert len(losses) == 3 and all(loss == loss for loss in losses) and 0 < deviation < 0.08
    assert sg.get_device_errors() == 0


@pytest.mark.parametrize("tokens,width,hidden,experts", [(300, 256, 512, 6), (257, 130, 264, 5)])
def test_the_example_in_4_bits_is_near_bf16(cuda, tokens, width, hidden, experts):
    path = pathlib.Path(__file__).resolve().parent.parent / "examples" / "moe_layer.py"
    spec = importlib.util.spec_from_file_location("moe_layer", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    _, _, deviation = example.train_and_serve(tokens, width, hidden, experts, steps=2)
    # Two products of two operands each, whose values are off by 2^-2 of themselves at most
    # (test_a_layer_served_in_4_bits); outputs of nothing are off by 1, wrong ones by more.
    assert 0 < deviation < 4 * 0.25 / 3 ** 0.5


def test_one_handle_on_two_streams(cuda, lib):
    """Calls that use the handle's workspace (partial sums, laid-out scales) wait for
    each other, whichever streams they are on."""
    n, k = 20000, 1024
    gen = generator(5)
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(torch.bfloat16)  # noqa: E731
    h_, dy = [rand(n, k) for _ in range(2)], [rand(n, k) for _ in range(2)]
    codes = [[torch.randint(0, 256, (6144, k), generator=gen, device="cuda").to(torch.uint8) for _ in range(2)] for _ in range(2)]
    scales = [[torch.randint(118, 128, (6144, k // 16), generator=gen, device="cuda").to(torch.uint8) for _ in range(2)] for _ in range(2)]
    new = lambda: ([torch.empty(k, device="cuda") for _ in range(2)], [torch.empty(n, k, dtype=torch.bfloat16, device="cuda") for _ in range(2)],  # noqa: E731
                   [torch.empty(6144, 6144, dtype=torch.bfloat16, device="cuda") for _ in range(2)])

    def call(h, i, dw, dx, y):
        h.rms_norm_backward(k, n, BF16, dy[i], k, h_[i], k, None, EPS, None, k, dx[i], k, 0.0, dw[i])
        h.gemm_fp4(6144, 6144, 2 * k, codes[i][0], k, scales[i][0], k // 16, codes[i][1], k, scales[i][1], k // 16, y[i], BF16, 6144)

    with lib.Handle() as h:
        want = new()
        for i in range(2):
            call(h, i, *want)
            torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(2)]
        got = new()
        torch.cuda.synchronize()
        for _ in range(4):
            for i in range(2):
                h.set_stream(streams[i])
                call(h, i, *got)
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_two_handles_at_once(cuda, lib):
    """Two layers on two streams, each with its own handle."""
    made_ = [made(500, 256, 320, 6, seed) for seed in (3, 4)]
    handles = [lib.Handle() for _ in range(2)]
    try:
        layers = [Layer(h, *m[:-1]) for h, m in zip(handles, made_)]
        for layer, m in zip(layers, made_):
            layer.forward(), layer.backward(m[-1])
        torch.cuda.synchronize()
        want = [[v.clone() for v in (layer.out, layer.dx, layer.dw, layer.dw1, layer.dw2, layer.dgate)] for layer in layers]
        streams = [torch.cuda.Stream() for _ in range(2)]
        for h, s in zip(handles, streams):
            h.set_stream(s)
        for _ in range(5):
            for layer, m, s in zip(layers, made_, streams):
                with torch.cuda.stream(s):
                    layer.forward(), layer.backward(m[-1])
        torch.cuda.synchronize()
        for layer, w in zip(layers, want):
            got = (layer.out, layer.dx, layer.dw, layer.dw1, layer.dw2, layer.dgate)
            assert all(torch.equal(a, b) for a, b in zip(got, w))
    finally:
        for h in handles:
            h.close()
