"""A mixture-of-experts layer on the library's products: trained in BF16, its
experts' updates orthogonalised, then served in 8 bits.

    python examples/moe_layer.py [--tokens 2048] [--width 512] [--hidden 1024] [--experts 8]

Each token goes to one expert e: y = W2[e] relu(W1[e] x). The forward and token
gradient products are sgblasGroupedGemmN, the weight gradients
sgblasGroupedGemmK (into FP32), the update of every expert's matrices one
sgblasOrthogonalize per weight tensor, and serving quantises the weights once
(128 x 128 blocks) and the tokens per call (1 x 128) for sgblasGroupedGemmFp8.
Routing, the activation and the loss are torch's.

Tensors are row-major; the library reads the same memory as column-major
matrices, so a [tokens, k] tensor is a k x tokens matrix.
"""
from __future__ import annotations

import argparse
import pathlib
import sys

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parent.parent))

import torch

import sgblas_b200 as sg

BF16, FP32 = sg.SGBLAS_TYPE_BF16, sg.SGBLAS_TYPE_FP32
BLOCK = 128


class Experts:
    """Two weight tensors, [experts, hidden, width] and [experts, width, hidden]."""

    def __init__(self, handle: sg.Handle, experts: int, width: int, hidden: int, gen):
        self.h, self.experts = handle, experts
        make = lambda rows, cols: torch.randn(experts, rows, cols, generator=gen, device="cuda") / cols ** 0.5  # noqa: E731
        self.master = [make(hidden, width), make(width, hidden)]
        self.weights = [w.to(torch.bfloat16) for w in self.master]
        self.momentum = [torch.zeros_like(w) for w in self.master]

    def product(self, w, x, offsets):
        """Rows of x times the transposed weights of their expert."""
        m, k = w.shape[1:]
        y = torch.empty(x.shape[0], m, dtype=torch.bfloat16, device="cuda")
        self.h.grouped_gemm_n(sg.SGBLAS_OP_T, m, x.shape[0], k, self.experts, offsets, 1.0, w, k,
                              m * k, x, k, 0.0, y, BF16, m)
        return y

    def token_gradient(self, w, dy, offsets):
        m, k = w.shape[1:]
        dx = torch.empty(dy.shape[0], k, dtype=torch.bfloat16, device="cuda")
        self.h.grouped_gemm_n(sg.SGBLAS_OP_N, k, dy.shape[0], m, self.experts, offsets, 1.0, w, k,
                              m * k, dy, m, 0.0, dx, BF16, k)
        return dx

    def weight_gradient(self, w, x, dy, offsets):
        m, k = w.shape[1:]
        dw = torch.empty(w.shape, device="cuda")
        self.h.grouped_gemm_k(k, m, x.shape[0], self.experts, offsets, 1.0, x, k, dy, m, 0.0, dw,
                              FP32, k, m * k)
        return dw

    def forward(self, x, offsets):
        hidden = self.product(self.weights[0], x, offsets)
        act = torch.relu(hidden)
        return hidden, act, self.product(self.weights[1], act, offsets)

    def step(self, x, dy, hidden, act, offsets, rate):
        """One update from the gradient dy of the outputs; the tokens' gradient."""
        grads = [None, self.weight_gradient(self.weights[1], act, dy, offsets)]
        dhidden = self.token_gradient(self.weights[1], dy, offsets) * (hidden > 0)
        grads[0] = self.weight_gradient(self.weights[0], x, dhidden, offsets)
        dx = self.token_gradient(self.weights[0], dhidden, offsets)
        for master, weight, momentum, grad in zip(self.master, self.weights, self.momentum, grads):
            momentum.mul_(0.9).add_(grad)
            e, rows, cols = master.shape
            update = torch.empty(master.shape, dtype=torch.bfloat16, device="cuda")
            self.h.orthogonalize(cols, rows, e, 5, (3.4445, -4.7750, 2.0315), 1e-7,
                                 max(1.0, rows / cols) ** 0.5, momentum, FP32, cols, rows * cols,
                                 update, cols, rows * cols)
            master.sub_(update.float(), alpha=rate)
            weight.copy_(master)
        return dx

    # ---- in 8 bits -------------------------------------------------------------

    def quantize(self):
        """(values, scales) of each weight tensor, a scale per 128 x 128 block."""
        out = []
        for w in self.weights:
            e, rows, cols = w.shape
            kb, nb = -(-cols // BLOCK), -(-rows // BLOCK)
            q = torch.empty(e, rows, cols, dtype=torch.uint8, device="cuda")
            s = torch.empty(e, nb, kb, device="cuda")
            self.h.quantize_fp8(cols, rows, BLOCK, w, BF16, cols, q, cols, s, kb, batch=e,
                                stride_x=rows * cols, stride_q=rows * cols, stride_scale=nb * kb)
            out.append((q, s))
        return out

    def product_fp8(self, weights, x, offsets):
        q, s = weights
        e, m, k = q.shape
        kb = -(-k // BLOCK)
        xq = torch.empty(x.shape, dtype=torch.uint8, device="cuda")
        xs = torch.empty(x.shape[0], kb, device="cuda")
        self.h.quantize_fp8(k, x.shape[0], 1, x, BF16, k, xq, k, xs, kb)
        y = torch.empty(x.shape[0], m, dtype=torch.bfloat16, device="cuda")
        self.h.grouped_gemm_fp8(m, x.shape[0], k, e, offsets, q, k, m * k, s, kb, s.shape[1] * kb, xq,
                                k, xs, kb, y, BF16, m)
        return y

    def serve(self, quantized, x, offsets):
        return self.product_fp8(quantized[1], torch.relu(self.product_fp8(quantized[0], x, offsets)),
                                offsets)


def route(x, router):
    """Tokens sorted by expert, and where each expert's begin (on the device)."""
    expert = (x @ router).argmax(dim=1)
    order = torch.argsort(expert, stable=True)
    counts = torch.bincount(expert, minlength=router.shape[1])
    offsets = torch.zeros(router.shape[1] + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = counts.cumsum(0)
    return order, offsets


def main(tokens=2048, width=512, hidden=1024, experts=8, steps=30, seed=0, quiet=False):
    """Trains on a fixed random map; returns the losses and the 8-bit deviation."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    router = torch.randn(width, experts, generator=gen, device="cuda")
    target = torch.randn(width, width, generator=gen, device="cuda") / width ** 0.5
    losses = []
    with sg.Handle() as h:
        h.set_stream(torch.cuda.current_stream())
        layer = Experts(h, experts, width, hidden, gen)
        for step in range(steps):
            x = torch.randn(tokens, width, generator=gen, device="cuda")
            order, offsets = route(x, router)
            x = x[order].to(torch.bfloat16)
            want = x.float() @ target
            hid, act, y = layer.forward(x, offsets)
            diff = y.float() - want
            losses.append(diff.square().mean().item())
            dy = (2.0 / diff.numel() * diff).to(torch.bfloat16)
            layer.step(x, dy, hid, act, offsets, rate=0.02)
        x = torch.randn(64, width, generator=gen, device="cuda")   # a batch being decoded
        order, offsets = route(x, router)
        x = x[order].to(torch.bfloat16)
        full = layer.forward(x, offsets)[2].float()
        small = layer.serve(layer.quantize(), x, offsets).float()
        deviation = ((small - full).norm() / full.norm()).item()
    if not quiet:
        print(f"loss {losses[0]:.4f} -> {losses[-1]:.4f} in {steps} steps; "
              f"8-bit serving is {100 * deviation:.2f} % off BF16; "
              f"device errors {sg.get_device_errors()}")
    return losses, deviation


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    for name, default in (("tokens", 2048), ("width", 512), ("hidden", 1024), ("experts", 8), ("steps", 30)):
        parser.add_argument(f"--{name}", type=int, default=default)
    main(**vars(parser.parse_args()))
