"""The operators of a mixture-of-experts layer and of its optimiser, as measured: sizes, inputs, plain forms.

Matrices are torch tensors in row-major order; the library reads the same
memory as column-major matrices (a token is a column). Five passes:

forward        Y[t] = W[e(t)] X[t] for tokens sorted by expert, bfloat16
backward       dX[t] = W[e(t)]^T dY[t] and dW[e] = sum over t of e: dY[t] X[t]^T
fp8            the forward product in 8-bit floating point (e4m3), one scale
               for each 128 values of a token and one for each 128 x 128 block
               of the weights; with groups == 1, one ordinary linear layer
quantize       to e4m3 with a scale for each 1 x 128 or 128 x 128 block
orthogonalize  five Newton-Schulz steps on a batch of gradients
"""
import math

import torch

own = False

# Quintic Newton-Schulz: X <- a X + b (X X^T) X + c (X X^T)^2 X. These
# coefficients take singular values of (0, 1] to about 0.7 .. 1.2 in five steps.
STEPS = 5
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
EPS = 1e-7
FP8_MAX = 448.0
AMAX_FLOOR = 2.0 ** -100   # a block of zeros gets this as its largest magnitude
BLOCK = 128

_handle = None


def listed():
    return [
        # A decoding step of a small model: eight tokens, most experts idle.
        {"name": "forward decode 8", "op": "forward", "groups": 8, "tokens": 8, "m": 1024, "k": 1024, "out": "bf16"},
        # A batch of sequences decoding together: every weight is read for a few tokens.
        {"name": "forward decode 192", "op": "forward", "groups": 32, "tokens": 192, "m": 2048, "k": 4096, "out": "bf16"},
        # A prompt or a training batch: sixteen experts, full tiles.
        {"name": "forward 16384", "op": "forward", "groups": 16, "tokens": 16384, "m": 4096, "k": 4096, "out": "bf16"},
        # Ragged training step of a small model, sizes that divide no tile.
        {"name": "backward ragged 3001", "op": "backward", "groups": 24, "tokens": 3001, "m": 1000, "k": 1537, "out": "fp32"},
        # Training step: gradients of tokens (bf16) and of the weights (fp32).
        {"name": "backward 16384", "op": "backward", "groups": 16, "tokens": 16384, "m": 2048, "k": 4096, "out": "fp32"},
        # One token through one linear layer of 8-bit weights.
        {"name": "fp8 linear 1", "op": "fp8", "groups": 1, "tokens": 1, "m": 4096, "k": 4096, "out": "bf16"},
        # Decoding with 8-bit experts.
        {"name": "fp8 experts 384", "op": "fp8", "groups": 32, "tokens": 384, "m": 2048, "k": 2048, "out": "bf16"},
        # A prompt through one large linear layer.
        {"name": "fp8 linear 8192", "op": "fp8", "groups": 1, "tokens": 8192, "m": 8192, "k": 4096, "out": "bf16"},
        # Activations of a few tokens before an 8-bit product, odd length.
        {"name": "quantize 333 tokens", "op": "quantize", "rows": 333, "k": 1537, "block": 1, "type": "bf16"},
        # Activations of a prompt.
        {"name": "quantize 16384 tokens", "op": "quantize", "rows": 16384, "k": 8192, "block": 1, "type": "bf16"},
        # Updates of a batch of small projections.
        {"name": "orthogonalize 8x256x512", "op": "orthogonalize", "batch": 8, "rows": 256, "cols": 512, "type": "bf16"},
        # The update of one large projection.
        {"name": "orthogonalize 4096x2048", "op": "orthogonalize", "batch": 1, "rows": 4096, "cols": 2048, "type": "fp32"},
    ]


def _size(rng, low, high):
    """Spread over the logarithm: half are multiples of 64, a quarter of 8, a quarter anything."""
    v = math.exp(rng.uniform(math.log(low), math.log(high)))
    step = rng.choice([64, 64, 8, 1])
    return max(low, min(high, int(v / step + 0.5) * step))


def draw(rng):
    op = rng.choice(["forward", "forward", "backward", "fp8", "fp8", "quantize", "orthogonalize"])
    if op in ("forward", "backward", "fp8"):
        groups = int(round(math.exp(rng.uniform(0.0 if op == "fp8" else math.log(2), math.log(64)))))
        m, k = _size(rng, 128, 4096), _size(rng, 128, 4096)
        top = min(16384.0, 1.6e11 / (m * k))   # no more products than the largest listed case has
        tokens = int(math.exp(rng.uniform(0.0, math.log(top))))
        return {"op": op, "groups": groups, "tokens": tokens, "m": m, "k": k, "out": rng.choice(["bf16", "bf16", "fp32"])}
    if op == "quantize":
        k = _size(rng, 128, 8192)
        rows = int(math.exp(rng.uniform(0.0, math.log(16384.0))))
        return {"op": op, "rows": rows, "k": k, "block": rng.choice([1, 1, BLOCK]), "type": rng.choice(["bf16", "fp32"])}
    rows, cols = _size(rng, 64, 4096), _size(rng, 64, 4096)
    cost = max(rows, cols) * min(rows, cols) ** 2
    most = max(1, min(16, int(1.7e10 / cost)))
    if cost > 1.7e10:
        cols = min(cols, 2048)
        rows = min(rows, int(1.7e10 / (cols * min(rows, cols))))
    return {"op": op, "batch": int(math.exp(rng.uniform(0.0, math.log(most + 0.5)))), "rows": rows, "cols": cols,
            "type": rng.choice(["bf16", "fp32"])}


# ---- inputs ------------------------------------------------------------------

def _shares(groups):
    """How often each expert is chosen: routers are uneven, here by about a factor of five."""
    p = [1.0 / (e + groups / 4.0 + 1.0) for e in range(groups)]
    return [v / sum(p) for v in p]


def _type(name):
    return {"bf16": torch.bfloat16, "fp32": torch.float32}[name]


def _activations(gen, rows, k, type_):
    """Normal values, a few channels of which are ten times as large."""
    x = torch.randn(rows, k, generator=gen, device="cuda")
    x[:, torch.randperm(k, generator=gen, device="cuda")[: max(1, k // 100)]] *= 10.0
    return x.to(type_)


def _padded(x, rows, cols):
    """`x` with zeros after its last two axes' ends, up to multiples of `rows` and `cols`."""
    r, c = x.shape[-2:]
    return torch.nn.functional.pad(x, (0, -c % cols, 0, -r % rows))


def _quantized(x, block):
    """e4m3 values and the scale of each `block` x 128 block of the last two axes."""
    r, c = x.shape[-2:]
    v = _padded(x.float(), block, BLOCK)
    v = v.reshape(*v.shape[:-2], v.shape[-2] // block, block, v.shape[-1] // BLOCK, BLOCK)
    scale = v.abs().amax(dim=(-3, -1)).clamp(min=AMAX_FLOOR) / FP8_MAX
    q = (v / scale[..., :, None, :, None]).to(torch.float8_e4m3fn)
    q = q.reshape(*q.shape[:-4], q.shape[-4] * block, q.shape[-2] * BLOCK)[..., :r, :c].contiguous()
    return q, scale


def _routing(case, seed, gen):
    """Where each expert's tokens begin among all, on the device, and the fullest expert's count."""
    groups, tokens = case["groups"], case["tokens"]
    if groups == 1:
        return None, tokens
    p = torch.tensor(_shares(groups), device="cuda")[torch.randperm(groups, generator=gen, device="cuda")]
    chosen = torch.multinomial(p, tokens, replacement=True, generator=gen)
    counts = torch.bincount(chosen, minlength=groups)
    offsets = torch.zeros(groups + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = counts.cumsum(0)
    return offsets, int(counts.max())


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = {"case": case}
    op = case["op"]
    if op == "quantize":
        rows, k, block = case["rows"], case["k"], case["block"]
        s["x"] = _activations(gen, rows, k, _type(case["type"]))
        s["q"] = torch.empty(rows, k, dtype=torch.float8_e4m3fn, device="cuda")
        s["scale"] = torch.empty(-(-rows // block), -(-k // BLOCK), device="cuda")
        return s
    if op == "orthogonalize":
        b, r, c = case["batch"], case["rows"], case["cols"]
        rank = max(1, min(r, c) // 8)   # gradients: a few strong directions over noise
        g = torch.randn(b, r, rank, generator=gen, device="cuda") @ torch.randn(b, rank, c, generator=gen, device="cuda")
        g = 1e-3 * (g / math.sqrt(rank) + 0.3 * torch.randn(b, r, c, generator=gen, device="cuda"))
        s["g"] = g.to(_type(case["type"]))
        s["o"] = torch.empty(b, r, c, dtype=torch.bfloat16, device="cuda")
        return s
    groups, tokens, m, k = case["groups"], case["tokens"], case["m"], case["k"]
    s["offsets"], s["most"] = _routing(case, seed, gen)
    x = _activations(gen, tokens, k, torch.bfloat16)
    w = (torch.randn(groups, m, k, generator=gen, device="cuda") / math.sqrt(k)).to(torch.bfloat16)
    if op == "fp8":
        s["x"], s["x_scale"] = _quantized(x, 1)
        s["w"], s["w_scale"] = _quantized(w, BLOCK)
    else:
        s["x"], s["w"] = x, w
    if op == "backward":
        s["dy"] = (0.01 * torch.randn(tokens, m, generator=gen, device="cuda")).to(torch.bfloat16)
        s["dx"] = torch.empty(tokens, k, dtype=torch.bfloat16, device="cuda")
        s["dw"] = torch.empty(groups, m, k, dtype=_type(case["out"]), device="cuda")
    else:
        s["y"] = torch.empty(tokens, m, dtype=_type(case["out"]), device="cuda")
    return s


# ---- the plain forms -----------------------------------------------------------

def _places(s):
    """Each token's expert and its place among that expert's tokens."""
    row = torch.arange(s["case"]["tokens"], device="cuda")
    expert = torch.searchsorted(s["offsets"][1:].contiguous(), row, right=True)
    return expert, row - s["offsets"][expert]


def _by_expert(s, x, expert, place):
    """The rows of `x` by expert and place, zeros where an expert has fewer tokens than the fullest."""
    v = torch.zeros(s["case"]["groups"], s["most"], x.shape[1], device="cuda")
    v[expert, place] = x
    return v


def _grouped(s, x, w):
    """Rows of `x` times the transposed `w` of their expert, in 32 bits."""
    if s["offsets"] is None:
        return x @ w[0].t()
    expert, place = _places(s)
    return (_by_expert(s, x, expert, place) @ w.transpose(1, 2))[expert, place]


def _spread(scale, rows, cols, block):
    """A block's scale at each of its values."""
    v = scale.repeat_interleave(BLOCK, dim=-1)[..., :cols]
    return v if block == 1 else v.repeat_interleave(block, dim=-2)[..., :rows, :]


def _plain(s):
    case = s["case"]
    op = case["op"]
    if op == "forward":
        return _grouped(s, s["x"].float(), s["w"].float()).to(s["y"].dtype)
    if op == "backward":
        expert, place = _places(s)
        x = _by_expert(s, s["x"].float(), expert, place)
        dy = _by_expert(s, s["dy"].float(), expert, place)
        dx = (dy @ s["w"].float())[expert, place]
        return dx.to(torch.bfloat16), (dy.transpose(1, 2) @ x).to(s["dw"].dtype)
    if op == "fp8":
        tokens, m, k = case["tokens"], case["m"], case["k"]
        x = s["x"].float() * _spread(s["x_scale"], tokens, k, 1)
        w = s["w"].float() * _spread(s["w_scale"], m, k, BLOCK)
        return _grouped(s, x, w).to(s["y"].dtype)
    if op == "quantize":
        return _quantized(s["x"], case["block"])
    a, b, c = COEFFICIENTS
    g = s["g"].float()
    x = g / (g.square().sum(dim=(1, 2), keepdim=True).sqrt() + EPS)
    tall = x.shape[1] > x.shape[2]
    x = x.transpose(1, 2) if tall else x
    for _ in range(STEPS):
        gram = x @ x.transpose(1, 2)
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    x = x.transpose(1, 2) if tall else x
    return x.to(torch.bfloat16)


# ---- the library's calls ---------------------------------------------------------

def _library(s):
    global _handle
    import sgblas_b200 as sg
    if _handle is None:
        _handle = sg.Handle()
    h, case = _handle, s["case"]
    op = case["op"]
    if op == "quantize":
        rows, k = case["rows"], case["k"]
        h.quantize_fp8(k, rows, case["block"], s["x"], sg.SGBLAS_TYPE_BF16 if case["type"] == "bf16" else sg.SGBLAS_TYPE_FP32,
                       k, s["q"], k, s["scale"], -(-k // BLOCK))
        return s["q"], s["scale"]
    if op == "orthogonalize":
        b, r, c = case["batch"], case["rows"], case["cols"]
        h.orthogonalize(c, r, b, STEPS, COEFFICIENTS, EPS, 1.0, s["g"],
                        sg.SGBLAS_TYPE_BF16 if case["type"] == "bf16" else sg.SGBLAS_TYPE_FP32, c, r * c, s["o"], c, r * c)
        return s["o"]
    groups, tokens, m, k = case["groups"], case["tokens"], case["m"], case["k"]
    out = sg.SGBLAS_TYPE_BF16 if case["out"] == "bf16" else sg.SGBLAS_TYPE_FP32
    if op == "forward":
        h.grouped_gemm_n(sg.SGBLAS_OP_T, m, tokens, k, groups, s["offsets"], 1.0, s["w"], k, m * k, s["x"], k, 0.0, s["y"], out, m)
        return s["y"]
    if op == "backward":
        h.grouped_gemm_n(sg.SGBLAS_OP_N, k, tokens, m, groups, s["offsets"], 1.0, s["w"], k, m * k, s["dy"], m, 0.0, s["dx"],
                         sg.SGBLAS_TYPE_BF16, k)
        h.grouped_gemm_k(k, m, tokens, groups, s["offsets"], 1.0, s["x"], k, s["dy"], m, 0.0, s["dw"], out, k, m * k)
        return s["dx"], s["dw"]
    blocks = -(-k // BLOCK)
    if groups == 1:
        h.gemm_fp8(m, tokens, k, s["w"], k, s["w_scale"], blocks, s["x"], k, s["x_scale"], blocks, s["y"], out, m)
    else:
        h.grouped_gemm_fp8(m, tokens, k, groups, s["offsets"], s["w"], k, m * k, s["w_scale"], blocks, blocks * -(-m // BLOCK),
                           s["x"], k, s["x_scale"], blocks, s["y"], out, m)
    return s["y"]


def run(state):
    return _library(state) if own else _plain(state)


# ---- what cannot be left out -----------------------------------------------------

def work(case):
    op = case["op"]
    size = {"bf16": 2, "fp32": 4}
    if op == "quantize":
        n = case["rows"] * case["k"]
        return {"bytes": n * (size[case["type"]] + 1) + 4 * -(-case["rows"] // case["block"]) * -(-case["k"] // BLOCK), "flops": 2 * n}
    if op == "orthogonalize":
        s, l = sorted((case["rows"], case["cols"]))
        step = l * s * (s + 1) + s * s * (s + 1) + 2 * l * s * s   # the two symmetric products by halves
        return {"bytes": case["batch"] * s * l * (size[case["type"]] + 2), "flops": case["batch"] * STEPS * step}
    groups, t, m, k = case["groups"], case["tokens"], case["m"], case["k"]
    chosen = sum(1.0 - (1.0 - p) ** t for p in _shares(groups))   # experts that have a token
    if op == "forward":
        return {"bytes": 2 * (t * k + chosen * m * k) + size[case["out"]] * t * m, "flops": 2 * t * m * k}
    if op == "fp8":
        return {"bytes": (t * k + chosen * m * k) * (1 + 4 / BLOCK) + size[case["out"]] * t * m, "flops": 2 * t * m * k}
    return {"bytes": 2 * (t * (2 * k + m) + chosen * m * k) + size[case["out"]] * groups * m * k, "flops": 4 * t * m * k}


# ---- the definitions in 64 bits -----------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        x = s["x"].double()
        rows, k, block = case["rows"], case["k"], case["block"]
        q = torch.empty_like(x)
        scale = torch.empty(s["scale"].shape, dtype=torch.float64, device="cuda")
        for j in range(0, k, BLOCK):
            part = x[:, j:j + BLOCK]
            top = part.abs().amax(dim=1)
            if block > 1:
                top = torch.stack([t.amax() for t in top.split(block)])
            scale[:, j // BLOCK] = top.clamp(min=AMAX_FLOOR) / FP8_MAX
            q[:, j:j + BLOCK] = part / scale[:, j // BLOCK].repeat_interleave(block)[:rows, None]
        return q, scale   # the values before their rounding to 8 bits
    if op == "orthogonalize":
        a, b, c = COEFFICIENTS
        out = []
        for g in s["g"].double():
            x = g / (torch.linalg.matrix_norm(g) + EPS)
            for _ in range(STEPS):
                if x.shape[0] <= x.shape[1]:
                    p = x @ x.mT
                    x = a * x + b * (p @ x) + c * (p @ (p @ x))
                else:
                    p = x.mT @ x
                    x = a * x + b * (x @ p) + c * ((x @ p) @ p)
            out.append(x)
        return torch.stack(out)
    groups, tokens, m, k = case["groups"], case["tokens"], case["m"], case["k"]
    ends = [0, tokens] if s["offsets"] is None else s["offsets"].tolist()
    y = torch.zeros(tokens, m, dtype=torch.float64, device="cuda")
    dx = torch.zeros(tokens, k, dtype=torch.float64, device="cuda")
    dw = torch.zeros(groups, m, k, dtype=torch.float64, device="cuda") if op == "backward" else None
    for e in range(groups):
        lo, hi = ends[e], ends[e + 1]
        x, w = s["x"][lo:hi].double(), s["w"][e].double()
        if op == "fp8":
            for j in range(0, k, BLOCK):
                for i in range(0, m, BLOCK):
                    w[i:i + BLOCK, j:j + BLOCK] *= s["w_scale"][e, i // BLOCK, j // BLOCK].double()
                x[:, j:j + BLOCK] *= s["x_scale"][lo:hi, j // BLOCK, None].double()
        if op == "backward":
            dy = s["dy"][lo:hi].double()
            dx[lo:hi] = dy @ w
            dw[e] = dy.mT @ x
        else:
            y[lo:hi] = x @ w.mT
    return (dx, dw) if op == "backward" else y
