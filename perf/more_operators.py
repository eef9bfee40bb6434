"""The operators around an expert layer's products, as measured: sizes, inputs, plain forms.

Matrices are torch tensors in row-major order; the library reads the same
memory as column-major matrices (a token is a column). Six passes:

norm              h = x + r, y = h / sqrt(mean h^2 + eps) * w, as it is or in
                  8 bits (e4m3) with a scale for each 128 values
norm_backward     gradients of x (and r) and of w
dispatch          the experts that each token goes to, sorted: where each
                  expert's rows begin, each choice's row, and the rows
combine           each token's rows back, weighted and added
combine_backward  gradients of the rows and of the weights
linear4           a linear layer, or the experts', in 4 bits (e2m1 with a power
                  of two for each 32 values): quantisation of the tokens and
                  the product with weights quantised before
"""
import math

import torch

own = False

EPS = 1e-6
FP8_MAX = 448.0
AMAX_FLOOR = 2.0 ** -100   # a block of zeros gets this as its largest magnitude
BLOCK = 128
BLOCK4 = 32
VALUES4 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)   # magnitudes of e2m1 by their code

_handle = None


def listed():
    return [
        # One token being decoded: the norm before an 8-bit layer.
        {"name": "norm e4m3 1 token", "op": "norm", "tokens": 1, "k": 4096, "type": "bf16", "out": "e4m3", "residual": True},
        # A training batch of a large model.
        {"name": "norm 16384 tokens", "op": "norm", "tokens": 16384, "k": 4096, "type": "bf16", "out": "same", "residual": True},
        # A small batch of odd length, everything in 32 bits.
        {"name": "norm backward 333x1537", "op": "norm_backward", "tokens": 333, "k": 1537, "type": "fp32", "residual": False},
        # The backward pass of the training batch.
        {"name": "norm backward 16384", "op": "norm_backward", "tokens": 16384, "k": 4096, "type": "bf16", "residual": True},
        # Sixteen sequences decoding, four experts each.
        {"name": "dispatch 16 tokens", "op": "dispatch", "tokens": 16, "top": 4, "groups": 32, "k": 2048, "type": "bf16"},
        # A training batch over many small experts.
        {"name": "dispatch 8192 tokens", "op": "dispatch", "tokens": 8192, "top": 8, "groups": 64, "k": 2048, "type": "bf16"},
        # The same batches on their way back.
        {"name": "combine 16 tokens", "op": "combine", "tokens": 16, "top": 4, "groups": 32, "k": 2048, "type": "bf16"},
        {"name": "combine 8192 tokens", "op": "combine", "tokens": 8192, "top": 8, "groups": 64, "k": 2048, "type": "bf16"},
        # Ragged training step of a small model, sizes that divide nothing.
        {"name": "combine backward ragged 3001", "op": "combine_backward", "tokens": 3001, "top": 3, "groups": 24, "k": 1537, "type": "bf16"},
        {"name": "combine backward 8192", "op": "combine_backward", "tokens": 8192, "top": 8, "groups": 64, "k": 2048, "type": "bf16"},
        # Decoding with experts in 4 bits.
        {"name": "linear4 experts 384", "op": "linear4", "groups": 32, "tokens": 384, "m": 2048, "k": 2048, "out": "bf16"},
        # A prompt through one large linear layer.
        {"name": "linear4 8192", "op": "linear4", "groups": 1, "tokens": 8192, "m": 8192, "k": 4096, "out": "bf16"},
    ]


def _size(rng, low, high):
    """Spread over the logarithm: half are multiples of 64, a quarter of 8, a quarter anything."""
    v = math.exp(rng.uniform(math.log(low), math.log(high)))
    step = rng.choice([64, 64, 8, 1])
    return max(low, min(high, int(v / step + 0.5) * step))


def _count(rng, high):
    return int(math.exp(rng.uniform(0.0, math.log(high + 0.5))))


def draw(rng):
    op = rng.choice(["norm", "norm_backward", "dispatch", "combine", "combine_backward", "linear4", "linear4"])
    if op in ("norm", "norm_backward"):
        k, type_ = _size(rng, 64, 8192), rng.choice(["bf16", "bf16", "fp32"])
        size = 2 if type_ == "bf16" else 4
        tokens = _count(rng, min(16384, 16384 * 4096 * 2 // (k * size)))
        case = {"op": op, "tokens": tokens, "k": k, "type": type_, "residual": rng.choice([True, True, False])}
        if op == "norm":
            case["out"] = rng.choice(["e4m3", "same"])
        return case
    if op == "linear4":
        groups = int(round(math.exp(rng.uniform(0.0, math.log(64)))))
        m, k = _size(rng, 128, 8192), _size(rng, 128, 4096)
        top = min(8192, int(2.7e11 / (m * k)))
        return {"op": op, "groups": groups, "tokens": _count(rng, top), "m": m, "k": k, "out": rng.choice(["bf16", "bf16", "fp32"])}
    top, groups = rng.choice([1, 2, 3, 4, 6, 8]), rng.choice([8, 24, 32, 64, 128])
    k, type_ = _size(rng, 64, 4096), rng.choice(["bf16", "bf16", "fp32"])
    size = 2 if type_ == "bf16" else 4
    tokens = _count(rng, min(8192, 8192 * 8 * 2048 * 2 // (k * top * size)))
    return {"op": op, "tokens": tokens, "top": top, "groups": groups, "k": k, "type": type_}


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


def _up(v, unit):
    return -(-v // unit) * unit


def _groups(case, seed, gen):
    """Where each expert's tokens begin among all, on the device, and the fullest expert's count."""
    groups, tokens = case["groups"], case["tokens"]
    if groups == 1:
        return None, tokens
    p = torch.tensor(_shares(groups), device="cuda")[torch.randperm(groups, generator=gen, device="cuda")]
    counts = torch.bincount(torch.multinomial(p, tokens, replacement=True, generator=gen), minlength=groups)
    offsets = torch.zeros(groups + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = counts.cumsum(0)
    return offsets, int(counts.max())


def _chosen(case, gen):
    """Different experts for each token; a few tokens are padding and have none."""
    tokens, top, groups = case["tokens"], case["top"], case["groups"]
    p = torch.tensor(_shares(groups), device="cuda").log()[torch.randperm(groups, generator=gen, device="cuda")]
    noise = -torch.log(-torch.log(torch.rand(tokens, groups, generator=gen, device="cuda").clamp(1e-7, 1 - 1e-7)))
    expert = torch.topk(p + noise, top, dim=1).indices.to(torch.int32)
    expert[tokens - tokens // 32:] = -1
    return expert


def _codes4(v):
    """Codes of the nearest e2m1 values, ties to the even code; the sign is bit 3."""
    a = v.abs()
    code = (a > 0.25).to(torch.uint8)
    for border, tie_up in ((0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        code += (a >= border) if tie_up else (a > border)
    return code + 8 * torch.signbit(v).to(torch.uint8)


def _power(byte):
    """2^(byte - 127) in 32 bits, from the bits."""
    bits = byte.to(torch.int32)
    return torch.where(bits == 0, torch.full_like(bits, 1 << 22), bits << 23).view(torch.float32)


def _quantized4(x, row, scale_row):
    """Packed e2m1 codes and scale bytes of the last axis, rows padded to `row` and `scale_row` bytes."""
    k = x.shape[-1]
    v = torch.nn.functional.pad(x.float(), (0, -k % BLOCK4)).unflatten(-1, (-1, BLOCK4))
    exponent = (v.abs().amax(dim=-1).view(torch.int32) >> 23)
    byte = torch.where(exponent == 255, exponent, (exponent - 2).clamp(min=0))
    inverse = torch.where(byte == 254, torch.full_like(byte, 1 << 22), (254 - byte) << 23).view(torch.float32)
    codes = _codes4((v * inverse[..., None]).flatten(-2))
    packed = codes[..., 0::2] | (codes[..., 1::2] << 4)
    packed = packed[..., : (k + 1) // 2]
    byte = byte.to(torch.uint8)
    return (torch.nn.functional.pad(packed, (0, row - packed.shape[-1])),
            torch.nn.functional.pad(byte, (0, scale_row - byte.shape[-1])))


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = {"case": case}
    op = case["op"]
    k, tokens = case["k"], case["tokens"]
    if op in ("norm", "norm_backward"):
        type_ = _type(case["type"])
        s["x"] = _activations(gen, tokens, k, type_)
        s["w"] = (1.0 + 0.2 * torch.randn(k, generator=gen, device="cuda")).to(type_)
        if op == "norm":
            s["r"] = (4.0 * torch.randn(tokens, k, generator=gen, device="cuda")).to(type_) if case["residual"] else None
            s["h"] = torch.empty_like(s["x"]) if case["residual"] else None
            if case["out"] == "e4m3":
                s["q"] = torch.empty(tokens, k, dtype=torch.float8_e4m3fn, device="cuda")
                s["scale"] = torch.empty(tokens, -(-k // BLOCK), device="cuda")
            else:
                s["y"] = torch.empty_like(s["x"])
        else:
            s["dy"] = (0.01 * torch.randn(tokens, k, generator=gen, device="cuda")).to(type_)
            s["dh"] = (0.01 * torch.randn(tokens, k, generator=gen, device="cuda")).to(type_) if case["residual"] else None
            s["dx"] = torch.empty_like(s["x"])
            s["dw"] = torch.empty(k, device="cuda")
        return s
    if op == "linear4":
        m, groups = case["m"], case["groups"]
        s["offsets"], s["most"] = _groups(case, seed, gen)
        s["x"] = _activations(gen, tokens, k, torch.bfloat16)
        s["row"], s["scale_row"] = _up((k + 1) // 2, 16), _up(-(-k // BLOCK4), 16)   # bytes, whole units of 16
        w = torch.randn(groups, m, k, generator=gen, device="cuda") / math.sqrt(k)
        s["w"], s["w_scale"] = _quantized4(w.to(torch.bfloat16), s["row"], s["scale_row"])
        s["q"] = torch.empty(tokens, s["row"], dtype=torch.uint8, device="cuda")
        s["q_scale"] = torch.empty(tokens, s["scale_row"], dtype=torch.uint8, device="cuda")
        s["y"] = torch.empty(tokens, m, dtype=_type(case["out"]), device="cuda")
        return s
    type_, top, groups = _type(case["type"]), case["top"], case["groups"]
    s["expert"] = _chosen(case, gen)
    rows = tokens * top
    if op == "dispatch":
        s["x"] = _activations(gen, tokens, k, type_)
        s["offsets"] = torch.empty(groups + 1, dtype=torch.int32, device="cuda")
        s["place"] = torch.empty(tokens, top, dtype=torch.int32, device="cuda")
        s["y"] = torch.zeros(rows, k, dtype=type_, device="cuda")   # rows that no choice has stay zero
        return s
    s["place"] = _sorted(s["expert"], groups)[1]
    s["weight"] = torch.softmax(torch.randn(tokens, top, generator=gen, device="cuda"), dim=1)
    s["x"] = _activations(gen, rows, k, type_)
    if op == "combine":
        s["y"] = torch.empty(tokens, k, dtype=type_, device="cuda")
    else:
        s["dy"] = (0.01 * torch.randn(tokens, k, generator=gen, device="cuda")).to(type_)
        s["dx"] = torch.zeros(rows, k, dtype=type_, device="cuda")
        s["dweight"] = torch.empty(tokens, top, device="cuda")
    return s


# ---- the plain forms -----------------------------------------------------------

def _sorted(expert, groups):
    """Where each expert's rows begin, and the row of each choice (-1: none)."""
    flat = expert.flatten().long()
    key = torch.where((flat >= 0) & (flat < groups), flat, torch.full_like(flat, groups))
    order = torch.sort(key, stable=True).indices
    place = torch.empty_like(order)
    place[order] = torch.arange(order.numel(), device=order.device)
    counts = (key[:, None] == torch.arange(groups, device=key.device)).sum(dim=0)
    offsets = torch.zeros(groups + 1, dtype=torch.int32, device=key.device)
    offsets[1:] = counts.cumsum(0)
    return offsets, torch.where(key < groups, place, torch.full_like(place, -1)).to(torch.int32).view(expert.shape)


def _values4(packed, byte, k):
    """What codes and scale bytes stand for, in 32 bits."""
    table = torch.tensor(VALUES4 + tuple(-v for v in VALUES4), device=packed.device)
    codes = torch.stack((packed & 15, packed >> 4), dim=-1).flatten(-2)[..., :k]
    return table[codes.long()] * _power(byte).repeat_interleave(BLOCK4, dim=-1)[..., :k]


def _plain(s):
    case = s["case"]
    op = case["op"]
    if op == "norm":
        x = s["x"]
        h = x if s["r"] is None else (x.float() + s["r"].float()).to(x.dtype)
        f = h.float()
        v = f * (1.0 / torch.sqrt(f.square().mean(dim=1, keepdim=True) + EPS)) * s["w"].float()
        first = () if s["r"] is None else (h,)
        if case["out"] == "same":
            return first + (v.to(x.dtype),)
        k = case["k"]
        blocks = torch.nn.functional.pad(v, (0, -k % BLOCK)).unflatten(1, (-1, BLOCK))
        scale = blocks.abs().amax(dim=2).clamp(min=AMAX_FLOOR) / FP8_MAX
        q = (blocks * (1.0 / scale)[:, :, None]).flatten(1)[:, :k].to(torch.float8_e4m3fn)
        return first + (q, scale)
    if op == "norm_backward":
        f, dy, w = s["x"].float(), s["dy"].float(), s["w"].float()
        r = 1.0 / torch.sqrt(f.square().mean(dim=1, keepdim=True) + EPS)
        g = dy * w
        dx = r * (g - f * (r * r * (f * g).mean(dim=1, keepdim=True)))
        if s["dh"] is not None:
            dx = dx + s["dh"].float()
        return dx.to(s["x"].dtype), (dy * (f * r)).sum(dim=0)
    if op == "linear4":
        k, m, tokens = case["k"], case["m"], case["tokens"]
        x = _values4(*_quantized4(s["x"], s["row"], s["scale_row"]), k)
        w = _values4(s["w"], s["w_scale"], k)
        if s["offsets"] is None:
            return (x @ w[0].t()).to(s["y"].dtype)
        row = torch.arange(tokens, device="cuda")
        expert = torch.searchsorted(s["offsets"][1:].contiguous(), row, right=True)
        place = row - s["offsets"][expert]
        v = torch.zeros(case["groups"], s["most"], k, device="cuda")
        v[expert, place] = x
        return (v @ w.transpose(1, 2))[expert, place].to(s["y"].dtype)
    if op == "dispatch":
        offsets, place = _sorted(s["expert"], case["groups"])
        y = torch.zeros_like(s["y"])
        token, choice = torch.nonzero(place >= 0, as_tuple=True)
        y[place[token, choice].long()] = s["x"][token]
        return offsets, place, y
    there = s["place"] >= 0
    at = s["place"].clamp(min=0).long()
    weight = torch.where(there, s["weight"], torch.zeros_like(s["weight"]))
    if op == "combine":
        y = torch.zeros(case["tokens"], case["k"], device="cuda")
        for j in range(case["top"]):
            y += weight[:, j, None] * s["x"][at[:, j]].float()
        return y.to(s["x"].dtype)
    dy = s["dy"].float()
    dx, dweight = torch.zeros_like(s["dx"]), torch.zeros_like(s["dweight"])
    for j in range(case["top"]):
        token = torch.nonzero(there[:, j]).flatten()
        row = at[token, j]
        dx[row] = (weight[token, j, None] * dy[token]).to(dx.dtype)
        dweight[token, j] = (dy[token] * s["x"][row].float()).sum(dim=1)
    return dx, dweight


# ---- the library's calls ---------------------------------------------------------

def _library(s):
    global _handle
    import sgblas_b200 as sg
    if _handle is None:
        _handle = sg.Handle()
    h, case = _handle, s["case"]
    op, k, tokens = case["op"], case["k"], case["tokens"]
    code = {"bf16": sg.SGBLAS_TYPE_BF16, "fp32": sg.SGBLAS_TYPE_FP32}
    if op == "norm":
        first = () if s["r"] is None else (s["h"],)
        if case["out"] == "same":
            h.rms_norm(k, tokens, code[case["type"]], s["x"], k, s["r"], k, s["w"], EPS, s["h"], k, y=s["y"], ldy=k)
            return first + (s["y"],)
        h.rms_norm(k, tokens, code[case["type"]], s["x"], k, s["r"], k, s["w"], EPS, s["h"], k, q=s["q"], ldq=k,
                   scale=s["scale"], ldscale=-(-k // BLOCK))
        return first + (s["q"], s["scale"])
    if op == "norm_backward":
        h.rms_norm_backward(k, tokens, code[case["type"]], s["dy"], k, s["x"], k, s["w"], EPS, s["dh"], k, s["dx"], k, 0.0, s["dw"])
        return s["dx"], s["dw"]
    if op == "linear4":
        m, groups, out = case["m"], case["groups"], code[case["out"]]
        row, scale_row = s["row"], s["scale_row"]
        h.quantize_fp4(k, tokens, s["x"], sg.SGBLAS_TYPE_BF16, k, s["q"], row, s["q_scale"], scale_row)
        if groups == 1:
            h.gemm_fp4(m, tokens, k, s["w"], row, s["w_scale"], scale_row, s["q"], row, s["q_scale"], scale_row, s["y"], out, m)
        else:
            h.grouped_gemm_fp4(m, tokens, k, groups, s["offsets"], s["w"], row, m * row, s["w_scale"], scale_row, m * scale_row,
                               s["q"], row, s["q_scale"], scale_row, s["y"], out, m)
        return s["y"]
    top, groups, type_ = case["top"], case["groups"], code[case["type"]]
    rows = tokens * top
    if op == "dispatch":
        h.sort_tokens(tokens, top, groups, s["expert"], s["offsets"], s["place"])
        h.scatter_tokens(k, tokens, top, rows, s["place"], None, s["x"], type_, k, s["y"], k)
        return s["offsets"], s["place"], s["y"]
    if op == "combine":
        h.gather_tokens(k, tokens, top, rows, s["place"], s["weight"], s["x"], type_, k, s["y"], k)
        return s["y"]
    h.gather_tokens_backward(k, tokens, top, rows, s["place"], s["weight"], s["dy"], type_, k, s["x"], k, s["dx"], k, s["dweight"])
    return s["dx"], s["dweight"]


def run(state):
    return _library(state) if own else _plain(state)


# ---- what cannot be left out -----------------------------------------------------

def work(case):
    op, k, t = case["op"], case["k"], case["tokens"]
    size = {"bf16": 2, "fp32": 4}
    if op == "norm":
        e = size[case["type"]]
        out = 1 + 4 / BLOCK if case["out"] == "e4m3" else e
        return {"bytes": t * k * (e * (3 if case["residual"] else 1) + out) + e * k, "flops": 6 * t * k}
    if op == "norm_backward":
        e = size[case["type"]]
        return {"bytes": t * k * e * (4 if case["residual"] else 3) + (e + 4) * k, "flops": 12 * t * k}
    if op == "linear4":
        groups, m = case["groups"], case["m"]
        reached = sum(1.0 - (1.0 - p) ** t for p in _shares(groups))   # experts that have a token
        return {"bytes": 2 * t * k + reached * m * k * (0.5 + 1 / BLOCK4) + size[case["out"]] * t * m, "flops": 2 * t * m * k}
    e, top = size[case["type"]], case["top"]
    live = t - t // 32   # the rest is padding
    if op == "dispatch":
        return {"bytes": live * k * e * (1 + top) + 8 * t * top, "flops": 0}
    if op == "combine":
        return {"bytes": (live * top + t) * k * e + 8 * t * top, "flops": 2 * live * top * k}
    return {"bytes": live * k * e * (1 + 2 * top) + 12 * t * top, "flops": 3 * live * top * k}


# ---- the definitions in 64 bits -----------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    op, k, tokens = case["op"], case["k"], case["tokens"]
    if op == "norm":
        h = s["x"].double()
        if s["r"] is not None:
            h = (s["x"].double() + s["r"].double()).to(s["x"].dtype).double()   # held in the type
        v = s["w"].double() * h / (torch.linalg.vector_norm(h, dim=1, keepdim=True) ** 2 / k + EPS) ** 0.5
        first = () if s["r"] is None else (h,)
        if case["out"] == "same":
            return first + (v,)
        q, scale = torch.empty_like(v), torch.empty(tokens, -(-k // BLOCK), dtype=torch.float64, device="cuda")
        for j in range(0, k, BLOCK):
            part = v[:, j:j + BLOCK]
            scale[:, j // BLOCK] = part.abs().amax(dim=1).clamp(min=AMAX_FLOOR) / FP8_MAX
            q[:, j:j + BLOCK] = part / scale[:, j // BLOCK, None]
        return first + (q, scale)   # the values before their rounding to 8 bits
    if op == "norm_backward":
        h, dy, w = s["x"].double(), s["dy"].double(), s["w"].double()
        length = (torch.linalg.vector_norm(h, dim=1, keepdim=True) ** 2 / k + EPS) ** 0.5
        unit = h / length
        g = w * dy
        dx = (g - unit * torch.einsum("tk,tk->t", unit, g)[:, None] / k) / length
        if s["dh"] is not None:
            dx += s["dh"].double()
        return dx, torch.einsum("tk,tk->k", unit, dy)
    if op == "linear4":
        m, groups = case["m"], case["groups"]
        step = torch.tensor([1, 2, 4], dtype=torch.float64, device="cuda")
        # Tokens by the definition: a block's power of two, then the grid's spacing at each value.
        x = torch.nn.functional.pad(s["x"].double(), (0, -k % BLOCK4)).unflatten(1, (-1, BLOCK4))
        power = torch.exp2(torch.frexp(x.abs().amax(dim=2, keepdim=True)).exponent.double() - 3)
        v = (x / power).clamp(-6.0, 6.0)
        gap = 0.5 * step[(v.abs() >= 2).long() + (v.abs() >= 4).long()]
        x = (torch.round(v / gap) * gap * power).flatten(1)[:, :k]
        value = torch.tensor(VALUES4, dtype=torch.float64, device="cuda")
        ends = [0, tokens] if s["offsets"] is None else s["offsets"].tolist()
        y = torch.zeros(tokens, m, dtype=torch.float64, device="cuda")
        for e in range(groups):
            if ends[e] == ends[e + 1]:
                continue
            w = torch.empty(m, 2 * s["row"], dtype=torch.float64, device="cuda")
            for half, code in enumerate((s["w"][e] % 16, s["w"][e] // 16)):
                w[:, half::2] = value[(code % 8).long()] * torch.where(code < 8, 1.0, -1.0)
            w = w[:, :k] * torch.exp2(s["w_scale"][e].double() - 127)[:, torch.arange(k, device="cuda") // BLOCK4]
            y[ends[e]:ends[e + 1]] = x[ends[e]:ends[e + 1]] @ w.mT
        return y
    top, groups = case["top"], case["groups"]
    if op == "dispatch":
        expert = s["expert"].tolist()
        lists = [[] for _ in range(groups)]
        for t, row in enumerate(expert):
            for j, e in enumerate(row):
                if 0 <= e < groups:
                    lists[e].append((t, j))
        offsets, order = [0], []
        for part in lists:
            order += part
            offsets.append(len(order))
        place = [[-1] * top for _ in range(tokens)]
        for at, (t, j) in enumerate(order):
            place[t][j] = at
        y = torch.zeros(tokens * top, k, dtype=torch.float64, device="cuda")
        if order:
            y[:len(order)] = s["x"].double()[torch.tensor([t for t, _ in order], device="cuda")]
        return (torch.tensor(offsets, dtype=torch.int32, device="cuda"), torch.tensor(place, dtype=torch.int32, device="cuda"), y)
    place, weight = s["place"].long(), s["weight"].double()
    token = torch.arange(tokens, device="cuda")[:, None].expand(tokens, top)[place >= 0]
    row, factor = place[place >= 0], weight[place >= 0][:, None]
    if op == "combine":
        y = torch.zeros(tokens, k, dtype=torch.float64, device="cuda")
        return y.index_add_(0, token, factor * s["x"].double()[row])
    dx = torch.zeros(tokens * top, k, dtype=torch.float64, device="cuda")
    dx[row] = factor * s["dy"].double()[token]
    dweight = torch.zeros(tokens, top, dtype=torch.float64, device="cuda")
    dweight[place >= 0] = torch.einsum("rk,rk->r", s["dy"].double()[token], s["x"].double()[row])
    return dx, dweight
