"""Dense layers whose rows are held in eight bits: what their speed and exactness are measured on.

Inference keeps the rows between a norm and a product as whole numbers with one scale a row, and weights as whole numbers
with one scale an output channel:

  norm      (x + r, the norm of it in 8 bits), LayerNorm or RMSNorm:  scale = max |y| / 127,  code = y / scale to the nearest
  product   y = sx sw (codes of x) (codes of w)^T + b, GELU behind it on request
  mlp       both layers of an MLP behind such rows, the hidden layer's (fp16) rows in 8 bits again

Training keeps what the backward pass of a layer reads of its input in 8 bits, in groups of 16 numbers of a row with a scale of
four significant bits each, the smallest multiple of 2^-24 of them with 127 scales reaching the group's largest number:

  kept_linear   y = x W^T + b;  dx = dy W,  dW = dy^T x',  db = the sum of dy, x' what the codes of x stand for
  kept_mlp      h = x W1^T + b1, y = GELU(h) W2^T + b2;  dh = (dy W2) GELU'(h'),  dW2 = dy^T GELU(h'),  dx = dh W1,  dW1 = dh^T x'

Where `own` is true, run() calls the framework; otherwise it computes the same in elementary operations.
"""
import math

import torch

own = False

GROUP = 16
# channels of the levels of Swin3D-S and Swin3D-L
WIDTHS = (48, 80, 96, 160, 192, 320, 384, 640)


def listed():
    return [
        # the norm in front of a block's qkv at the deepest level of one room: a call of a few microseconds
        dict(name="norm_deepest", kind="norm", rows=811, channels=384, norm="layer", residual="fp16"),
        # ... at the first level of Swin3D-S on a room of 200,000 voxels
        dict(name="norm_first", kind="norm", rows=199327, channels=48, norm="layer", residual="fp16"),
        # a network with root-mean-square norms, second level of Swin3D-L's widths on two large rooms, residual in fp32
        dict(name="norm_rms_large", kind="norm", rows=149993, channels=160, norm="rms", residual="fp32"),
        # qkv at the deepest level of Swin3D-L on a small scan: a handful of tiles
        dict(name="product_deepest", kind="product", rows=390, inputs=640, outputs=1920, gelu=False),
        # fc1 with GELU at the first level of Swin3D-S: bound by its rows, K no multiple of 32
        dict(name="product_first", kind="product", rows=199327, inputs=48, outputs=192, gelu=True),
        # qkv at the second level of Swin3D-L, two large rooms
        dict(name="product_second_large", kind="product", rows=149993, inputs=160, outputs=480, gelu=False),
        # fc2 at the third level of Swin3D-L, two large rooms: the longest sums on many rows
        dict(name="product_third_large", kind="product", rows=37499, inputs=1280, outputs=320, gelu=False),
        # a block's MLP at inference, third level of Swin3D-S on a room
        dict(name="mlp_third", kind="mlp", rows=12421, channels=192, hidden=768),
        # the training pass of a block's qkv at the deepest level of Swin3D-S
        dict(name="kept_linear_deepest", kind="kept_linear", rows=811, inputs=384, outputs=1152),
        # ... at the first level
        dict(name="kept_linear_first", kind="kept_linear", rows=199327, inputs=48, outputs=144),
        # the training pass of a block's MLP, third level of Swin3D-S
        dict(name="kept_mlp_third", kind="kept_mlp", rows=12421, channels=192, hidden=768),
        # ... at the second level of Swin3D-L, two large rooms: the heaviest MLP there is
        dict(name="kept_mlp_second_large", kind="kept_mlp", rows=149993, channels=160, hidden=640),
    ]


def draw(rng):
    def cost(case):
        done = work(case)
        return max(done["bytes"], done["flops"] / 100)      # (products in 16 bits: some hundred operations a byte)

    most = max(cost(case) for case in listed())
    while True:
        case = _drawn(rng)
        if cost(case) <= most:
            return case


def _drawn(rng):
    def between(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(("norm", "norm", "product", "product", "product", "mlp", "kept_linear", "kept_linear", "kept_mlp", "kept_mlp"))
    if kind == "norm":
        channels = rng.choice((rng.choice(WIDTHS), 4 * rng.randint(1, 256), 4 * rng.randint(257, 640)))
        return dict(kind=kind, rows=between(1, 24_000_000 // channels), channels=channels, norm=rng.choice(("layer", "rms")),
                    residual=rng.choice(("fp16", "fp16", "fp32", "none")))
    width = rng.choice((rng.choice(WIDTHS), rng.choice(WIDTHS), 16 * rng.randint(1, 40)))
    if kind == "product":
        inputs, outputs = rng.choice(((width, 3 * width), (width, width), (width, 4 * width), (4 * width, width), (width, 8 * rng.randint(1, 200))))
        return dict(kind=kind, rows=between(1, min(600_000, 80_000_000 // (inputs + outputs))), inputs=inputs, outputs=outputs,
                    gelu=rng.random() < 0.3)
    if kind == "kept_linear":
        inputs, outputs = rng.choice(((width, 3 * width), (width, width), (width, 4 * width), (4 * width, width)))
        return dict(kind=kind, rows=between(1, min(300_000, 60_000_000 // (inputs + outputs))), inputs=inputs, outputs=outputs)
    return dict(kind=kind, rows=between(1, min(200_000, 20_000_000 // width)), channels=width, hidden=rng.choice((4, 4, 2)) * width)


def _rounded_to_8_bits(values):
    """(codes, scales) of fp32 rows, as a program that quantizes its weights has them."""
    scales = values.abs().amax(1) / 127
    codes = torch.round(values / scales.clamp(min=1e-30).unsqueeze(1)).to(torch.int8)
    return codes, scales


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed * 1_000_003 + 17)

    def normal(*shape):
        return torch.randn(shape, device="cuda", generator=gen)

    m, kind = case["rows"], case["kind"]
    state = dict(kind=kind)
    if kind == "norm":
        c = case["channels"]
        # a residual stream: channels of different spread and a few that stand out
        spread = torch.exp(0.7 * normal(c)) * torch.where(torch.rand(c, device="cuda", generator=gen) < 0.03, 8.0, 1.0)
        state["x"] = normal(m, c) * spread + 0.5 * normal(c)
        state["residual"] = None if case["residual"] == "none" else normal(m, c) * 0.5
        if case["residual"] == "fp16":
            state["residual"] = state["residual"].half()
        norm = (torch.nn.LayerNorm(c, device="cuda") if case["norm"] == "layer" else torch.nn.RMSNorm(c, eps=1e-6, device="cuda"))
        norm.weight.data.copy_(1 + 0.2 * normal(c))
        if case["norm"] == "layer":
            norm.bias.data.copy_(0.1 * normal(c))
        state["norm"] = norm.requires_grad_(False)
        return state
    if kind in ("product", "mlp"):
        k = case["inputs"] if kind == "product" else case["channels"]
        state["codes"], state["scales"] = _rounded_to_8_bits(normal(m, k) * torch.exp(0.3 * normal(m, 1)))
        sizes = [(case["outputs"], k)] if kind == "product" else [(case["hidden"], k), (k, case["hidden"])]
        state["weights"] = [_rounded_to_8_bits(normal(*size) / math.sqrt(size[1])) for size in sizes]
        state["biases"] = [0.1 * normal(size[0]) for size in sizes]
        state["gelu"] = case.get("gelu", False)
        return state
    c = case["inputs"] if kind == "kept_linear" else case["channels"]
    sizes = [(case["outputs"], c)] if kind == "kept_linear" else [(case["hidden"], c), (c, case["hidden"])]
    # a linear layer has its parameters in fp32, the MLP in fp16 with fp32 copies in the optimizer: either is a program's choice
    dtype = torch.float32 if kind == "kept_linear" else torch.float16
    state["x"] = (normal(m, c) * torch.exp(0.5 * normal(c))).half().requires_grad_()
    state["weights"] = [(normal(*size) / math.sqrt(size[1])).to(dtype).requires_grad_() for size in sizes]
    state["biases"] = [(0.1 * normal(size[0])).to(dtype).requires_grad_() for size in sizes]
    state["dy"] = (normal(m, sizes[-1][0]) * torch.exp(0.5 * normal(m, 1))).half()
    return state


# ---- the framework's calls ----------------------------------------------------------------------------------------------

def _run_own(state):
    from swin3d_amd import eight_bits

    kind = state["kind"]
    if kind == "norm":
        summed, rows = eight_bits.add_norm_int8(state["x"], state["residual"], state["norm"])
        return {"sum": summed, "rows": rows.values(torch.float16)}
    if kind in ("product", "mlp"):
        rows = eight_bits.Int8Rows(state["codes"], state["scales"])
        weights = [eight_bits.Int8Rows(*w) for w in state["weights"]]
        if kind == "product":
            return {"y": eight_bits.linear_int8(rows, weights[0], state["biases"][0], gelu=state["gelu"])}
        return {"y": eight_bits.mlp_int8(rows, weights[0], state["biases"][0], weights[1], state["biases"][1])}
    x, weights, biases = state["x"], state["weights"], state["biases"]
    if kind == "kept_linear":
        y = eight_bits.checkpointed_linear(x, weights[0], biases[0])
        dx, dw, db = torch.autograd.grad(y, (x, weights[0], biases[0]), state["dy"])
        return {"y": y, "dx": dx, "dw": dw, "db": db}
    y = eight_bits.checkpointed_mlp(x, weights[0], biases[0], weights[1], biases[1])
    dx, dw1, db1, dw2, db2 = torch.autograd.grad(y, (x, weights[0], biases[0], weights[1], biases[1]), state["dy"])
    return {"y": y, "dx": dx, "dw1": dw1, "db1": db1, "dw2": dw2, "db2": db2}


# ---- plain forms ----------------------------------------------------------------------------------------------------------

def _gelu(x):
    return 0.5 * x * (1 + torch.erf(x * math.sqrt(0.5)))


def _gelu_slope(x):
    return 0.5 * (1 + torch.erf(x * math.sqrt(0.5))) + x * torch.exp(-0.5 * x * x) / math.sqrt(2 * math.pi)


def _whole(y):
    """(codes as fp32 numbers, scales) of fp32 rows"""
    largest = y.abs().amax(1, keepdim=True)
    codes = torch.round(127 * y / largest.clamp(min=1e-30))
    return codes, largest / 127


def _kept(x):
    """What the checkpoint of fp16 rows stands for, in fp32."""
    m, c = x.shape
    groups = x.float().view(m, c // GROUP, GROUP)
    # (64 bits: a quotient next to a border of the scales' four bits)
    least = groups.abs().amax(2, keepdim=True).double() / 127
    _, exponent = torch.frexp(least)
    unit = ((exponent - 4).clamp(min=-24).long() + 1023 << 52).view(torch.float64)      # 2 to the power of that
    scale = (torch.ceil(least / unit) * unit).float()
    codes = torch.round(groups / torch.where(scale > 0, scale, torch.ones_like(scale)))
    return (codes * scale).view(m, c)


def _run_plain(state):
    kind = state["kind"]
    if kind == "norm":
        norm, x = state["norm"], state["x"]
        summed = x if state["residual"] is None else x + state["residual"].float()
        if isinstance(norm, torch.nn.LayerNorm):
            centred = summed - summed.mean(1, keepdim=True)
            y = centred * torch.rsqrt(centred.square().mean(1, keepdim=True) + norm.eps) * norm.weight + norm.bias
        else:
            y = summed * torch.rsqrt(summed.square().mean(1, keepdim=True) + norm.eps) * norm.weight
        codes, scales = _whole(y)
        return {"sum": summed, "rows": (codes * scales).half()}
    if kind in ("product", "mlp"):
        codes, scales = state["codes"].float(), state["scales"].unsqueeze(1)
        (w, sw), b = state["weights"][0], state["biases"][0]
        y = codes @ w.float().t() * (scales * sw) + b
        if kind == "product":
            return {"y": (_gelu(y) if state["gelu"] else y).half()}
        codes, scales = _whole(_gelu(y).half().float())
        (w, sw), b = state["weights"][1], state["biases"][1]
        return {"y": (codes @ w.float().t() * (scales * sw) + b).half()}
    x, dy = state["x"].detach(), state["dy"].float()
    weights, biases = state["weights"], state["biases"]
    w1, b1 = weights[0].detach().half().float(), biases[0].detach().half().float()
    h = x.float() @ w1.t() + b1
    if kind == "kept_linear":
        return {"y": h.half(), "dx": (dy @ w1).half(), "dw": dy.t() @ _kept(x), "db": dy.sum(0)}
    h = h.half()
    w2, b2 = weights[1].detach().float(), biases[1].detach().float()
    y = _gelu(h.float()) @ w2.t() + b2
    kept_h = _kept(h)
    dh = (dy @ w2) * _gelu_slope(kept_h)
    return {"y": y.half(), "dx": (dh @ w1).half(), "dw1": (dh.t() @ _kept(x)).half(), "db1": dh.sum(0).half(),
            "dw2": (dy.t() @ _gelu(kept_h)).half(), "db2": dy.sum(0).half()}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- in 64 bits -----------------------------------------------------------------------------------------------------------

def _exact_gelu(x):
    return x * torch.special.ndtr(x)


def _exact_codes(y):
    """Rows y in whole steps of a 127th of their largest number, and the steps."""
    step = torch.linalg.vector_norm(y, ord=math.inf, dim=1, keepdim=True) / 127
    whole = torch.where(step > 0, torch.round(y / torch.where(step > 0, step, 1.0)), 0.0)
    return whole, step


def _exact_kept(x):
    """Rows of fp16 numbers in whole steps of their groups' scales: every scale there is, in ascending order, and the first that suffices."""
    fours = torch.arange(1, 16, dtype=torch.float64, device=x.device)
    scales = torch.unique(torch.cat([fours * 2.0 ** e for e in range(-24, 8)]))
    groups = x.double().reshape(-1, GROUP)
    step = scales[torch.searchsorted(scales * 127, torch.linalg.vector_norm(groups, ord=math.inf, dim=1))].unsqueeze(1)
    return (torch.round(groups / step) * step).view(x.shape)


def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    if kind == "norm":
        norm = state["norm"]
        summed = state["x"].double() if state["residual"] is None else torch.add(state["x"].double(), state["residual"].double())
        if case["norm"] == "layer":
            variance, mean = torch.var_mean(summed, dim=1, correction=0, keepdim=True)
            y = torch.addcmul(norm.bias.double(), (summed - mean) / torch.sqrt(variance + norm.eps), norm.weight.double())
        else:
            y = summed / torch.sqrt(torch.linalg.vector_norm(summed, dim=1, keepdim=True) ** 2 / summed.shape[1] + norm.eps) * norm.weight.double()
        whole, step = _exact_codes(y)
        return {"sum": summed, "rows": whole * step}
    if kind in ("product", "mlp"):
        rows = state["codes"].double() * state["scales"].double().unsqueeze(1)
        for i, ((w, sw), b) in enumerate(zip(state["weights"], state["biases"])):
            if i == 1:
                whole, step = _exact_codes(rows.half().double())
                rows = whole * step
            rows = torch.addmm(b.double(), rows, (w.double() * sw.double().unsqueeze(1)).t())
            if i == 0 and (kind == "mlp" or case["gelu"]):
                rows = _exact_gelu(rows)
        return {"y": rows}
    x, dy = state["x"].detach(), state["dy"].double()
    w = [t.detach().half().double() for t in state["weights"]]
    b = [t.detach().half().double() for t in state["biases"]]
    if kind == "kept_linear":
        return {"y": torch.addmm(b[0], x.double(), w[0].t()), "dx": torch.mm(dy, w[0]), "dw": torch.mm(_exact_kept(x).t(), dy).t(),
                "db": torch.sum(dy, 0)}
    h = torch.addmm(b[0], x.double(), w[0].t()).half()
    kept = _exact_kept(h)
    slope = torch.special.ndtr(kept) + kept * torch.exp(-kept * kept / 2) / math.sqrt(2 * math.pi)
    dh = torch.mm(dy, w[1]) * slope
    return {"y": torch.addmm(b[1], _exact_gelu(h.double()), w[1].t()), "dx": torch.mm(dh, w[0]), "dw1": torch.mm(dh.t(), _exact_kept(x)),
            "db1": torch.sum(dh, 0), "dw2": torch.mm(dy.t(), _exact_gelu(kept)), "db2": torch.sum(dy, 0)}


def work(case):
    m, kind = case["rows"], case["kind"]
    if kind == "norm":
        c = case["channels"]
        residual = {"fp16": 2, "fp32": 4, "none": 0}[case["residual"]]
        summed = 0 if case["residual"] == "none" else 4
        # the stream in, the sum out, and the values of the rows, as they come back here
        return {"bytes": m * c * (4 + residual + summed + 2) + 8 * c, "flops": 12 * m * c}
    if kind == "product":
        k, n = case["inputs"], case["outputs"]
        return {"bytes": m * k + n * k + 4 * (m + 2 * n) + 2 * m * n, "flops": 2 * m * n * k}
    if kind == "mlp":
        c, hidden = case["channels"], case["hidden"]
        return {"bytes": m * (c + 4) + 2 * c * hidden + 8 * (c + hidden) + 2 * m * c, "flops": 4 * m * c * hidden}
    kept = 1 + 1 / GROUP
    if kind == "kept_linear":
        k, n = case["inputs"], case["outputs"]
        # x, dy and the parameters in, y, dx and the gradients out, the checkpoint out and in
        return {"bytes": m * (2 * k + 2 * n) * 2 + 2 * kept * m * k + 2 * 4 * (n * k + n), "flops": 6 * m * n * k}
    c, hidden = case["channels"], case["hidden"]
    return {"bytes": m * 4 * c * 2 + 2 * kept * m * (c + hidden) + 2 * 2 * (2 * c * hidden + c + hidden), "flops": 12 * m * c * hidden}
