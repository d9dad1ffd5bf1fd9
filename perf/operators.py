"""Operators of 8-bit products, with their plain forms: the norm before a product, the gate and the plain rows that a
product reads (all leave 8-bit integers with one scale a row), and the product itself.

Widths and row counts are those of the dense decoders that ``bench.py`` runs (width 4,096 with 6,144 q/k/v rows, 14,336 hidden
units and 32 x 128 heads; width 5,120 with 25,600 hidden units and 64 x 128 heads): 1 to 64 rows are decode steps, hundreds to
thousands are prompts.
"""
import math

import torch

own = False  # True: the framework's kernels; False: the plain forms below

DEVICE = "cuda"
TYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
TINY = 2.0 ** -126  # the smallest scale: a row of zeros has codes 0 and this scale
EPS = 1e-5


def listed():
    return [
        # the second norm of a layer in a decode step of one sequence: latency
        {"name": "norm-1x4096", "op": "norm", "rows": 1, "width": 4096, "add": "float32", "weight": "bfloat16"},
        # the same in a prompt of ordinary length, what is added in 16 bits
        {"name": "norm-2048x4096", "op": "norm", "rows": 2048, "width": 4096, "add": "bfloat16", "weight": "bfloat16"},
        # several long prompts in one step, an odd number of tokens, the wider decoder
        {"name": "norm-8191x5120", "op": "norm", "rows": 8191, "width": 5120, "add": "float32", "weight": "float32"},
        # the gate of a decode step of eight sequences
        {"name": "gate-8x14336", "op": "gate", "rows": 8, "width": 14336, "act": "silu", "type": "bfloat16"},
        # the gate of a prompt, the wider decoder, the other activation
        {"name": "gate-2000x25600", "op": "gate", "rows": 2000, "width": 25600, "act": "gelu_tanh", "type": "bfloat16"},
        # attention's output before the output product: 64 sequences, and a prompt
        {"name": "rows-64x4096", "op": "rows", "rows": 64, "width": 4096, "type": "bfloat16"},
        {"name": "rows-4096x8192", "op": "rows", "rows": 4096, "width": 8192, "type": "bfloat16"},
        # q, k and v of one sequence's token: the smallest product
        {"name": "product-1x6144x4096", "op": "product", "rows": 1, "outputs": 6144, "inputs": 4096, "type": "float32",
         "bias": False},
        # the feed-forward's last product for eight sequences: a long sum
        {"name": "product-8x4096x14336", "op": "product", "rows": 8, "outputs": 4096, "inputs": 14336, "type": "float32",
         "bias": False},
        # gate and up rows for 64 sequences
        {"name": "product-64x28672x4096", "op": "product", "rows": 64, "outputs": 28672, "inputs": 4096, "type": "bfloat16",
         "bias": False},
        # a short prompt, nothing a multiple of anything, with a bias
        {"name": "product-333x5003x1999", "op": "product", "rows": 333, "outputs": 5003, "inputs": 1999, "type": "float32",
         "bias": True},
        # gate and up rows of a long prompt: the tensor cores' rate
        {"name": "product-8192x28672x4096", "op": "product", "rows": 8192, "outputs": 28672, "inputs": 4096,
         "type": "bfloat16", "bias": False},
    ]


def draw(rng):
    def spread(lo, hi):
        n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
        step = rng.choice([1, 1, 4, 16, 128])
        return min(hi, max(lo, n // step * step))

    op = rng.choice(["norm", "gate", "rows", "product", "product", "product"])
    if op == "product":
        while True:
            rows, outputs, inputs = spread(1, 8192), spread(64, 28672), spread(64, 25600)
            if rows * outputs * inputs <= 8192 * 28672 * 4096:
                return {"op": op, "rows": rows, "outputs": outputs, "inputs": inputs,
                        "type": rng.choice(["bfloat16", "float32"]), "bias": rng.random() < 0.5}
    rows = spread(1, 8191)
    if op == "norm":
        return {"op": op, "rows": rows, "width": spread(64, 5120), "add": rng.choice(["bfloat16", "float32", "none"]),
                "weight": rng.choice(["bfloat16", "float32"])}
    if op == "gate":
        return {"op": op, "rows": min(rows, 2000), "width": spread(64, 25600), "act": rng.choice(["silu", "gelu_tanh"]),
                "type": rng.choice(["bfloat16", "float32"])}
    return {"op": op, "rows": min(rows, 4096), "width": spread(64, 8192), "type": rng.choice(["bfloat16", "float32"])}


def _room(rows, width):
    """An int8 matrix whose rows begin every 16 bytes, as the product's copies ask for."""
    return torch.empty((rows, -(-width // 16) * 16), dtype=torch.int8, device=DEVICE)[:, :width]


def _coded(x):
    """x as 8-bit integers with a scale a row: what a program holds of its weights, or got from the operators before."""
    scales = (x.abs().amax(dim=1) / 127).clamp_min(TINY)
    codes = _room(*x.shape)
    codes.copy_((x / scales[:, None]).round_())
    return codes, scales


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=DEVICE)

    state = {"case": case}
    rows = case["rows"]
    if case["op"] == "product":
        outputs, inputs = case["outputs"], case["inputs"]
        # some input channels are several times the others, as in a decoder's stream
        x = normal(rows, inputs) * (1 + 3 * (torch.rand(inputs, generator=gen, device=DEVICE) < 0.02))
        state["codes"], state["scales"] = _coded(x)
        state["weight"], state["weight_scales"] = _coded(normal(outputs, inputs) * 0.02)
        state["bias"] = normal(outputs) * 0.1 if case["bias"] else None
        state["out"] = torch.empty((rows, outputs), dtype=TYPES[case["type"]], device=DEVICE)
        return state
    width = case["width"]
    if case["op"] == "norm":
        state["x"] = normal(rows, width) * (1 + 3 * (torch.rand(width, generator=gen, device=DEVICE) < 0.02))
        state["add"] = None if case["add"] == "none" else (normal(rows, width) * 0.3).to(TYPES[case["add"]])
        state["weight"] = (1 + 0.1 * normal(width)).to(TYPES[case["weight"]])
        state["sum"] = torch.empty((rows, width), device=DEVICE)
    elif case["op"] == "gate":
        state["gate_up"] = normal(rows, 2 * width).to(TYPES[case["type"]])
    else:
        state["x"] = normal(rows, width).to(TYPES[case["type"]])
    state["codes"] = _room(rows, width)
    state["scales"] = torch.empty(rows, device=DEVICE)
    state["values"] = torch.empty((rows, width), dtype=torch.bfloat16, device=DEVICE)
    return state


def _plain_coded(y):
    """The values that y's 8-bit integers stand for, in the 16 bits of the decoder's activations, and the scales."""
    scales = (y.abs().amax(dim=1) / 127).clamp_min(TINY)
    codes = (y / scales[:, None]).round()
    return (codes * scales[:, None]).to(torch.bfloat16), scales


def _plain(state):
    case = state["case"]
    if case["op"] == "product":
        out = state["codes"].float() @ state["weight"].float().t()
        out = out * state["scales"][:, None] * state["weight_scales"]
        if state["bias"] is not None:
            out = out + state["bias"]
        return out.to(TYPES[case["type"]])
    if case["op"] == "norm":
        s = state["x"] if state["add"] is None else state["x"] + state["add"].float()
        y = s / torch.sqrt((s * s).mean(dim=1, keepdim=True) + EPS) * state["weight"].float()
        return (s, *_plain_coded(y))
    if case["op"] == "gate":
        g, u = state["gate_up"].float().split(case["width"], dim=1)
        if case["act"] == "silu":
            return _plain_coded(g / (1 + torch.exp(-g)) * u)
        return _plain_coded(0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g * g * g))) * u)
    return _plain_coded(state["x"].float())


def _own(state):
    from xeno_rt_b200.csrc import ops

    case = state["case"]
    if case["op"] == "product":
        ops.gemm_int8(state["out"], state["codes"], state["scales"], state["weight"], state["weight_scales"],
                      bias=state["bias"])
        return state["out"]
    codes, scales, values = state["codes"], state["scales"], state["values"]
    if case["op"] == "norm":
        ops.rmsnorm_int8(codes, scales, state["x"], state["weight"], EPS, add=state["add"],
                         out=None if state["add"] is None else state["sum"])
    elif case["op"] == "gate":
        ops.swiglu_int8(codes, scales, state["gate_up"], case["act"])
    else:
        ops.quantize_rows(codes, scales, state["x"])
    torch.mul(codes, scales[:, None], out=values)
    if case["op"] == "norm":
        return state["x"] if state["add"] is None else state["sum"], values, scales
    return values, scales


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    rows = case["rows"]
    if case["op"] == "product":
        outputs, inputs = case["outputs"], case["inputs"]
        out_bytes = 2 if case["type"] == "bfloat16" else 4
        return {"bytes": (rows + outputs) * (inputs + 4) + rows * outputs * out_bytes + (4 * outputs if case["bias"] else 0),
                "flops": 2 * rows * outputs * inputs}
    width = case["width"]
    if case["op"] == "norm":
        added = {"none": 0, "bfloat16": 2 + 4, "float32": 4 + 4}[case["add"]]  # what is added, and the sum written
        return {"bytes": rows * (width * (4 + added + 1) + 4) + width * (2 if case["weight"] == "bfloat16" else 4),
                "flops": 8 * rows * width}
    size = 2 if case["type"] == "bfloat16" else 4
    inputs = 2 * width if case["op"] == "gate" else width
    return {"bytes": rows * (inputs * size + width + 4), "flops": (12 if case["op"] == "gate" else 4) * rows * width}


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "product":
        # whole numbers below 2^53: the sum is exact
        total = torch.matmul(state["codes"].double(), state["weight"].double().T)
        total *= torch.outer(state["scales"].double(), state["weight_scales"].double())
        return total if state["bias"] is None else total + state["bias"].double()
    if case["op"] == "norm":
        first = state["x"].double()
        if state["add"] is not None:
            first = first + state["add"].double()
        rms = (first.square().sum(dim=1) / case["width"] + EPS).sqrt()
        value = first * state["weight"].double() / rms[:, None]
    elif case["op"] == "gate":
        both = state["gate_up"].double()
        gate, up = both[:, :case["width"]], both[:, case["width"]:]
        if case["act"] == "silu":
            value = gate * torch.sigmoid(gate) * up
        else:
            value = gate * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (gate + 0.044715 * gate ** 3)) * up
    else:
        value = state["x"].double()
    step = torch.clamp(value.abs().max(dim=1).values / 127, min=TINY)
    coded = torch.round(value / step[:, None]) * step[:, None]
    return (first, coded, step) if case["op"] == "norm" else (coded, step)
