"""The 8-bit operators that this engine is timed on: a norm and a quantisation whose outputs are rows of 8-bit integers with a scale
each, and the matrix product of such rows.

``listed()`` names the cases, ``draw(rng)`` gives further ones of the same ranges.  A case is one call of one operator:

* ``"norm"``: ``kernels.rmsnorm_int8``, the stream [tokens, width] takes a sublayer's output and is normed for the next product;
* ``"quantize"``: ``kernels.quantize_int8``, the rows of a matrix: activations ahead of a product, or a weight when it is loaded;
* ``"product"``: ``kernels.gemm_int8``, rows by weight rows, in bfloat16 or float32, plain or with the gated activation in its epilogue.

With ``own`` false the same results are formed from elementary torch operations.  The layer sizes are those of the benchmark's Qwen3
shapes (width 4,096 with 32 heads and a feed-forward of 12,288; width 5,120 with 17,408), beside odd ones.  What is held in 8 bits comes
back as the values it stands for, code times scale in float32.  ``exact`` restates the operators in 64-bit arithmetic.
"""
import torch

own = False

EPS = 1e-6
TYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
DEVICE = "cuda"


def listed():
    return [
        # one user's reply: the norm ahead of a layer's first product
        dict(name="norm_decode_1", op="norm", tokens=1, width=4096, delta="bfloat16"),
        # a full batch of replies, the sublayer's output in 32 bits
        dict(name="norm_batch_64", op="norm", tokens=64, width=5120, delta="float32"),
        # the benchmark's prompt
        dict(name="norm_prompt_2048", op="norm", tokens=2048, width=4096, delta="bfloat16"),
        # the input of a feed-forward's second product, the benchmark's small batch
        dict(name="quantize_batch_8", op="quantize", tokens=8, width=12288, dtype="bfloat16"),
        # the same in a prompt of no round length and a model of no round width, 32-bit activations
        dict(name="quantize_odd", op="quantize", tokens=1531, width=4999, dtype="float32"),
        # a weight when a model is loaded: gate and up of one layer
        dict(name="quantize_weight", op="quantize", tokens=24576, width=4096, dtype="bfloat16"),
        # one user's reply: queries, keys and values
        dict(name="product_decode_1", op="product", tokens=1, outputs=6144, width=4096, out="bfloat16", gated=False),
        # the benchmark's small batch: gate and up with the activation
        dict(name="product_gated_8", op="product", tokens=8, outputs=24576, width=4096, out="bfloat16", gated=True),
        # a full batch of replies: the feed-forward's second product, long rows and few outputs
        dict(name="product_batch_64", op="product", tokens=64, outputs=4096, width=12288, out="bfloat16", gated=False),
        # nothing round: a question's prompt, 32-bit results
        dict(name="product_odd", op="product", tokens=301, outputs=5003, width=2055, out="float32", gated=False),
        # the benchmark's prompt: queries, keys and values
        dict(name="product_prompt_2048", op="product", tokens=2048, outputs=6144, width=4096, out="bfloat16", gated=False),
        # a step of several prompts: gate and up with the activation
        dict(name="product_gated_4096", op="product", tokens=4096, outputs=24576, width=4096, out="bfloat16", gated=True),
    ]


def _between(rng, low, high):
    """A whole number between the two, spread over the logarithm."""
    return max(low, min(high, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    op = rng.choice(["norm", "quantize", "product", "product"])
    if op == "norm":
        return dict(op=op, tokens=_between(rng, 1, 4096), width=_between(rng, 64, 8192), delta=rng.choice(["bfloat16", "float32"]))
    if op == "quantize":
        return dict(op=op, tokens=_between(rng, 1, 4096), width=_between(rng, 64, 16384), dtype=rng.choice(["bfloat16", "float32"]))
    tokens, outputs, width = _between(rng, 1, 4096), _between(rng, 64, 24576), _between(rng, 64, 16384)
    while tokens * outputs * width > 4096 * 24576 * 4096 or outputs * width > 24576 * 4096:
        tokens, outputs, width = _between(rng, 1, 4096), _between(rng, 64, 24576), _between(rng, 64, 16384)
    if rng.random() < 0.5:      # a model's sizes are mostly multiples of 64
        outputs, width = (outputs + 63) // 64 * 64, (width + 63) // 64 * 64
    gated = rng.random() < 0.4
    return dict(op=op, tokens=tokens, outputs=outputs // 2 * 2 if gated else outputs, width=width, gated=gated,
                out="bfloat16" if gated else rng.choice(["bfloat16", "float32"]))


def _device():
    return DEVICE if torch.cuda.is_available() else "cpu"


def _activations(g, rows, width):
    """Rows as they come in a model: channels of different size, a few of them far above the others."""
    channel = torch.exp(0.5 * torch.randn(width, generator=g, device=g.device))
    far = torch.rand(width, generator=g, device=g.device) < 0.002
    return torch.randn(rows, width, generator=g, device=g.device) * torch.where(far, 20.0 * channel, channel)


def _codes(values):
    """Rows of 8-bit codes that start on 16-byte borders, and their scales."""
    rows, width = values.shape
    scales = values.abs().amax(dim=1).clamp_min(1e-30) / 127.0
    held = torch.zeros(rows, (width + 15) // 16 * 16, dtype=torch.int8, device=values.device)
    held[:, :width] = torch.round(values / scales[:, None]).clamp_(-127, 127).to(torch.int8)
    return held[:, :width], scales


def prepare(case, seed):
    g = torch.Generator(device=_device())
    g.manual_seed(int(seed))
    tokens, width = case["tokens"], case["width"]
    if case["op"] == "norm":
        return {"op": "norm", "x": _activations(g, tokens, width), "delta": (0.1 * _activations(g, tokens, width)).to(TYPES[case["delta"]]),
                "weight": (1.0 + 0.1 * torch.randn(width, generator=g, device=g.device)).to(torch.bfloat16)}
    if case["op"] == "quantize":
        return {"op": "quantize", "x": _activations(g, tokens, width).to(TYPES[case["dtype"]])}
    a, a_scales = _codes(_activations(g, tokens, width))
    w, w_scales = _codes(0.02 * torch.randn(case["outputs"], width, generator=g, device=g.device))
    return {"op": "product", "a": a, "a_scales": a_scales, "w": w, "w_scales": w_scales, "out": TYPES[case["out"]], "gated": case["gated"]}


def run(state):
    if own:
        from spyinfer_b200 import kernels
        if state["op"] == "norm":
            got = kernels.rmsnorm_int8(state["x"], state["weight"], EPS, delta=state["delta"], write_back=True)
            return {"values": got.codes * got.scales[:, None], "stream": state["x"]}
        if state["op"] == "quantize":
            got = kernels.quantize_int8(state["x"])
            return {"values": got.codes * got.scales[:, None]}
        return {"result": kernels.gemm_int8(kernels.Int8Rows(state["a"], state["a_scales"]), kernels.Int8Rows(state["w"], state["w_scales"]),
                                            out_dtype=state["out"], epilogue="swiglu" if state["gated"] else None)}
    if state["op"] == "norm":
        x = state["x"]
        x.add_(state["delta"].float())
        inverse = torch.rsqrt((x * x).mean(dim=1) + EPS)
        codes, largest = _plain_codes(x * state["weight"].float())
        return {"values": codes * (largest / 127.0 * inverse)[:, None], "stream": x}
    if state["op"] == "quantize":
        codes, largest = _plain_codes(state["x"].float())
        return {"values": codes * (largest / 127.0)[:, None]}
    sums = state["a"].float() @ state["w"].float().t()
    z = sums * state["a_scales"][:, None] * state["w_scales"]
    if state["gated"]:
        gate, up = z[:, 0::2], z[:, 1::2]
        z = gate / (1.0 + torch.exp(-gate)) * up
    return {"result": z.to(state["out"])}


def _plain_codes(y):
    """The nearest integers to 127 y / max |y|, ties to even, and the largest sizes.  In 64 bits: which side of a half a quotient lies on is
    decided in the last bits."""
    largest = y.abs().amax(dim=1)
    return torch.round(y.double() * 127.0 / largest.double().clamp_min(1e-300)[:, None]).float(), largest


def work(case):
    tokens, width = case["tokens"], case["width"]
    if case["op"] == "norm":     # stream and output in, stream, codes and scales out
        size = 2 if case["delta"] == "bfloat16" else 4
        return {"bytes": tokens * width * (4 + size + 4 + 1) + 2 * width + 4 * tokens, "flops": 8 * tokens * width}
    if case["op"] == "quantize":
        size = 2 if case["dtype"] == "bfloat16" else 4
        return {"bytes": tokens * width * (size + 1) + 4 * tokens, "flops": 4 * tokens * width}
    outputs = case["outputs"]
    size = 2 if case["out"] == "bfloat16" else 4
    return {"bytes": tokens * width + outputs * width + 4 * (tokens + outputs) + size * tokens * (outputs // 2 if case["gated"] else outputs),
            "flops": 2 * tokens * outputs * width}


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "product":
        a = state["a"].to(torch.float64) * state["a_scales"].to(torch.float64).unsqueeze(1)
        w = state["w"].to(torch.float64) * state["w_scales"].to(torch.float64).unsqueeze(1)
        if not case["gated"]:
            return {"result": torch.matmul(a, w.transpose(0, 1))}
        gate, up = torch.matmul(a, w[0::2].transpose(0, 1)), torch.matmul(a, w[1::2].transpose(0, 1))
        return {"result": gate * torch.sigmoid(gate) * up}
    if case["op"] == "norm":
        # the stream and the row that is quantised are 32-bit numbers, by the operator's definition
        stream = (state["x"].to(torch.float64) + state["delta"].to(torch.float64)).to(torch.float32).to(torch.float64)
        row = (stream * state["weight"].to(torch.float64)).to(torch.float32).to(torch.float64)
        factor = 1.0 / torch.sqrt(torch.sum(stream.square(), 1, keepdim=True) / case["width"] + EPS)
    else:
        row, factor = state["x"].to(torch.float64), 1.0
    top = torch.max(row.abs(), 1, keepdim=True).values
    step = torch.where(top > 0, top / 127.0, torch.ones_like(top))
    # nearest integer, ties to even: of the two whole numbers around the quotient of 127 row and top, compared without dividing
    low = torch.floor(row / step)
    low = low - (low * top > 127.0 * row).to(torch.float64) + ((low + 1.0) * top <= 127.0 * row).to(torch.float64)
    rest, half = 2.0 * (127.0 * row - low * top), top
    up_one = (rest > half) | ((rest == half) & (torch.remainder(low, 2.0) == 1.0))
    values = torch.where(top > 0, (low + up_one.to(torch.float64)) * step * factor, torch.zeros_like(row))
    return {"values": values, "stream": stream} if case["op"] == "norm" else {"values": values}
