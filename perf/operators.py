"""The operators of 8-bit linear layers, measured: what they are called with, their plain forms and their values in 64 bits.

A linear layer in 8 bits multiplies rows held in e4m3 with a float32 scale for each 128 values of a row by a weight held in
e4m3 with a scale for each block of 128 x 128.  Four operators make it up:

* ``norm``: the residual's addition and the root-mean-square norm, whose result is a product's rows;
* ``gated``: the gated activation between a feed-forward's two products, whose result is the second one's rows;
* ``quantize``: rows that come from elsewhere (an attention's output), or a weight in blocks, when a model is loaded;
* ``product``: the product itself.

With amax the largest magnitude of a block and a = max(amax, 448 * 2^-126), a block's scale is a / 448 and its values are
round(x * (448 / a)) to e4m3 (ties to even), so that the largest magnitude becomes 448, the largest e4m3 value.
"""
import math

import torch

own = False

BLOCK = 128
TOP = 448.0
LEAST = TOP * 2.0 ** -126
EPS = 1e-6
_TYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


def listed():
    return [
        # the query, key and value projection of one decoded token, hidden size 4096 with 32 + 2 * 8 heads of 128
        {"name": "product_1x6144x4096", "op": "product", "m": 1, "n": 6144, "k": 4096, "out": "bfloat16"},
        # the product behind the activation of a batch of eight, added to a float32 residual afterwards
        {"name": "product_8x4096x12288", "op": "product", "m": 8, "n": 4096, "k": 12288, "out": "float32"},
        # the gate and up projection of a batch of 64 decoded tokens, feed-forward size 12288
        {"name": "product_64x24576x4096", "op": "product", "m": 64, "n": 24576, "k": 4096, "out": "bfloat16"},
        # a short prompt's ragged portion at a width that is no multiple of a block, in either direction
        {"name": "product_203x1000x2064", "op": "product", "m": 203, "n": 1000, "k": 2064, "out": "bfloat16"},
        # the gate and up projection of a prompt portion of 2,048 tokens: compute
        {"name": "product_2048x24576x4096", "op": "product", "m": 2048, "n": 24576, "k": 4096, "out": "bfloat16"},
        # one decoded token behind a product cut into four parts, hidden size 4096
        {"name": "norm_1x4096_parts4", "op": "norm", "t": 1, "e": 4096, "parts": 4, "add": "float32"},
        # a prompt portion, hidden size 5120, an addend in bfloat16
        {"name": "norm_2048x5120", "op": "norm", "t": 2048, "e": 5120, "parts": 1, "add": "bfloat16"},
        # a batch of eight decoded tokens, 12,288 features
        {"name": "gated_8x12288", "op": "gated", "t": 8, "f": 12288, "in": "bfloat16"},
        # a prompt portion of 2,048 tokens
        {"name": "gated_2048x12288", "op": "gated", "t": 2048, "f": 12288, "in": "bfloat16"},
        # the attention's output of 32 decoded tokens, the first 4,096 columns of rows of 4,608
        {"name": "quantize_32x4096_strided", "op": "quantize", "t": 32, "k": 4096, "stride": 4608, "rows": 1, "in": "bfloat16"},
        # the attention's output of a prompt portion
        {"name": "quantize_2048x4096", "op": "quantize", "t": 2048, "k": 4096, "stride": 4096, "rows": 1, "in": "bfloat16"},
        # a weight of a model being loaded
        {"name": "quantize_blocks_12288x4096", "op": "quantize", "t": 12288, "k": 4096, "stride": 4096, "rows": 128, "in": "bfloat16"},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("product", "product", "norm", "gated", "quantize"))
    if op == "product":
        m, n, k = _log(rng, 1, 4096), _log(rng, 64, 25600), 16 * _log(rng, 4, 1600)
        while m * n * k > 2048 * 24576 * 4096:
            m = max(1, m // 2)
        return {"op": op, "m": m, "n": n, "k": k, "out": rng.choice(("bfloat16", "bfloat16", "float32"))}
    if op == "norm":
        t, e = _log(rng, 1, 4096), _log(rng, 64, 8192)
        parts = rng.choice((1, 1, 2, 3, 4)) if t <= 128 else 1
        return {"op": op, "t": t, "e": e, "parts": parts, "add": "float32" if parts > 1 else rng.choice(("bfloat16", "float32"))}
    if op == "gated":
        return {"op": op, "t": _log(rng, 1, 2048), "f": _log(rng, 64, 25600), "in": rng.choice(("bfloat16", "bfloat16", "float32"))}
    rows = rng.choice((1, 1, 128))
    t, k = (_log(rng, 1, 4096), _log(rng, 64, 12288)) if rows == 1 else (_log(rng, 64, 12288), _log(rng, 64, 4096))
    return {"op": op, "t": t, "k": k, "stride": k + (0 if rows == 128 else 8 * rng.randrange(0, 65)), "rows": rows, "in": rng.choice(("bfloat16", "bfloat16", "float32"))}


def _blocks(x, rows):
    """The largest magnitude of each block of `rows` x 128 (both may end inside a block), and those spread back over x's places."""
    t, k = x.shape
    tb, kb = -(-t // rows), -(-k // BLOCK)
    padded = x.new_zeros(tb * rows, kb * BLOCK)
    padded[:t, :k] = x.abs()
    amax = padded.view(tb, rows, kb, BLOCK).amax(dim=(1, 3))
    return amax, amax.repeat_interleave(rows, 0)[:t].repeat_interleave(BLOCK, 1)[:, :k]


def _quantize(x, rows):
    """float32 x in e4m3 with a scale for each block."""
    amax, spread = _blocks(x, rows)
    top = torch.tensor(TOP, device=x.device)                 # (a quotient with a number would be a product with its reciprocal)
    return (x * torch.div(top, spread.clamp(min=LEAST))).to(torch.float8_e4m3fn), torch.div(amax.clamp(min=LEAST), top)


def _values(q, scales, rows):
    """What e4m3 values with scales stand for, in the scales' type."""
    t, k = q.shape
    return q.to(scales.dtype) * scales.repeat_interleave(rows, 0)[:t].repeat_interleave(BLOCK, 1)[:, :k]


def _heavy(shape, g, device):
    """Values as activations have them: normal, with a few columns some times larger."""
    x = torch.randn(shape, generator=g, device=device)
    return x * torch.where(torch.rand(shape[-1], generator=g, device=device) < 0.01, 12.0, 1.0)


def prepare(case, seed):
    device = "cuda"
    g = torch.Generator(device=device).manual_seed(seed)
    op = case["op"]
    state = {"case": case}
    if op == "product":
        x, w = _heavy((case["m"], case["k"]), g, device), torch.randn(case["n"], case["k"], generator=g, device=device) * 0.02
        state["x"], state["xs"] = _quantize(x, 1)
        state["w"], state["ws"] = _quantize(w, BLOCK)
    elif op == "norm":
        shape = (case["t"], case["e"]) if case["parts"] == 1 else (case["parts"], case["t"], case["e"])
        state["x"] = 3.0 * _heavy((case["t"], case["e"]), g, device)
        state["add"] = torch.randn(shape, generator=g, device=device).to(_TYPES[case["add"]])
        state["weight"] = 1.0 + 0.2 * torch.randn(case["e"], generator=g, device=device)
    elif op == "gated":
        state["gate_up"] = (2.0 * _heavy((case["t"], 2 * case["f"]), g, device)).to(_TYPES[case["in"]])
    else:
        whole = _heavy((case["t"], case["stride"]), g, device) * (0.02 if case["rows"] == BLOCK else 1.0)
        state["x"] = whole.to(_TYPES[case["in"]])[:, :case["k"]]
    return state


def _run_own(state):
    from purhie_b200.csrc import fp8
    case = state["case"]
    op = case["op"]
    if op == "product":
        return fp8.gemm(state["x"], state["xs"], state["w"], state["ws"], out_dtype=_TYPES[case["out"]])
    if op == "norm":
        x_out = torch.empty_like(state["x"])
        q, scales = fp8.add_rmsnorm(state["x"], state["add"], state["weight"], EPS, add_splits=case["parts"], x_out=x_out)
        return {"x": x_out, "q": q, "scales": scales}
    if op == "gated":
        q, scales = fp8.gated(state["gate_up"])
        return {"q": q, "scales": scales}
    q, scales = fp8.quantize(state["x"], block_rows=case["rows"])
    return {"q": q, "scales": scales}


def run(state):
    if own:
        return _run_own(state)
    case = state["case"]
    op = case["op"]
    if op == "product":
        y = _values(state["x"], state["xs"], 1) @ _values(state["w"], state["ws"], BLOCK).t()
        return y.to(_TYPES[case["out"]])
    if op == "norm":
        add = state["add"].float()
        x = state["x"] + (add.sum(0) if case["parts"] > 1 else add)
        q, scales = _quantize(x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * state["weight"], 1)
        return {"x": x, "q": q, "scales": scales}
    if op == "gated":
        pairs = state["gate_up"].float().view(case["t"], case["f"], 2)
        q, scales = _quantize(pairs[..., 0] / (1.0 + torch.exp(-pairs[..., 0])) * pairs[..., 1], 1)
        return {"q": q, "scales": scales}
    q, scales = _quantize(state["x"].float(), case["rows"])
    return {"q": q, "scales": scales}


def work(case):
    op = case["op"]
    kb = lambda k: -(-k // BLOCK)  # noqa: E731
    size = lambda name: 2 if name == "bfloat16" else 4  # noqa: E731
    if op == "product":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * k + 4 * m * kb(k) + n * k + 4 * kb(n) * kb(k) + m * n * size(case["out"]), "flops": 2.0 * m * n * k}
    if op == "norm":
        t, e = case["t"], case["e"]
        return {"bytes": t * e * (4 + case["parts"] * size(case["add"]) + 4 + 1) + 4 * e + 4 * t * kb(e), "flops": t * e * (7.0 + case["parts"])}
    if op == "gated":
        t, f = case["t"], case["f"]
        return {"bytes": t * f * (2 * size(case["in"]) + 1) + 4 * t * kb(f), "flops": 8.0 * t * f}
    t, k, rows = case["t"], case["k"], case["rows"]
    return {"bytes": t * k * (size(case["in"]) + 1) + 4 * -(-t // rows) * kb(k), "flops": 3.0 * t * k}


def _nearest_e4m3(v):
    """The nearest e4m3 value of each float64, ties to the even one: a step of 2^(e - 3), and of 2^-9 below 2^-6."""
    exponent = torch.frexp(v.abs())[1] - 1
    step = torch.ldexp(torch.ones_like(v), exponent.clamp(min=-6) - 3)
    return (torch.round(v / step) * step).clamp(-TOP, TOP)


def _quantize_exact(y, rows):
    t, k = y.shape
    q = torch.empty_like(y)
    scales = y.new_empty(-(-t // rows), -(-k // BLOCK))
    for j in range(scales.shape[1]):
        part = y[:, j * BLOCK:(j + 1) * BLOCK]
        top = part.abs().amax(1)
        if rows > 1:
            top = torch.stack([p.amax() for p in top.split(rows)])
        scales[:, j] = torch.clamp(top, min=LEAST) / TOP
        q[:, j * BLOCK:(j + 1) * BLOCK] = _nearest_e4m3(part / scales[:, j].repeat_interleave(rows)[:t, None])
    return {"q": q, "scales": scales}


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "product":
        m, n, k = case["m"], case["n"], case["k"]
        y = torch.zeros(m, n, dtype=torch.float64, device=s["x"].device)
        at = torch.arange(n, device=y.device) // BLOCK
        for j in range(-(-k // BLOCK)):
            cut = slice(j * BLOCK, (j + 1) * BLOCK)
            y += (s["x"][:, cut].double() @ s["w"][:, cut].double().t()) * s["xs"][:, j, None].double() * s["ws"][at, j].double()
        return y
    if op == "norm":
        x = s["x"].double()
        for part in s["add"].view(case["parts"], case["t"], case["e"]):
            x = x + part.double()
        root = torch.sqrt((x * x).sum(1, keepdim=True) / case["e"] + EPS)
        return {"x": x, **_quantize_exact(s["weight"].double() * x / root, 1)}
    if op == "gated":
        gate, up = s["gate_up"].double()[:, 0::2], s["gate_up"].double()[:, 1::2]
        return _quantize_exact(gate * torch.sigmoid(gate) * up, 1)
    return _quantize_exact(s["x"].double(), case["rows"])
