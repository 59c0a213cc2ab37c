"""The operators of the 8-bit linear path: what is measured, and their plain forms.

Three operators that run one after the other in front of and inside a linear
layer whose weights and activations are 8-bit floating point (e4m3):

  norm      root-mean-square normalisation of the rows of x (plus a residual),
            times a weight per column; the result in x's type, or in e4m3 with
            one fp32 scale for every 128 columns of a row
  quantize  x in e4m3 with one scale for 128 columns of a row (activations), or
            for a block of 128 rows by 128 columns (weights, laid out once)
  matmul    y = relu?(sum over blocks of 128 k's of a_scale * b_scale * (A . B^T)
            + bias), A [m, k] and B [n, k] in e4m3 with the scales above

Scales: amax = max(|block|, 2**-96), scale = amax / 448, q = e4m3(x * (448 / amax)).
e4m3 rows are stored with a row stride that is a multiple of 16 bytes.
"""
import importlib
import math

import torch

own = False

BLOCK = 128
FMAX = 448.0
FLOOR = 2.0 ** -96
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
E4M3 = torch.float8_e4m3fn


def listed():
    return [
        # one token of a decoding step: latency of a single row
        {"name": "norm one row", "op": "norm", "rows": 1, "cols": 4096, "type": "bf16", "residual": True, "quantize": True},
        # the vision / encoder width of this repository's MatMul workload, fp32 as its tensors are
        {"name": "norm fp32 width 768", "op": "norm", "rows": 4096, "cols": 768, "type": "f32", "residual": False, "quantize": False},
        # a prompt of 8192 tokens in front of a wide layer
        {"name": "norm prompt", "op": "norm", "rows": 8192, "cols": 8192, "type": "bf16", "residual": True, "quantize": True},
        # a width that is no multiple of a block or of a vector
        {"name": "norm odd width", "op": "norm", "rows": 333, "cols": 5001, "type": "f16", "residual": True, "quantize": True},
        # a decoding batch's activations after an activation function
        {"name": "quantize batch", "op": "quantize", "rows": 64, "cols": 14336, "block_rows": 1, "type": "bf16"},
        # a prompt's activations, fp32
        {"name": "quantize prompt", "op": "quantize", "rows": 8192, "cols": 4096, "block_rows": 1, "type": "f32"},
        # weights at load time, ragged in both directions
        {"name": "quantize weights", "op": "quantize", "rows": 5000, "cols": 2050, "block_rows": 128, "type": "bf16"},
        # one token through a linear layer: bound by the weights' bytes
        {"name": "matmul one row", "op": "matmul", "m": 1, "n": 4096, "k": 4096, "type": "bf16", "bias": False, "relu": False},
        # the classifier of this repository's ResNet-50 at a small batch
        {"name": "matmul classifier", "op": "matmul", "m": 17, "n": 1000, "k": 2048, "type": "f32", "bias": True, "relu": True},
        # a decoding batch through a wide layer
        {"name": "matmul batch", "op": "matmul", "m": 200, "n": 8192, "k": 4096, "type": "bf16", "bias": False, "relu": False},
        # ragged in every direction
        {"name": "matmul ragged", "op": "matmul", "m": 1777, "n": 5000, "k": 1100, "type": "f16", "bias": True, "relu": False},
        # a prompt of 8192 tokens through a wide layer: bound by the tensor cores
        {"name": "matmul prompt", "op": "matmul", "m": 8192, "n": 8192, "k": 8192, "type": "bf16", "bias": False, "relu": False},
    ]


def _spread(rng, low, high):
    """A whole number, spread over the logarithm of the range."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["norm", "quantize", "matmul", "matmul"])
    kind = rng.choice(["f32", "f16", "bf16"])
    if op == "matmul":
        m, n, k = _spread(rng, 1, 8192), _spread(rng, 64, 14336), _spread(rng, 64, 14336)
        while m * n * k > 8192 ** 3:
            m = max(1, m // 2)
        return {"op": op, "m": m, "n": n, "k": k, "type": kind, "bias": rng.random() < 0.5, "relu": rng.random() < 0.3}
    rows, cols = _spread(rng, 1, 8192), _spread(rng, 64, 14336)
    while rows * cols > 2 ** 25:
        rows = max(1, rows // 2)
    if op == "norm":
        return {"op": op, "rows": rows, "cols": cols, "type": kind, "residual": rng.random() < 0.7, "quantize": rng.random() < 0.6}
    return {"op": op, "rows": rows, "cols": cols, "block_rows": rng.choice([1, 128]), "type": kind}


# ------------------------------------------------------------------ inputs
def _normal(shape, gen):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)


def _activations(rows, cols, gen):
    """Hidden states: normal values whose size differs by row, a few columns far larger than the others, as trained models have them."""
    size = torch.exp(0.5 * _normal((rows, 1), gen))
    loud = 1.0 + 20.0 * (torch.rand((1, cols), generator=gen, device="cuda") < 0.004).float()
    return _normal((rows, cols), gen).mul_(size).mul_(loud)


def _padded(q):
    """The same values with a row stride that is a multiple of 16 bytes."""
    rows, cols = q.shape
    held = torch.zeros((rows, (cols + 15) // 16 * 16), dtype=torch.uint8, device=q.device)
    held[:, :cols] = q.view(torch.uint8)
    return held.view(E4M3)[:, :cols]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    s = {"case": case}
    if case["op"] == "norm":
        t = TYPES[case["type"]]
        s["x"] = _activations(case["rows"], case["cols"], gen).to(t)
        s["residual"] = (3.0 * _activations(case["rows"], case["cols"], gen)).to(t) if case["residual"] else None
        s["weight"] = (1.0 + 0.2 * _normal((case["cols"],), gen)).to(t)
    elif case["op"] == "quantize":
        t = TYPES[case["type"]]
        x = _activations(case["rows"], case["cols"], gen) if case["block_rows"] == 1 else 0.02 * _normal((case["rows"], case["cols"]), gen)
        s["x"] = x.to(t)
    else:
        m, n, k = case["m"], case["n"], case["k"]
        q, qs = _plain_quantize(_activations(m, k, gen), 1)
        s["a"], s["a_scale"] = _padded(q), qs.t().contiguous().t()  # the scales of one block of k's lie side by side
        q, s["b_scale"] = _plain_quantize(_normal((n, k), gen).mul_(k ** -0.5), 128)
        s["b"] = _padded(q)
        s["bias"] = 0.5 * _normal((n,), gen) if case["bias"] else None
    if own:
        _prepare_own(s)
    return s


# ------------------------------------------------------------------ plain forms
def _plain_quantize(x, block_rows):
    """x fp32 [rows, cols] -> e4m3 [rows, cols], fp32 scales [ceil(rows / block_rows), ceil(cols / 128)]."""
    rows, cols = x.shape
    rb, cb = -(-rows // block_rows), -(-cols // BLOCK)
    if rb * block_rows == rows and cb * BLOCK == cols:
        v = x.reshape(rb, block_rows, cb, BLOCK)
    else:
        v = torch.zeros((rb * block_rows, cb * BLOCK), dtype=torch.float32, device=x.device)
        v[:rows, :cols] = x
        v = v.view(rb, block_rows, cb, BLOCK)
    amax = v.abs().amax(dim=(1, 3), keepdim=True).clamp(min=FLOOR)
    q = (v * (FMAX / amax)).clamp(-FMAX, FMAX).to(E4M3).view(rb * block_rows, cb * BLOCK)[:rows, :cols]
    return q, (amax / FMAX).view(rb, cb)


def _plain_norm(x, residual, weight, quantize):
    t = x.dtype
    h = x.float() if residual is None else x.float() + residual.float()
    y = h * torch.rsqrt(h.square().mean(dim=1, keepdim=True) + 1e-5) * weight.float()
    out = list(_plain_quantize(y, 1)) if quantize else [y.to(t)]
    return out if residual is None else out + [h.to(t)]


def _plain_matmul(a, a_scale, b, b_scale, bias, relu, t):
    k = a.shape[1]
    fa = a.float() * a_scale.repeat_interleave(BLOCK, dim=1)[:, :k]
    fb = b.float() * b_scale.repeat_interleave(BLOCK, dim=0)[: b.shape[0]].repeat_interleave(BLOCK, dim=1)[:, :k]
    y = fa @ fb.t()
    y = y if bias is None else y + bias
    return [(torch.relu(y) if relu else y).to(t)]


def run(state):
    if own:
        return state["call"]()
    c = state["case"]
    if c["op"] == "norm":
        return _plain_norm(state["x"], state["residual"], state["weight"], c["quantize"])
    if c["op"] == "quantize":
        return list(_plain_quantize(state["x"].float(), c["block_rows"]))
    return _plain_matmul(state["a"], state["a_scale"], state["b"], state["b_scale"], state["bias"], c["relu"], TYPES[c["type"]])


# ------------------------------------------------------------------ the framework's calls
_context = None


def _prepare_own(s):
    """The operator objects a program builds once: run() calls compute() on the tensors it has in hand."""
    global _context
    ob = importlib.import_module("onnx-rs_b200")
    if _context is None:
        _context = ob.ExecutionContext(ob.Handle(0))
    ctx, c = _context, s["case"]
    if c["op"] == "norm":
        op = ob.RMSNormalization(epsilon=1e-5, quantize=c["quantize"])
        s["call"] = lambda: op.compute([s["x"], s["weight"]], ctx, residual=s["residual"])
    elif c["op"] == "quantize":
        op = ob.QuantizeBlocks(block_rows=c["block_rows"])
        s["call"] = lambda: op.compute([s["x"]], ctx)
    else:
        op = ob.MatMulBlockScaled(dtype=TYPES[c["type"]], relu=c["relu"])
        s["call"] = lambda: op.compute([s["a"], s["a_scale"], s["b"], s["b_scale"], s["bias"]], ctx)


# ------------------------------------------------------------------ work
def work(case):
    if case["op"] == "matmul":
        m, n, k = case["m"], case["n"], case["k"]
        kb, nb = -(-k // BLOCK), -(-n // BLOCK)
        return {"bytes": m * k + n * k + 4 * (m * kb + nb * kb) + SIZES[case["type"]] * m * n + (4 * n if case["bias"] else 0),
                "flops": 2 * m * n * k}
    rows, cols, e = case["rows"], case["cols"], SIZES[case["type"]]
    cb = -(-cols // BLOCK)
    if case["op"] == "quantize":
        return {"bytes": rows * cols * (e + 1) + 4 * cb * -(-rows // case["block_rows"]), "flops": 3 * rows * cols}
    out = rows * cols + 4 * rows * cb if case["quantize"] else rows * cols * e
    return {"bytes": rows * cols * e * (3 if case["residual"] else 1) + cols * e + out, "flops": 6 * rows * cols}


# ------------------------------------------------------------------ the definition in 64 bits
def _to_e4m3(v):
    """Nearest e4m3 value, ties to even: 3 fraction bits, exponents from 2**-6, multiples of 2**-9 below."""
    exponent = torch.frexp(v.abs())[1].clamp(min=-5) - 1
    step = torch.ldexp(torch.ones_like(v), exponent - 3)
    return ((v / step).round() * step).clamp(-FMAX, FMAX)


def _exact_quantize(x, block_rows):
    rows, cols = x.shape
    rb, cb = -(-rows // block_rows), -(-cols // BLOCK)
    big = torch.nn.functional.pad(x.abs(), (0, cb * BLOCK - cols, 0, rb * block_rows - rows))
    big = big.unflatten(1, (cb, BLOCK)).amax(2).unflatten(0, (rb, block_rows)).amax(1).clamp(min=FLOOR)
    r = torch.arange(rows, device=x.device) // block_rows
    c = torch.arange(cols, device=x.device) // BLOCK
    return _to_e4m3(x * FMAX / big[r][:, c]), big / FMAX


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quantize":
        return list(_exact_quantize(s["x"].double(), case["block_rows"]))
    if case["op"] == "norm":
        h = s["x"].double()
        if case["residual"]:
            h = h + s["residual"].double()
        y = s["weight"].double() * h / torch.sqrt((h * h).sum(1, keepdim=True) / case["cols"] + 1e-5)
        out = list(_exact_quantize(y, 1)) if case["quantize"] else [y]
        return out + [h] if case["residual"] else out
    y = torch.zeros((case["m"], case["n"]), dtype=torch.float64, device="cuda")
    rows = torch.arange(case["n"], device="cuda") // BLOCK
    for j in range(-(-case["k"] // BLOCK)):
        at = slice(j * BLOCK, min(case["k"], (j + 1) * BLOCK))
        a = s["a"][:, at].double() * s["a_scale"][:, j: j + 1].double()
        b = s["b"][:, at].double() * s["b_scale"][rows, j: j + 1].double()
        y.addmm_(a, b.t())
    if case["bias"]:
        y += s["bias"].double()
    return [y.clamp(min=0) if case["relu"] else y]
