"""The 8-bit operators as cases: what is measured of them, and their plain forms.

op "store"     quantize_s8 and dequantize_s8: a matrix into int8 codes with a scale for each token (axis 1) or channel (axis 0), and back
op "product"   gemm_s8: the product of int8 codes with a scale for each token and channel, with bias and GELU or without
op "forward"   gemm_bias_gelu_checkpoint: the fused product, and what its backward pass needs in 8 bits
op "backward"  gemm_bias_gelu_backward: the gradients from the 8-bit checkpoint
"""
import math

import torch

own = False  # run() makes the framework's calls where this is true, and computes the plain forms where it is not

K0, K1 = 0.7978845608028654, 0.044715  # the GELU's tanh form
GRAD_STEPS, GRAD_ZERO = 200, 26        # code of a GELU derivative d: rint(200 d) + 26
TINY = 2.0 ** -126                     # least scale
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}

MOST_VALUES = 16384 * 14336            # of a stored matrix
MOST_PRODUCT = 16384 * 14336 * 4096    # M N K of a product


def listed():
    return [
        # one token's activations, as a decoding step quantises them: latency
        {"name": "store token", "op": "store", "rows": 1, "cols": 4096, "axis": 1, "type": "bf16"},
        # a long batch's MLP activations, kept for the backward pass and restored in it
        {"name": "store batch", "op": "store", "rows": 16384, "cols": 14336, "axis": 1, "type": "bf16"},
        # a weight matrix quantised by output channel when a model is loaded
        {"name": "store weights", "op": "store", "rows": 4096, "cols": 14336, "axis": 0, "type": "f32"},
        # one decoding step of one sequence through the MLP's first product: the weights' bytes
        {"name": "product token", "op": "product", "M": 1, "N": 14336, "K": 4096, "bias": True, "gelu": True, "type": "bf16"},
        # a decoding step of a batch through the MLP's second product
        {"name": "product tokens", "op": "product", "M": 37, "N": 4096, "K": 14336, "bias": False, "gelu": False, "type": "bf16"},
        # odd sizes, whose rows no wide load fits; logits kept in 32 bits
        {"name": "product odd", "op": "product", "M": 333, "N": 1001, "K": 2050, "bias": True, "gelu": False, "type": "f32"},
        # the prompts of a batch
        {"name": "product prompt", "op": "product", "M": 16384, "N": 14336, "K": 4096, "bias": True, "gelu": True, "type": "bf16"},
        # a training step's forward pass of a toy layer, and of a full one
        {"name": "forward small", "op": "forward", "M": 200, "N": 136, "K": 72},
        {"name": "forward large", "op": "forward", "M": 16384, "N": 14336, "K": 4096},
        # their backward passes, and one of a ragged batch through a square layer
        {"name": "backward small", "op": "backward", "M": 77, "N": 512, "K": 512},
        {"name": "backward ragged", "op": "backward", "M": 1999, "N": 2048, "K": 2048},
        {"name": "backward large", "op": "backward", "M": 8192, "N": 14336, "K": 4096},
    ]


def draw(rng):
    def spread(low, high, step=1):  # even in the logarithm
        return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))) / step) * step))

    op = rng.choice(("store", "product", "forward", "backward"))
    if op == "store":
        cols = spread(8, 16384)
        return {"op": op, "rows": min(spread(1, 16384), MOST_VALUES // cols), "cols": cols, "axis": rng.choice((1, 1, 0)),
                "type": rng.choice(("bf16", "f32"))}
    if op == "product":
        step = rng.choice((16, 16, 16, 1))  # most models' widths are whole 16-byte rows
        N, K = spread(16, 16384, step), spread(16, 16384, step)
        return {"op": op, "M": min(spread(1, 16384), MOST_PRODUCT // (N * K)), "N": N, "K": K, "bias": rng.random() < 0.5,
                "gelu": rng.random() < 0.5, "type": rng.choice(("bf16", "f32"))}
    N, K = spread(8, 16384, 8), spread(8, 16384, 8)
    M = min(spread(1, 16384), MOST_PRODUCT // (N * K) // (2 if op == "backward" else 1))
    return {"op": op, "M": M, "N": N, "K": K}


def activations(rows, cols, gen):
    """Normal values whose channels have gains of their own, a few of them large, as a model's activations have."""
    gain = torch.exp(0.5 * torch.randn(cols, device="cuda", generator=gen))
    return torch.randn(rows, cols, device="cuda", generator=gen) * gain


def codes_of(x, axis):
    """The codes, and their scales: both quotients in 64 bits (the scale then rounded), as one next to a half step may be
    rounded past it in 32."""
    scale = (x.abs().amax(axis, keepdim=True).double() / 127).float().clamp(min=TINY)
    return torch.round(x.double() / scale).clamp(-127, 127).float(), scale


def gelu(x):
    return 0.5 * x * (1 + torch.tanh(K0 * (x + K1 * x * x * x)))


def gelu_grad(x):
    x = x.clamp(-12, 12)  # beyond, the derivative is 0 or 1 in any type used here
    t = torch.tanh(K0 * (x + K1 * x * x * x))
    return 0.5 * (1 + t) + 0.5 * x * (1 - t * t) * K0 * (1 + 3 * K1 * x * x)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    if case["op"] == "store":
        s["x"] = activations(case["rows"], case["cols"], gen).to(TYPES[case["type"]])
        return s
    M, N, K = case["M"], case["N"], case["K"]
    a = activations(M, K, gen)
    b = torch.randn(K, N, device="cuda", generator=gen) / math.sqrt(K)
    if case["op"] == "product":
        for name, x, axis in (("a", a, 1), ("b", b, 0)):
            codes, scale = codes_of(x, axis)
            s[name], s["scale_" + name] = codes.to(torch.int8), scale.reshape(-1)
        s["bias_values"] = 0.1 * torch.randn(N, device="cuda", generator=gen) if case["bias"] else None
        return s
    s["b"] = b.bfloat16()
    if case["op"] == "forward":
        s["a"], s["bias_values"] = a.bfloat16(), 0.1 * torch.randn(N, device="cuda", generator=gen)
        return s
    codes, scale = codes_of(a.bfloat16().float(), 1)
    s["a"], s["scale_a"] = codes.to(torch.int8), scale.reshape(-1)
    d = gelu_grad(torch.randn(M, N, device="cuda", generator=gen))
    s["d"] = (torch.round(GRAD_STEPS * d) + GRAD_ZERO).to(torch.uint8)
    s["dc"] = (0.01 * torch.randn(M, N, device="cuda", generator=gen)).bfloat16()
    return s


def run_own(s):
    import ptxforge_b200 as pf

    if s["op"] == "store":
        codes, scale = pf.quantize_s8(s["x"], axis=s["axis"])
        return {"values": pf.dequantize_s8(codes, scale, axis=s["axis"], dtype=TYPES[s["type"]]), "scale": scale}
    if s["op"] == "product":
        return {"c": pf.gemm_s8(s["a"], s["b"], s["scale_a"], s["scale_b"], s["bias_values"], gelu=s["gelu"], dtype=TYPES[s["type"]])}
    if s["op"] == "forward":
        c, saved = pf.gemm_bias_gelu_checkpoint(s["a"], s["b"], s["bias_values"])
        return {"c": c, "a": saved.input(), "d": saved.gelu_grad()}
    saved = pf.Checkpoint(s["a"], s["scale_a"], s["d"])
    da, db, dbias = pf.gemm_bias_gelu_backward(s["dc"], s["b"], saved)
    return {"da": da, "db": db, "dbias": dbias}


def run(s):
    if own:
        return run_own(s)
    if s["op"] == "store":
        codes, scale = codes_of(s["x"].float(), s["axis"])
        return {"values": (codes * scale).to(TYPES[s["type"]]), "scale": scale.reshape(-1)}
    if s["op"] == "product":
        x = torch.matmul(s["a"].float(), s["b"].float()) * s["scale_a"][:, None] * s["scale_b"]
        if s["bias_values"] is not None:
            x = x + s["bias_values"]
        return {"c": (gelu(x) if s["gelu"] else x).to(TYPES[s["type"]])}
    if s["op"] == "forward":
        a = s["a"].float()
        codes, scale = codes_of(a, 1)
        z = torch.matmul(a, s["b"].float()) + s["bias_values"]
        d = torch.round(GRAD_STEPS * gelu_grad(z)) / GRAD_STEPS
        return {"c": gelu(z).bfloat16(), "a": (codes * scale).bfloat16(), "d": d.bfloat16()}
    dz = s["dc"].float() * ((s["d"].float() - GRAD_ZERO) / GRAD_STEPS)
    a = s["a"].float() * s["scale_a"][:, None]
    da, db = torch.matmul(dz, s["b"].float().t()), torch.matmul(a.t(), dz)
    return {"da": da.bfloat16(), "db": db.bfloat16(), "dbias": dz.sum(0)}


def work(case):
    if case["op"] == "store":  # the matrix in, the scales and the restored matrix out
        size, lines = {"bf16": 2, "f32": 4}[case["type"]], case["rows"] if case["axis"] else case["cols"]
        return {"bytes": 2 * size * case["rows"] * case["cols"] + 4 * lines, "flops": 0}
    M, N, K = case["M"], case["N"], case["K"]
    if case["op"] == "product":
        size = {"bf16": 2, "f32": 4}[case["type"]]
        return {"bytes": M * K + K * N + 4 * (M + N + (N if case["bias"] else 0)) + size * M * N, "flops": 2 * M * N * K}
    if case["op"] == "forward":  # A, B and the bias in; C and the two restored checkpoints out
        return {"bytes": 2 * M * K + 2 * K * N + 4 * N + 2 * M * N + 2 * M * K + 2 * M * N, "flops": 2 * M * N * K}
    return {"bytes": 2 * M * N + M * N + M * K + 4 * M + 2 * K * N + 2 * M * K + 2 * K * N + 4 * N, "flops": 4 * M * N * K}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "store":
        x = s["x"].double()
        scale = torch.linalg.vector_norm(x, math.inf, dim=case["axis"], keepdim=True).div(127).float().double()
        scale = torch.where(scale < TINY, TINY, scale)
        return {"values": torch.floor(x.div_(scale).abs() + 0.5).mul_(s["x"].sign().double()).mul_(scale), "scale": scale.flatten()}
    sigmoid_gelu = lambda x: x * torch.sigmoid(2 * K0 * x * (1 + K1 * x ** 2))  # noqa: E731
    if case["op"] == "product":
        x = torch.einsum("mk,kn->mn", s["a"].double(), s["b"].double())
        x = torch.einsum("mn,m,n->mn", x, s["scale_a"].double(), s["scale_b"].double())
        if s["bias_values"] is not None:
            x += s["bias_values"].double()
        return {"c": sigmoid_gelu(x) if case["gelu"] else x}
    if case["op"] == "forward":
        a = s["a"].double()
        z = torch.addmm(s["bias_values"].double(), a, s["b"].double())
        p = torch.sigmoid(2 * K0 * z * (1 + K1 * z ** 2))
        d = p + 2 * K0 * z * p * (1 - p) * (1 + 3 * K1 * z ** 2)
        c = z.mul_(p)
        scale = torch.linalg.vector_norm(a, math.inf, dim=1, keepdim=True).div(127).float().double().clamp_min(TINY)
        return {"c": c, "a": torch.floor(a / scale + 0.5) * scale, "d": torch.floor(d * GRAD_STEPS + 0.5) / GRAD_STEPS}
    dz = torch.einsum("mn,mn->mn", s["dc"].double(), (s["d"].double() - GRAD_ZERO) / GRAD_STEPS)
    a = torch.einsum("mk,m->mk", s["a"].double(), s["scale_a"].double())
    return {"da": torch.einsum("mn,kn->mk", dz, s["b"].double()), "db": torch.einsum("mk,mn->kn", a, dz), "dbias": torch.einsum("mn->n", dz)}
