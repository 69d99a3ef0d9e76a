"""The operators of a transformer's dense sublayer as measurable cases: layer
norm and its backward pass, the matrix product with bias, activation and
residual in its epilogue and its backward pass, and the gated feed-forward
projections (both products, the activation and their product) and theirs.

With ``own`` false, ``run`` computes an operator in elementary torch
operations, in 32 bits whatever the inputs' type, rounded once at the end. With
``own`` true it launches the framework's operator program
(``tcacomp_amd.operators``), as a user's program does: on tensors that are
already on the GPU, into output tensors that the caller owns. The compiled
program is the handle such a program keeps, one for each set of attributes.

``listed`` holds fixed points of the ranges, ``draw`` any point of them:

  norms      1 to 65536 rows of 16 to 32768 elements, f32, bf16 and f16
  products   M (tokens) from 1 to 8192, K and N (features) from 64 to 8192,
             bf16 and f16; half of them with K and N multiples of 64, as
             weights mostly are, the others odd as they come

Weights are stored [K][N] (features in by features out).
"""
import functools
import math

import torch

own = False

DEVICE = "cuda"
EPS = 1e-5
ELEMS = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # The norm before a projection while one token is generated: latency.
        {"name": "norm_one_token", "op": "norm", "elem": "bf16", "r": 1, "c": 4096, "stats": False},
        # The repository's layernorm workload, its statistics kept for training.
        {"name": "norm_f32_1024", "op": "norm", "elem": "f32", "r": 32768, "c": 1024, "stats": True},
        # A training step's norm: its input's gradient joins the residual path's, the weights' gradients are summed over the batch.
        {"name": "norm_backward_4096", "op": "norm_backward", "elem": "bf16", "r": 8192, "c": 4096},
        # Odd rows of odd length: rows that no vector divides, partial blocks.
        {"name": "norm_backward_odd", "op": "norm_backward", "elem": "f16", "r": 1001, "c": 1501},
        # The projection back to the residual stream while one token is generated: the weight is read once.
        {"name": "linear_one_token", "op": "linear", "elem": "bf16", "m": 1, "k": 4096, "n": 4096, "act": "none", "residual": True, "save": False},
        # The repository's contraction workload with the whole epilogue.
        {"name": "linear_4096", "op": "linear", "elem": "bf16", "m": 4096, "k": 4096, "n": 4096, "act": "gelu", "residual": True, "save": False},
        # A ragged batch through odd features, pre-activation kept for training.
        {"name": "linear_odd", "op": "linear", "elem": "f16", "m": 1001, "k": 1003, "n": 1501, "act": "gelu", "residual": False, "save": True},
        # The gradients of an ordinary projection.
        {"name": "linear_backward_2048", "op": "linear_backward", "elem": "bf16", "m": 2048, "k": 1024, "n": 4096},
        # Sixteen sequences generating together: both weights are read once.
        {"name": "gated_decode_16", "op": "gated", "elem": "bf16", "m": 16, "k": 4096, "n": 8192, "save": False},
        # A training step's gated projections, pre-activations kept.
        {"name": "gated_train", "op": "gated", "elem": "bf16", "m": 4096, "k": 2048, "n": 8192, "save": True},
        # ... and their backward pass: the largest case.
        {"name": "gated_backward", "op": "gated_backward", "elem": "bf16", "m": 4096, "k": 2048, "n": 8192},
        # A small batch through odd features, in f16.
        {"name": "gated_backward_odd", "op": "gated_backward", "elem": "f16", "m": 500, "k": 769, "n": 2049},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(("norm", "norm_backward", "linear", "linear", "linear_backward", "gated", "gated", "gated_backward"))
    if op in ("norm", "norm_backward"):
        c = _log(rng, 16, 32768)
        if rng.random() < 0.5:
            c = c // 8 * 8
        case = {"op": op, "elem": rng.choice(sorted(ELEMS)), "r": _log(rng, 1, min(65536, (1 << 26) // c)), "c": c}
        if op == "norm":
            case["stats"] = rng.random() < 0.5
        return case
    whole = rng.random() < 0.5
    while True:
        m, k, n = _log(rng, 1, 8192), _log(rng, 64, 8192), _log(rng, 64, 8192)
        if whole:
            k, n = k // 64 * 64, n // 64 * 64
        if m * k * n <= 1 << 35:
            break
    case = {"op": op, "elem": rng.choice(("bf16", "f16")), "m": m, "k": k, "n": n}
    if op == "linear":
        case["act"] = rng.choice(("none", "gelu"))
        case["residual"] = case["act"] == "none"
        case["save"] = case["act"] == "gelu" and rng.random() < 0.5
    if op == "gated":
        case["save"] = rng.random() < 0.5
    return case


def _normal(gen, shape, elem, scale=1.0, shift=0.0):
    return torch.randn(shape, generator=gen, device=DEVICE).mul_(scale).add_(shift).to(ELEMS[elem])


def prepare(case, seed):
    """The inputs, and the output tensors that the caller owns."""
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    e, op = case["elem"], case["op"]

    def out(*shape, elem=e):
        return torch.empty(shape, device=DEVICE, dtype=ELEMS[elem])

    if op in ("norm", "norm_backward"):
        r, c = case["r"], case["c"]
        # Activations have a scale and an offset of their own per row.
        scale = torch.rand((r, 1), generator=gen, device=DEVICE) * 2 + 0.25
        x = (torch.randn((r, c), generator=gen, device=DEVICE) * scale + (scale - 1) * 0.5).to(ELEMS[e])
        gamma = _normal(gen, (c,), e, 0.2, 1.0)
        if op == "norm":
            outs = [out(r, c)] + ([out(r, elem="f32"), out(r, elem="f32")] if case["stats"] else [])
            return {"case": case, "in": [x, gamma, _normal(gen, (c,), e, 0.2)], "out": outs}
        x64 = x.double()
        mean = x64.mean(1)
        rstd = ((x64 - mean[:, None]).square().mean(1) + EPS).rsqrt()
        dy, dres = _normal(gen, (r, c), e), _normal(gen, (r, c), e)
        return {"case": case, "in": [dy, x, gamma, mean.float(), rstd.float(), dres], "out": [out(r, c), out(c), out(c)]}
    m, k, n = case["m"], case["k"], case["n"]
    x, w = _normal(gen, (m, k), e), _normal(gen, (k, n), e, k ** -0.5)
    if op == "linear":
        ins = [x, w, _normal(gen, (n,), e, 0.2)] + ([_normal(gen, (m, n), e)] if case["residual"] else [])
        return {"case": case, "in": ins, "out": [out(m, n)] + ([out(m, n)] if case["save"] else [])}
    if op == "linear_backward":
        return {"case": case, "in": [_normal(gen, (m, n), e), x, w, _normal(gen, (m, n), e)],
                "out": [out(m, n), out(m, k), out(k, n), out(n)]}
    wu = _normal(gen, (k, n), e, k ** -0.5)
    if op == "gated":
        return {"case": case, "in": [x, w, wu], "out": [out(m, n) for _ in range(3 if case["save"] else 1)]}
    return {"case": case, "in": [_normal(gen, (m, n), e), x, w, wu, _normal(gen, (m, n), e), _normal(gen, (m, n), e)],
            "out": [out(m, n), out(m, n), out(m, k), out(k, n), out(k, n)]}


@functools.lru_cache(maxsize=None)
def _program(op, elem, act, residual, keep):
    from tcacomp_amd import compiler, operators

    made = {
        "norm": lambda: operators.layer_norm(elem, stats=keep),
        "norm_backward": lambda: operators.layer_norm_backward(elem, residual=True),
        "linear": lambda: operators.linear(elem, act=act, bias=True, residual=residual, save=keep),
        "linear_backward": lambda: operators.linear_backward(elem, act="gelu", bias=True),
        "gated": lambda: operators.gated(elem, act="silu", save=keep),
        "gated_backward": lambda: operators.gated_backward(elem, act="silu"),
    }[op]()
    return compiler.compile_program(made)


def run(state):
    case = state["case"]
    if own:
        keep = case.get("stats", False) or case.get("save", False)
        program = _program(case["op"], case["elem"], case.get("act", ""), case.get("residual", False), keep)
        program.launch(state["in"] + state["out"], scalars=(EPS,) if case["op"] == "norm" else ())
        return state["out"]
    to = ELEMS[case["elem"]]
    return [t.to(to) if t.dim() > 1 or case["op"] != "norm" else t
            for t in _plain[case["op"]](case, *(t.float() for t in state["in"]))]


def _norm(case, x, gamma, beta):
    mean = x.mean(1, keepdim=True)
    d = x - mean
    rstd = 1.0 / (d.square().mean(1, keepdim=True) + EPS).sqrt()
    y = d * rstd * gamma + beta
    return [y, mean[:, 0], rstd[:, 0]] if case["stats"] else [y]


def _norm_backward(case, dy, x, gamma, mean, rstd, dres):
    xhat = (x - mean[:, None]) * rstd[:, None]
    t = dy * gamma
    dx = rstd[:, None] * (t - t.mean(1, keepdim=True) - xhat * (t * xhat).mean(1, keepdim=True)) + dres
    return [dx, (dy * xhat).sum(0), dy.sum(0)]


def _gelu(z):
    return 0.5 * z * (1.0 + torch.erf(z * 0.5 ** 0.5))


def _gelu_slope(z):
    return 0.5 * (1.0 + torch.erf(z * 0.5 ** 0.5)) + z * torch.exp(-0.5 * z * z) * (2.0 * math.pi) ** -0.5


def _linear(case, x, w, b, res=None):
    z = x @ w + b
    y = _gelu(z) if case["act"] == "gelu" else z
    y = y + res if case["residual"] else y
    return [y, z] if case["save"] else [y]


def _linear_backward(case, dy, x, w, z):
    dz = dy * _gelu_slope(z)
    return [dz, dz @ w.t(), x.t() @ dz, dz.sum(0)]


def _gated(case, x, wg, wu):
    g, u = x @ wg, x @ wu
    h = g / (1.0 + torch.exp(-g)) * u
    return [h, g, u] if case["save"] else [h]


def _gated_backward(case, dh, x, wg, wu, g, u):
    s = 1.0 / (1.0 + torch.exp(-g))
    dg, du = dh * u * s * (1.0 + g * (1.0 - s)), dh * g * s
    return [dg, du, dg @ wg.t() + du @ wu.t(), x.t() @ dg, x.t() @ du]


_plain = {"norm": _norm, "norm_backward": _norm_backward, "linear": _linear, "linear_backward": _linear_backward,
          "gated": _gated, "gated_backward": _gated_backward}


def work(case):
    size = 4 if case["elem"] == "f32" else 2
    op = case["op"]
    if op in ("norm", "norm_backward"):
        r, c = case["r"], case["c"]
        if op == "norm":
            return {"bytes": size * (2 * r * c + 2 * c) + (8 * r if case["stats"] else 0), "flops": 8 * r * c}
        return {"bytes": size * (4 * r * c + 3 * c) + 8 * r, "flops": 14 * r * c}
    m, k, n = case["m"], case["k"], case["n"]
    if op == "linear":
        planes = 1 + case["residual"] + case["save"]
        return {"bytes": size * (m * k + k * n + n + planes * m * n), "flops": 2 * m * k * n}
    if op == "linear_backward":
        return {"bytes": size * (2 * m * k + 2 * k * n + n + 3 * m * n), "flops": 4 * m * k * n}
    if op == "gated":
        return {"bytes": size * (m * k + 2 * k * n + (3 if case["save"] else 1) * m * n), "flops": 4 * m * k * n}
    return {"bytes": size * (2 * m * k + 4 * k * n + 5 * m * n), "flops": 8 * m * k * n}


def exact(case, seed):
    """The operators' definitions in 64 bits on the same inputs."""
    op = case["op"]
    a = [t.double() for t in prepare(case, seed)["in"]]
    if op == "norm":
        x, gamma, beta = a
        c = case["c"]
        mean = x.sum(1) / c
        var = ((x - mean.unsqueeze(1)) ** 2).sum(1) / c
        rstd = (var + EPS) ** -0.5
        y = torch.addcmul(beta, (x - mean.unsqueeze(1)) * rstd.unsqueeze(1), gamma)
        return [y, mean, rstd][: 3 if case["stats"] else 1]
    if op == "norm_backward":
        dy, x, gamma, mean, rstd, dres = a
        c = case["c"]
        # d xhat_j / d x_i = rstd (delta_ij - 1 / c - xhat_i xhat_j / c)
        xhat = (x - mean.unsqueeze(1)) * rstd.unsqueeze(1)
        t = dy * gamma
        s1, s2 = t.sum(1, keepdim=True), (t * xhat).sum(1, keepdim=True)
        return [(t - (s1 + xhat * s2) / c) * rstd.unsqueeze(1) + dres, (dy * xhat).sum(0), dy.sum(0)]
    if op == "linear":
        z = torch.addmm(a[2], a[0], a[1])
        y = z * torch.special.ndtr(z) if case["act"] == "gelu" else z.clone()
        if case["residual"]:
            y += a[3]
        return [y, z][: 2 if case["save"] else 1]
    if op == "linear_backward":
        dy, x, w, z = a
        density = torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        dz = dy * (torch.special.ndtr(z) + z * density)
        return [dz, torch.mm(dz, w.T), torch.mm(x.T, dz), dz.sum(0)]
    if op == "gated":
        x, wg, wu = a
        g, u = torch.mm(x, wg), torch.mm(x, wu)
        return [g * torch.sigmoid(g) * u, g, u][: 3 if case["save"] else 1]
    dh, x, wg, wu, g, u = a
    s = torch.sigmoid(g)
    dg = dh * u * (s + g * s * (1 - s))
    du = dh * (g * s)
    return [dg, du, torch.mm(dg, wg.T) + torch.mm(du, wu.T), torch.mm(x.T, dg), torch.mm(x.T, du)]
