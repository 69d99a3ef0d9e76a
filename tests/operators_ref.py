"""The operator programs' definitions in 64 bits (torch, any device), and the
bounds that the GPU tests hold the kernels to. u = 2^-24 is half a step of f32
relative to the value; a result of type T adds half a step of T."""
import math

import torch

U = 2.0 ** -24
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def half_step(t, value):
    """Half a step of type t at |value|, its smallest numbers included."""
    fi = torch.finfo(t)
    return fi.eps / 2 * value.abs() + fi.smallest_normal * fi.eps / 2


# ------------------------------------------------------------- definitions

def layer_norm(x, gamma, beta, eps):
    mean = x.mean(1)
    d = x - mean[:, None]
    rstd = ((d * d).mean(1) + eps) ** -0.5
    y = d * rstd[:, None] * gamma
    return (y if beta is None else y + beta), mean, rstd


def layer_norm_backward(dy, x, gamma, mean, rstd, dres):
    h = (x - mean[:, None]) * rstd[:, None]
    t = dy * gamma
    dx = rstd[:, None] * (t - t.mean(1, keepdim=True) - h * (t * h).mean(1, keepdim=True))
    return (dx if dres is None else dx + dres), (dy * h).sum(0), dy.sum(0)


def act(name, z):
    if name == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z)
    if name == "silu":
        return z / (1 + torch.exp(-z))
    if name == "gelu":
        return z * torch.special.ndtr(z)
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    return z


def slope(name, z):
    if name == "relu":
        return torch.where(z <= 0, torch.zeros_like(z), torch.ones_like(z))
    if name == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    if name == "gelu":
        return torch.special.ndtr(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z ** 3))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    return torch.ones_like(z)


# ------------------------------------------------------------------ bounds

def layer_norm_bounds(x, gamma, beta, eps, out):
    """(y, mean, rstd). A sum of C terms in chains of at most D: a lane's 32
    values, six steps of a wave, 16 waves, and in long rows a lane's share of
    them. e_m and e_v are the errors of the mean and of the variance (the
    centred squares, and e_m^2, since the squares about a mean that is off
    by e_m exceed those about the mean by e_m^2)."""
    C = x.shape[1]
    D = C / 1024 + 64
    mean = x.mean(1, keepdim=True)
    d = x - mean
    var = (d * d).mean(1, keepdim=True)
    e_m = (D + 2) * U * x.abs().mean(1, keepdim=True) + 2 * U * mean.abs()
    # of every (x - m)^2: the difference's rounding and e_m, and the square's;
    # pairwise merges in long rows add two roundings of a mean a merge
    e_d = e_m + U * d.abs() + 2 * U * mean.abs() * (C > 8192) * D ** 0.5
    e_v = (2 * d.abs() * e_d).mean(1, keepdim=True) + (e_d * e_d).mean(1, keepdim=True) + (D + 4) * U * var
    rel = 0.5 * e_v / (var + eps) + 8 * U
    rstd = (var + eps) ** -0.5
    y = d * rstd * gamma
    b = (e_m + d.abs() * (rel + 6 * U)) * rstd * gamma.abs()
    if beta is not None:
        y = y + beta
        b = b + 2 * U * (y.abs() + beta.abs())
    return b + half_step(out, y), e_m[:, 0], (rel * rstd)[:, 0]


def layer_norm_backward_bounds(dy, x, gamma, mean, rstd, dres, out, weight):
    R, C = x.shape
    D = C / 1024 + 72
    h = (x - mean[:, None]) * rstd[:, None]
    t = dy * gamma
    rs = rstd[:, None]
    e = D * U * (t.abs().mean(1, keepdim=True) + h.abs() * (t * h).abs().mean(1, keepdim=True))
    want, dg, db = layer_norm_backward(dy, x, gamma, mean, rstd, dres)
    b = rs * (6 * U * t.abs() + e) + 4 * U * want.abs() + (0 if dres is None else 2 * U * dres.abs())
    # a chain over rows: a lane's share of them, 64 groups, the partial rows
    Dr = R / 128 + 128
    return (b + half_step(out, want), Dr * U * (dy * h).abs().sum(0) + half_step(weight, dg),
            Dr * U * dy.abs().sum(0) + half_step(weight, db))


def product_bound(a, b):
    """|error| of sum_k a[m, k] b[k, n] on the matrix cores, the framework's
    bar for contractions: 1e-5 sqrt(K) |a_m| |b_n|."""
    K = max(1, a.shape[1])
    return 1e-5 * math.sqrt(K) * a.norm(dim=1)[:, None] * b.norm(dim=0)[None, :]


def walk_bound(a, b):
    """|error| of the same sum where a and b are random of mean zero: the
    rounding errors of at most K + 64 additions (k, and the joins of waves and
    parts), each within a step, 2 U, of the partial sum there, add as a random
    walk. A partial sum is of the size of sqrt(sum a^2 b^2) or, on the way to a
    far result, of the result; eight deviations (Azuma: 2 exp(-32) an element).
    It is below what a partial sum rounded to 16 bits is off by."""
    K = max(1, a.shape[1])
    return 16 * U * math.sqrt(K + 64) * (((a * a) @ (b * b)).sqrt() + (a @ b).abs())


def act_error(z):
    """Relative error of an activation's or slope's terms in f32: the argument
    of exp or erfc carries a rounding of z^2 or z^3 (gelu_tanh: 1.6 z (1 +
    0.0447 z^2)), and each has a few roundings of its own."""
    return 4 * U * (16 + z * z + 0.3 * z.abs() ** 3)
