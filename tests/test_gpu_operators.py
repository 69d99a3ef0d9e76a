"""The operator programs on the GPU against their definitions in 64 bits
(operators_ref.py), with bounds derived there: rows and products from one
element to several tiles, odd sizes, every type and attribute, empty extents,
in-place residuals, values that are not finite, captured graphs."""
import zlib

import pytest
import torch

import operators_ref as ref
from tcacomp_amd import _lib, compiler, operators

pytestmark = pytest.mark.gpu
EPS = 1e-5
_programs = {}


def program(f, *a, **k):
    key = (f.__name__, a, tuple(sorted(k.items())))
    if key not in _programs:
        _programs[key] = compiler.compile_program(f(*a, **k))
    return _programs[key]


def rand(gen, shape, elem, scale=1.0, shift=0.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale + shift).to(ref.DTYPES[elem])


def gen_of(*seed):
    return torch.Generator(device="cuda").manual_seed(zlib.crc32(repr(seed).encode()))


def empty(shape, elem):
    """Filled, so that an element left unwritten shows."""
    return torch.full(shape, -12345.0, device="cuda", dtype=ref.DTYPES[elem])


def close(got, want, bound, what):
    got = got.double()
    assert got.shape == want.shape, what
    if not want.numel():
        return
    r = (got - want).abs() / bound
    worst = float(r.max())
    print("%s: worst error / bound %.3g" % (what, worst), flush=True)
    assert worst <= 1.0, "%s: element %d is %g off its bound" % (what, int(r.argmax()), worst)


# ------------------------------------------------------------- layer norm

ROWS = [(1, 1), (3, 7), (5, 8), (70, 64), (17, 129), (33, 512), (9, 1000), (5, 1024), (1, 2048), (6, 2049),
        (2, 4097), (3, 8192), (2, 8200), (2, 16385), (3, 32768), (2, 40001)]


@pytest.mark.parametrize("elem", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("R,C", ROWS)
def test_layer_norm(gpu, R, C, elem):
    print("layer_norm", R, C, elem, flush=True)
    g = gen_of("ln", R, C)
    x = rand(g, (R, C), elem, 1.5, 0.75)
    gamma, beta = rand(g, (C,), elem, 0.3, 1.0), rand(g, (C,), elem, 0.5)
    y, mean, rstd = empty((R, C), elem), empty((R,), "f32"), empty((R,), "f32")
    program(operators.layer_norm, elem, stats=True).launch([x, gamma, beta, y, mean, rstd], scalars=(EPS,))
    args = [t.double() for t in (x, gamma, beta)]
    want = ref.layer_norm(*args, EPS)
    bounds = ref.layer_norm_bounds(*args, EPS, ref.DTYPES[elem])
    for got, w, b, what in zip((y, mean, rstd), want, bounds, ("y", "mean", "rstd")):
        close(got, w, b, what)


def test_layer_norm_f32_weights_and_no_bias(gpu):
    g = gen_of("lnw")
    x = rand(g, (37, 1501), "bf16", 2.0, -1.0)
    gamma, beta = rand(g, (1501,), "f32", 0.3, 1.0), rand(g, (1501,), "f32", 0.5)
    y, mean, rstd = empty((37, 1501), "bf16"), empty((37,), "f32"), empty((37,), "f32")
    program(operators.layer_norm, "bf16", weight="f32", stats=True).launch([x, gamma, beta, y, mean, rstd], scalars=(EPS,))
    args = [t.double() for t in (x, gamma, beta)]
    close(y, ref.layer_norm(*args, EPS)[0], ref.layer_norm_bounds(*args, EPS, torch.bfloat16)[0], "f32 weights")
    x, gamma, y = x.half(), gamma.half(), empty((37, 1501), "f16")
    program(operators.layer_norm, "f16", bias=False).launch([x, gamma, y], scalars=(EPS,))
    x, gamma = x.double(), gamma.double()
    close(y, ref.layer_norm(x, gamma, None, EPS)[0], ref.layer_norm_bounds(x, gamma, None, EPS, torch.float16)[0], "no bias")


def test_layer_norm_large_mean(gpu):
    """A row far from zero: the variance is that of the centred values."""
    for C in (1000, 40000):
        g = gen_of("lnm", C)
        x = rand(g, (8, C), "f32", 1.0, 3000.0)
        gamma, beta, y = rand(g, (C,), "f32"), rand(g, (C,), "f32"), empty((8, C), "f32")
        program(operators.layer_norm, "f32").launch([x, gamma, beta, y], scalars=(EPS,))
        args = [t.double() for t in (x, gamma, beta)]
        close(y, ref.layer_norm(*args, EPS)[0], ref.layer_norm_bounds(*args, EPS, torch.float32)[0], "mean 3000, C %d" % C)


BACK_ROWS = [(1, 1), (3, 7), (70, 64), (130, 128), (100, 300), (1001, 501), (517, 1501), (300, 2048), (40, 4100),
             (11, 8192), (5, 16384), (70, 16400)]


@pytest.mark.parametrize("elem", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("R,C", BACK_ROWS)
def test_layer_norm_backward(gpu, R, C, elem):
    print("layer_norm_backward", R, C, elem, flush=True)
    g = gen_of("lnb", R, C)
    x, dy, dres = rand(g, (R, C), elem, 1.5, 0.75), rand(g, (R, C), elem), rand(g, (R, C), elem)
    gamma = rand(g, (C,), elem, 0.3, 1.0)
    mean = x.float().mean(1)
    rstd = (x.float().var(1, unbiased=False) + EPS).rsqrt()
    dx, dg, db = empty((R, C), elem), empty((C,), elem), empty((C,), elem)
    program(operators.layer_norm_backward, elem, residual=True).launch([dy, x, gamma, mean, rstd, dres, dx, dg, db])
    args = [t.double() for t in (dy, x, gamma, mean, rstd, dres)]
    t = ref.DTYPES[elem]
    for got, w, b, what in zip((dx, dg, db), ref.layer_norm_backward(*args), ref.layer_norm_backward_bounds(*args, t, t),
                               ("dx", "dgamma", "dbeta")):
        close(got, w, b, what)


def test_layer_norm_backward_f32_weights_and_no_bias(gpu):
    R, C = 700, 1030
    g = gen_of("lnbw")
    x, dy = rand(g, (R, C), "bf16", 1.5, 0.75), rand(g, (R, C), "bf16")
    gamma = rand(g, (C,), "f32", 0.3, 1.0)
    mean, rstd = x.float().mean(1), (x.float().var(1, unbiased=False) + EPS).rsqrt()
    dx, dg, db = empty((R, C), "bf16"), empty((C,), "f32"), empty((C,), "f32")
    program(operators.layer_norm_backward, "bf16", weight="f32").launch([dy, x, gamma, mean, rstd, dx, dg, db])
    args = [t.double() for t in (dy, x, gamma, mean, rstd)] + [None]
    for got, w, b, what in zip((dx, dg, db), ref.layer_norm_backward(*args),
                               ref.layer_norm_backward_bounds(*args, torch.bfloat16, torch.float32), ("dx", "dgamma", "dbeta")):
        close(got, w, b, what)
    x, dy, gamma = x.half(), dy.half(), gamma.half()
    dx, dg = empty((R, C), "f16"), empty((C,), "f16")
    program(operators.layer_norm_backward, "f16", bias=False).launch([dy, x, gamma, mean, rstd, dx, dg])
    args = [t.double() for t in (dy, x, gamma, mean, rstd)] + [None]
    for got, w, b in zip((dx, dg), ref.layer_norm_backward(*args), ref.layer_norm_backward_bounds(*args, torch.float16, torch.float16)):
        close(got, w, b, "no bias")


def test_layer_norm_empty(gpu):
    """No rows: zero gradients; rows of nothing: a mean and rstd of NaN."""
    z = lambda *s, elem="bf16": torch.empty(s, device="cuda", dtype=ref.DTYPES[elem])  # noqa: E731
    dg, db = empty((300,), "bf16"), empty((300,), "bf16")
    program(operators.layer_norm_backward, "bf16", residual=True).launch(
        [z(0, 300), z(0, 300), torch.ones(300, device="cuda").bfloat16(), z(0, elem="f32"), z(0, elem="f32"), z(0, 300), z(0, 300), dg, db])
    assert not dg.any() and not db.any()
    dg, db = empty((17000,), "bf16"), empty((17000,), "bf16")
    program(operators.layer_norm_backward, "bf16", residual=True).launch(
        [z(0, 17000), z(0, 17000), torch.ones(17000, device="cuda").bfloat16(), z(0, elem="f32"), z(0, elem="f32"), z(0, 17000),
         z(0, 17000), dg, db])
    assert not dg.any() and not db.any()
    mean, rstd = empty((5,), "f32"), empty((5,), "f32")
    program(operators.layer_norm, "bf16", stats=True).launch([z(5, 0), z(0), z(0), z(5, 0), mean, rstd], scalars=(EPS,))
    assert mean.isnan().all() and rstd.isnan().all()


def test_layer_norm_not_finite(gpu):
    """A NaN or an infinity stays in its row (and in its columns' gradients)."""
    for C in (40, 600, 5000, 40000):
        g = gen_of("lnn", C)
        x, gamma, beta = rand(g, (7, C), "f32"), rand(g, (C,), "f32"), rand(g, (C,), "f32")
        clean, y = empty((7, C), "f32"), empty((7, C), "f32")
        p = program(operators.layer_norm, "f32")
        p.launch([x, gamma, beta, clean], scalars=(EPS,))
        x[2, C // 2], x[5, C - 1] = float("nan"), float("inf")
        p.launch([x, gamma, beta, y], scalars=(EPS,))
        for r in range(7):
            assert bool(y[r].isnan().all()) if r in (2, 5) else torch.equal(y[r], clean[r]), (C, r)


def test_layer_norm_backward_in_place_residual(gpu):
    for R, C in ((130, 1501), (6, 17001)):
        g = gen_of("lnip", C)
        x, dy, dres = rand(g, (R, C), "bf16"), rand(g, (R, C), "bf16"), rand(g, (R, C), "bf16")
        gamma = rand(g, (C,), "bf16")
        mean, rstd = x.float().mean(1), (x.float().var(1, unbiased=False) + EPS).rsqrt()
        p = program(operators.layer_norm_backward, "bf16", residual=True)
        dx, dg, db = empty((R, C), "bf16"), empty((C,), "bf16"), empty((C,), "bf16")
        p.launch([dy, x, gamma, mean, rstd, dres, dx, dg, db])
        p.launch([dy, x, gamma, mean, rstd, dres, dres, dg, db])
        assert torch.equal(dx, dres)


# --------------------------------------------------------------- products

SHAPES = [(1, 1, 1), (3, 5, 7), (1, 64, 64), (2, 200, 300), (16, 128, 136), (17, 100, 33), (64, 72, 264), (65, 130, 131),
          (128, 64, 128), (200, 72, 264), (130, 1003, 150), (257, 515, 1026), (300, 328, 520)]
LINEAR = [("bf16", dict(bias=True, residual=True)), ("f16", dict(act="gelu", bias=True, residual=True)),
          ("bf16", dict(act="gelu", bias=True, save=True))]


def check_linear(elem, M, K, N, act="none", bias=False, residual=False, save=False):
    g = gen_of("lin", M, K, N)
    x, w = rand(g, (M, K), elem), rand(g, (K, N), elem, max(K, 1) ** -0.5)
    b, res = rand(g, (N,), elem, 0.5), rand(g, (M, N), elem)
    y, z = empty((M, N), elem), empty((M, N), elem)
    p = program(operators.linear, elem, act=act, bias=bias, residual=residual, save=save)
    p.launch([x, w] + [b] * bias + [res] * residual + [y] + [z] * save)
    t = ref.DTYPES[elem]
    x, w, b, res = (v.double() for v in (x, w, b, res))
    want_z = x @ w + (b if bias else 0)
    e_z = ref.product_bound(x, w) + 2 * ref.U * want_z.abs() + 1e-30
    a = ref.act(act, want_z)
    want = a + (res if residual else 0)
    # |act'| is at most 1.13 for every activation
    e_y = 1.2 * e_z + a.abs() * ref.act_error(want_z) + 2 * ref.U * want.abs()
    close(y, want, e_y + ref.half_step(t, want), "y")
    if save:
        close(z, want_z, e_z + ref.half_step(t, want_z), "z")


@pytest.mark.parametrize("elem,attrs", LINEAR, ids=["residual", "gelu_residual_f16", "gelu_save"])
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_linear(gpu, M, K, N, elem, attrs):
    print("linear", M, K, N, elem, attrs, flush=True)
    check_linear(elem, M, K, N, **attrs)


@pytest.mark.parametrize("elem,attrs", [
    ("bf16", dict()), ("bf16", dict(act="relu", save=True)), ("bf16", dict(act="gelu_tanh", bias=True, save=True)),
    ("f16", dict(act="silu", residual=True, save=True))], ids=["plain", "relu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("M,K,N", [(5, 96, 200), (150, 250, 171)])
def test_linear_attributes(gpu, M, K, N, elem, attrs):
    check_linear(elem, M, K, N, **attrs)


def gated_bounds(x, wg, wu, bg, bu, act, t):
    g, u = x @ wg + bg, x @ wu + bu
    e_g = ref.product_bound(x, wg) + 2 * ref.U * g.abs() + 1e-30
    e_u = ref.product_bound(x, wu) + 2 * ref.U * u.abs() + 1e-30
    a = ref.act(act, g)
    h = a * u
    e_a = 1.2 * e_g + a.abs() * ref.act_error(g)
    e_h = e_a * u.abs() + a.abs() * e_u + e_a * e_u + 2 * ref.U * h.abs()
    return [(h, e_h + ref.half_step(t, h)), (g, e_g + ref.half_step(t, g)), (u, e_u + ref.half_step(t, u))]


def check_gated(elem, M, K, N, act="silu", bias=False, save=False):
    g = gen_of("gated", M, K, N)
    x, wg, wu = rand(g, (M, K), elem), rand(g, (K, N), elem, max(K, 1) ** -0.5), rand(g, (K, N), elem, max(K, 1) ** -0.5)
    bg, bu = rand(g, (N,), elem, 0.5), rand(g, (N,), elem, 0.5)
    outs = [empty((M, N), elem) for _ in range(3 if save else 1)]
    program(operators.gated, elem, act=act, bias=bias, save=save).launch([x, wg, wu] + [bg, bu] * bias + outs)
    bg, bu = (bg.double(), bu.double()) if bias else (0.0, 0.0)
    for got, (w, b), what in zip(outs, gated_bounds(x.double(), wg.double(), wu.double(), bg, bu, act, ref.DTYPES[elem]), "hgu"):
        close(got, w, b, what)


@pytest.mark.parametrize("elem,save", [("bf16", True), ("f16", False)])
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_gated(gpu, M, K, N, elem, save):
    print("gated", M, K, N, elem, save, flush=True)
    check_gated(elem, M, K, N, save=save)


@pytest.mark.parametrize("elem,attrs", [
    ("f16", dict(act="gelu", bias=True, save=True)), ("bf16", dict(act="gelu_tanh", bias=True, save=True)),
    ("bf16", dict(act="none")), ("bf16", dict(act="relu", bias=True))], ids=["gelu", "gelu_tanh", "none", "relu"])
@pytest.mark.parametrize("M,K,N", [(5, 96, 200), (150, 250, 171)])
def test_gated_attributes(gpu, M, K, N, elem, attrs):
    check_gated(elem, M, K, N, **attrs)


def sum_bound(parts, t):
    """A column sum in chains of a lane's rows, 4 rows and the partial rows."""
    return (parts.shape[0] / 64 + 160) * ref.U * parts.abs().sum(0) + ref.half_step(t, parts.sum(0))


def check_linear_backward(elem, M, K, N, act="none", bias=False):
    g = gen_of("linb", M, K, N)
    t = ref.DTYPES[elem]
    dy, x, w = rand(g, (M, N), elem), rand(g, (M, K), elem), rand(g, (K, N), elem, max(K, 1) ** -0.5)
    z, dz = rand(g, (M, N), elem, 1.5), empty((M, N), elem)
    dx, dw, db = empty((M, K), elem), empty((K, N), elem), empty((N,), elem)
    has = act != "none"
    program(operators.linear_backward, elem, act=act, bias=bias).launch(
        [dy, x, w] + [z] * has + [dz] * has + [dx, dw] + [db] * bias)
    want_dz = dy.double() * ref.slope(act, z.double())
    e_dz = dy.double().abs() * 1.2 * ref.act_error(z.double()) + 2 * ref.U * want_dz.abs()
    if has:
        close(dz, want_dz, e_dz + ref.half_step(t, want_dz), "dz")
    used = (dz if has else dy).double()
    x, w = x.double(), w.double()
    want = used @ w.T
    close(dx, want, ref.product_bound(used, w.T) + ref.half_step(t, want) + 1e-30, "dx")
    want = x.T @ used
    close(dw, want, ref.product_bound(x.T, used) + ref.half_step(t, want) + 1e-30, "dw")
    if bias:
        close(db, want_dz.sum(0), e_dz.sum(0) + sum_bound(want_dz, t), "db")


@pytest.mark.parametrize("elem", ["bf16", "f16"])
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_linear_backward(gpu, M, K, N, elem):
    print("linear_backward", M, K, N, elem, flush=True)
    check_linear_backward(elem, M, K, N, act="gelu", bias=True)


@pytest.mark.parametrize("elem,attrs", [("bf16", dict()), ("bf16", dict(act="relu")), ("f16", dict(act="silu")),
                                        ("bf16", dict(bias=True)), ("f16", dict(bias=True))],
                         ids=["plain", "relu", "silu", "bias", "bias_f16"])
@pytest.mark.parametrize("M,K,N", [(5, 96, 200), (150, 250, 171), (3000, 40, 24)])
def test_linear_backward_attributes(gpu, M, K, N, elem, attrs):
    check_linear_backward(elem, M, K, N, **attrs)


def check_gated_backward(elem, M, K, N, act="silu", bias=False):
    gen = gen_of("gatedb", M, K, N)
    t = ref.DTYPES[elem]
    dh, x = rand(gen, (M, N), elem), rand(gen, (M, K), elem)
    wg, wu = rand(gen, (K, N), elem, max(K, 1) ** -0.5), rand(gen, (K, N), elem, max(K, 1) ** -0.5)
    g, u = rand(gen, (M, N), elem, 1.5), rand(gen, (M, N), elem)
    dg, du, dx = empty((M, N), elem), empty((M, N), elem), empty((M, K), elem)
    dwg, dwu, dbg, dbu = empty((K, N), elem), empty((K, N), elem), empty((N,), elem), empty((N,), elem)
    program(operators.gated_backward, elem, act=act, bias=bias).launch(
        [dh, x, wg, wu, g, u, dg, du, dx, dwg, dwu] + [dbg, dbu] * bias)
    d, gd, ud = dh.double(), g.double(), u.double()
    want_g, want_u = d * ud * ref.slope(act, gd), d * ref.act(act, gd)
    e_g = (d * ud).abs() * 1.2 * ref.act_error(gd) + 3 * ref.U * want_g.abs()
    e_u = want_u.abs() * (ref.act_error(gd) + 2 * ref.U)
    close(dg, want_g, e_g + ref.half_step(t, want_g), "dg")
    close(du, want_u, e_u + ref.half_step(t, want_u), "du")
    a, b, x, wg, wu = (v.double() for v in (dg, du, x, wg, wu))
    want = a @ wg.T + b @ wu.T
    close(dx, want, ref.product_bound(torch.cat([a, b], 1), torch.cat([wg, wu], 1).T) + ref.half_step(t, want) + 1e-30, "dx")
    for got, v, what in ((dwg, a, "dwg"), (dwu, b, "dwu")):
        want = x.T @ v
        close(got, want, ref.product_bound(x.T, v) + ref.half_step(t, want) + 1e-30, what)
    if bias:
        close(dbg, want_g.sum(0), e_g.sum(0) + sum_bound(want_g, t), "dbg")
        close(dbu, want_u.sum(0), e_u.sum(0) + sum_bound(want_u, t), "dbu")


@pytest.mark.parametrize("elem", ["bf16", "f16"])
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_gated_backward(gpu, M, K, N, elem):
    print("gated_backward", M, K, N, elem, flush=True)
    check_gated_backward(elem, M, K, N)


@pytest.mark.parametrize("elem,attrs", [("f16", dict(act="gelu", bias=True)), ("bf16", dict(act="gelu_tanh", bias=True)),
                                        ("bf16", dict(act="none"))], ids=["gelu", "gelu_tanh", "none"])
@pytest.mark.parametrize("M,K,N", [(5, 96, 200), (150, 250, 171), (3000, 40, 24)])
def test_gated_backward_attributes(gpu, M, K, N, elem, attrs):
    check_gated_backward(elem, M, K, N, **attrs)


@pytest.mark.parametrize("M,K,N", [(3592, 72, 3608), (3592, 264, 3600), (2056, 72, 3080), (1032, 40, 3080), (1504, 72, 2904),
                                   (1000, 40, 2304), (1032, 72, 1608)])
def test_large_planes(gpu, M, K, N):
    """Planes of many tiles, their last row and column of tiles partial, a
    reduction that ends inside a slice."""
    print("large planes", M, K, N, flush=True)
    check_linear("bf16", M, K, N, act="gelu", bias=True, residual=True)
    check_gated("f16", M, K, N, save=True)
    check_linear_backward("bf16", K, M, N, act="gelu", bias=True)  # dw of M x N
    check_gated_backward("f16", K, M, N)
    check_linear_backward("f16", M, N, K, bias=True)  # dx of M x N
    check_gated_backward("bf16", M, N, K)


def test_products_empty(gpu):
    """K = 0 leaves the bias and the residual; no tokens, zero weight gradients."""
    check_linear("bf16", 70, 0, 200, bias=True, residual=True)
    check_linear("bf16", 3, 0, 20, act="gelu", bias=True, save=True)
    check_gated("bf16", 70, 0, 90, save=True)
    check_gated("bf16", 3, 0, 90, save=True)
    for M, K, N in ((0, 40, 64), (30, 0, 64), (30, 40, 0)):
        check_linear("bf16", M, K, N, bias=True, residual=True)
        check_gated("bf16", M, K, N, save=True)
        check_linear_backward("bf16", M, K, N, act="gelu", bias=True)
        check_gated_backward("f16", M, K, N, act="gelu", bias=True)


def test_products_not_finite(gpu):
    """An infinity in one row of x, or in one column of w, stays there, in
    every row length that a slice of k ends inside of."""
    for M, K, N in ((5, 67, 90), (140, 130, 200), (140, 96, 264), (300, 67, 520)):
        g = gen_of("nf", M, K, N)
        x, w = rand(g, (M, K), "bf16"), rand(g, (K, N), "bf16")
        p = program(operators.linear, "bf16")
        clean, y = empty((M, N), "bf16"), empty((M, N), "bf16")
        p.launch([x, w, clean])
        x[1, K - 1], x[3, 0] = float("inf"), float("nan")
        w[K - 1, N - 1] = float("inf")
        p.launch([x, w, y])
        bad = torch.zeros((M, N), dtype=torch.bool, device="cuda")
        bad[1], bad[3], bad[:, N - 1] = True, True, True
        assert bool((~y[bad].isfinite()).all()) and torch.equal(y[~bad], clean[~bad]), (M, K, N)


@pytest.mark.parametrize("elem,act,bias", [("bf16", "silu", False), ("bf16", "gelu_tanh", True), ("f16", "gelu", True)])
def test_slopes_far_out(gpu, elem, act, bias):
    """Pre-activations of up to the type's largest value: a slope of exactly 1 or 0,
    a value of exactly g or 0, never a product of 0 and an overflow."""
    top = float(torch.finfo(ref.DTYPES[elem]).max)
    far = [v for v in (200.0, 1e4, 6e4, 1e13, 1e15, 1e19, 1e25, top) if v <= top]
    g = torch.tensor([[s * v for v in far for s in (1, -1)]], device="cuda").to(ref.DTYPES[elem])
    N = g.shape[1]
    one, w, x = torch.ones_like(g), rand(gen_of("far"), (8, N), elem), rand(gen_of("far"), (1, 8), elem)
    dg, du, dx, dwg, dwu = empty((1, N), elem), empty((1, N), elem), empty((1, 8), elem), empty((8, N), elem), empty((8, N), elem)
    db = [empty((N,), elem), empty((N,), elem)] * bias
    program(operators.gated_backward, elem, act=act, bias=bias).launch([one, x, w, w, g, one, dg, du, dx, dwg, dwu] + db)
    zero = torch.zeros_like(g)
    assert torch.equal(dg, torch.where(g > 0, one, zero)) and torch.equal(du, torch.where(g > 0, g, zero)), (dg, du)


def test_linear_in_place_residual(gpu):
    for M, K, N in ((3, 130, 200), (140, 96, 264), (260, 77, 301)):
        g = gen_of("lip", M, K, N)
        x, w, b, res = rand(g, (M, K), "bf16"), rand(g, (K, N), "bf16"), rand(g, (N,), "bf16"), rand(g, (M, N), "bf16")
        p = program(operators.linear, "bf16", bias=True, residual=True)
        y = empty((M, N), "bf16")
        p.launch([x, w, b, res, y])
        p.launch([x, w, b, res, res])
        assert torch.equal(y, res)


def test_runs_repeat_bit_for_bit(gpu):
    """No result depends on the order in which workgroups end."""
    g = gen_of("rep")
    x, w, b, res = rand(g, (7, 3000), "bf16"), rand(g, (3000, 640), "bf16"), rand(g, (640,), "bf16"), rand(g, (7, 640), "bf16")
    p = program(operators.linear, "bf16", bias=True, residual=True)
    outs = [empty((7, 640), "bf16") for _ in range(5)]
    for y in outs:
        p.launch([x, w, b, res, y])
    assert all(torch.equal(outs[0], y) for y in outs)
    dy, xs = rand(g, (3000, 700), "bf16"), rand(g, (3000, 700), "bf16")
    gamma, mean, rstd = rand(g, (700,), "bf16"), xs.float().mean(1), xs.float().std(1).reciprocal()
    p = program(operators.layer_norm_backward, "bf16", residual=True)
    outs = []
    for _ in range(5):
        o = [empty((3000, 700), "bf16"), empty((700,), "bf16"), empty((700,), "bf16")]
        p.launch([dy, xs, gamma, mean, rstd, dy] + o)
        outs.append(o)
    assert all(torch.equal(a, b) for o in outs for a, b in zip(outs[0], o))


# ------------------------------------------------------ together, as used

class Sublayer:
    """x + W_down (gated (norm x)): the programs of a pre-norm feed-forward
    sublayer, forward and backward, and the tensors that they own."""

    def __init__(self, M, D, F, elem="bf16"):
        self.programs = dict(
            norm=program(operators.layer_norm, elem, stats=True), norm_b=program(operators.layer_norm_backward, elem, residual=True),
            up=program(operators.gated, elem, save=True), up_b=program(operators.gated_backward, elem),
            down=program(operators.linear, elem, bias=True, residual=True), down_b=program(operators.linear_backward, elem, bias=True))
        g = gen_of("sub", M, D, F)
        self.x = rand(g, (M, D), elem, 1.0, 0.3)
        self.w = dict(gamma=rand(g, (D,), elem, 0.2, 1.0), beta=rand(g, (D,), elem, 0.2), wg=rand(g, (D, F), elem, D ** -0.5),
                      wu=rand(g, (D, F), elem, D ** -0.5), wd=rand(g, (F, D), elem, F ** -0.5), b=rand(g, (D,), elem, 0.2))
        self.dy = rand(g, (M, D), elem)
        e = lambda *s, t=elem: empty(s, t)  # noqa: E731
        self.t = dict(n=e(M, D), mean=e(M, t="f32"), rstd=e(M, t="f32"), h=e(M, F), g=e(M, F), u=e(M, F), y=e(M, D), dh=e(M, F),
                      dg=e(M, F), du=e(M, F), dn=e(M, D), dx=e(M, D))
        self.grads = {k: torch.empty_like(v) for k, v in self.w.items()}

    def step(self, noalloc=False):
        w, t, gr, p = self.w, self.t, self.grads, self.programs
        p["norm"].launch([self.x, w["gamma"], w["beta"], t["n"], t["mean"], t["rstd"]], scalars=(EPS,), noalloc=noalloc)
        p["up"].launch([t["n"], w["wg"], w["wu"], t["h"], t["g"], t["u"]], noalloc=noalloc)
        p["down"].launch([t["h"], w["wd"], w["b"], self.x, t["y"]], noalloc=noalloc)
        p["down_b"].launch([self.dy, t["h"], w["wd"], t["dh"], gr["wd"], gr["b"]], noalloc=noalloc)
        p["up_b"].launch([t["dh"], t["n"], w["wg"], w["wu"], t["g"], t["u"], t["dg"], t["du"], t["dn"], gr["wg"], gr["wu"]], noalloc=noalloc)
        p["norm_b"].launch([t["dn"], self.x, w["gamma"], t["mean"], t["rstd"], self.dy, t["dx"], gr["gamma"], gr["beta"]], noalloc=noalloc)

    def outputs(self):
        return {"y": self.t["y"], "dx": self.t["dx"], **self.grads}

    def exact(self):
        leaves = {k: v.double().requires_grad_() for k, v in {"x": self.x, **self.w}.items()}
        n = ref.layer_norm(leaves["x"], leaves["gamma"], leaves["beta"], EPS)[0]
        h = ref.act("silu", n @ leaves["wg"]) * (n @ leaves["wu"])
        y = leaves["x"] + h @ leaves["wd"] + leaves["b"]
        y.backward(self.dy.double())
        return {"y": y.detach(), "dx": leaves["x"].grad, **{k: leaves[k].grad for k in self.w}}


@pytest.mark.parametrize("M,D,F", [(3, 64, 200), (100, 128, 344), (257, 130, 515)])
def test_sublayer_forward_and_backward(gpu, M, D, F):
    """The programs one after the other against autograd in 64 bits. Each of
    the (at most nine) stored tensors between an input and a result is off by
    half a step at random: in the 2-norm their sum stays under the sum of
    their half steps."""
    s = Sublayer(M, D, F)
    s.step()
    for name, want in s.exact().items():
        off = float((s.outputs()[name].double() - want).norm() / want.norm())
        print(name, off, flush=True)
        assert off <= 9 * 2.0 ** -8, name


def test_sublayer_captured_and_replayed(gpu):
    """The step captured into a graph (no allocation while it is captured),
    replayed between the program's own eager steps, with new values in the
    same tensors: every replay equals the eager result."""
    s = Sublayer(200, 128, 344)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        s.step(noalloc=True)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.step(noalloc=True)
    g = gen_of("cap")
    for _ in range(4):
        s.x.copy_(rand(g, s.x.shape, "bf16"))
        s.dy.copy_(rand(g, s.dy.shape, "bf16"))
        s.step()
        torch.cuda.synchronize()
        want = {k: v.clone() for k, v in s.outputs().items()}
        for v in s.outputs().values():
            v.fill_(-1.0)
        graph.replay()
        torch.cuda.synchronize()
        for k, v in s.outputs().items():
            assert torch.equal(v, want[k]), k


def test_captured_workspace_outlives_a_larger_launch(gpu):
    """A graph keeps the workspace its launches were captured with when a
    later launch on that stream needs a larger one; and a launch that would
    have to allocate while its stream is captured is refused, the capture
    going on."""
    g = gen_of("capws")
    p = compiler.compile_program(operators.layer_norm_backward("bf16", residual=True))  # no workspaces yet

    def tensors(R, C):
        x, dy, dres = (rand(g, (R, C), "bf16") for _ in range(3))
        return [dy, x, rand(g, (C,), "bf16"), x.float().mean(1), x.float().std(1).reciprocal(), dres, empty((R, C), "bf16"),
                empty((C,), "bf16"), empty((C,), "bf16")]

    small, large = tensors(500, 300), tensors(700, 3000)
    p.launch(small)
    torch.cuda.synchronize()
    want = [t.clone() for t in small[6:]]
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        with pytest.raises(_lib.TcaError, match="being captured"):
            p.launch(small)
    with torch.cuda.stream(stream):
        p.launch(small)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        p.launch(small)
    for _ in range(3):
        with torch.cuda.stream(stream):
            p.launch(large)
        torch.cuda.synchronize()
        for t in small[6:]:
            t.fill_(-1.0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(t, w) for t, w in zip(small[6:], want))


def test_two_streams_at_once(gpu):
    """One program on two streams: each has a workspace of its own."""
    a, b = Sublayer(300, 128, 344), Sublayer(270, 256, 200)
    a.step()
    b.step()
    torch.cuda.synchronize()
    want = [{k: v.clone() for k, v in s.outputs().items()} for s in (a, b)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for s, st in zip((a, b), streams):
            with torch.cuda.stream(st):
                s.step()
    torch.cuda.synchronize()
    for s, w in zip((a, b), want):
        for k, v in s.outputs().items():
            assert torch.equal(v, w[k]), k


@pytest.mark.parametrize("N", [32768, 32767])
def test_planes_past_32_bit_offsets(gpu, N):
    """70000 rows: 2.3e9 elements, 4.6e9 bytes; the rows round the 2^31st element
    and the last ones, and the columns' sums over all rows."""
    M, K = 70000, 64
    g = gen_of("far", N)
    big = lambda: torch.empty((M, N), device="cuda", dtype=torch.bfloat16).normal_(generator=g)  # noqa: E731
    x, w = rand(g, (M, K), "bf16"), rand(g, (K, N), "bf16", K ** -0.5)
    rows, t = [0, 65535, 65536, 65537, M - 1], torch.bfloat16
    y = empty((M, N), "bf16")
    print("linear", flush=True)
    program(operators.linear, "bf16").launch([x, w, y])
    want = x[rows].double() @ w.double()
    close(y[rows], want, ref.product_bound(x[rows].double(), w.double()) + ref.half_step(t, want) + 1e-30, "y")
    print("layer_norm", flush=True)
    z, gamma, beta = big(), rand(g, (N,), "bf16", 0.3, 1.0), rand(g, (N,), "bf16", 0.5)
    program(operators.layer_norm, "bf16").launch([z, gamma, beta, y], scalars=(EPS,))
    args = [v.double() for v in (z[rows], gamma, beta)]
    close(y[rows], ref.layer_norm(*args, EPS)[0], ref.layer_norm_bounds(*args, EPS, t)[0], "norm")
    print("linear_backward", flush=True)
    dy, dz, dx, dw = y.normal_(generator=g), empty((M, N), "bf16"), empty((M, K), "bf16"), empty((K, N), "bf16")
    program(operators.linear_backward, "bf16", act="relu").launch([dy, x, w, z, dz, dx, dw])
    assert torch.equal(dz[rows], torch.where(z[rows] > 0, dy[rows], torch.zeros_like(dy[rows])))
    used = dz[rows].double()
    want = used @ w.double().T
    close(dx[rows], want, ref.product_bound(used, w.double().T) + ref.half_step(t, want) + 1e-30, "dx")
    used = dz[:, N - 40:].double()
    want = x.double().T @ used
    close(dw[:, N - 40:], want, ref.product_bound(x.double().T, used) + ref.half_step(t, want) + 1e-30, "dw")


def test_refusals_on_the_device(gpu):
    p = program(operators.linear, "bf16", bias=True, residual=True)
    t = lambda *s: torch.zeros(s, device="cuda", dtype=torch.bfloat16)  # noqa: E731
    with pytest.raises(_lib.TcaError, match="must equal"):
        p.launch([t(4, 8), t(9, 16), t(16), t(4, 16), t(4, 16)])
    with pytest.raises(_lib.TcaError, match="dtype"):
        p.launch([t(4, 8).float(), t(8, 16), t(16), t(4, 16), t(4, 16)])
    with pytest.raises(_lib.TcaError, match="16-byte aligned"):
        p.launch([t(4 * 8 + 1)[1:].view(4, 8), t(8, 16), t(16), t(4, 16), t(4, 16)])
    with pytest.raises(ValueError, match="contiguous"):
        p.launch([t(8, 4).t(), t(8, 16), t(16), t(4, 16), t(4, 16)])
    with pytest.raises(_lib.TcaError, match="takes 5 tensor"):
        p.launch([t(4, 8), t(8, 16), t(16), t(4, 16)])
    n = program(operators.layer_norm, "bf16")
    with pytest.raises(_lib.TcaError, match="scalar"):
        n.launch([t(4, 8), t(8), t(8), t(4, 8)])
