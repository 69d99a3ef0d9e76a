"""Layer norm where a workgroup walks several rows, whose loads run a row ahead
of the one at hand: every form that holds a row, with rows that fill it and rows
that end inside it, at least two whole turns of its grid and part of a third."""
import pytest
import torch

import operators_ref as ref
from test_gpu_operators import EPS, close, empty, gen_of, program, rand
from tcacomp_amd import operators

# (lanes, vectors of 16 bytes) that hold a row; workgroups launched at most.
FORWARD = [((16, 1), 2048), ((64, 1), 2048), ((64, 2), 2048), ((64, 4), 2048), ((256, 2), 2048), ((256, 4), 2048), ((1024, 2), 512),
           ((1024, 4), 512)]
BACKWARD = [((16, 1), 256), ((64, 1), 256), ((64, 2), 256), ((256, 1), 256), ((256, 2), 256), ((512, 2), 256), ((512, 4), 256)]


def cases(forms, block, elem):
    """(R, C) of each form: its longest row, and one that ends inside its last vector."""
    e = 4 if elem == "f32" else 8
    for (lanes, vectors), most in forms:
        if vectors == 4 and block == 512 and e == 8:
            continue  # (backward: 16-bit rows of that length are read twice)
        groups = max(1, block // lanes)
        for C in (lanes * vectors * e, lanes * vectors * e - e - 3):
            yield 2 * most * groups + groups + 1, C, "_%dx%d" % (lanes, vectors), most


@pytest.mark.parametrize("elem", ["f32", "bf16", "f16"])
def test_the_forms_and_their_turns(elem):
    """The grid that each case is launched on, without a GPU."""
    from test_operators import compiled, desc, norm_tensors, selected
    f, b = compiled(operators.layer_norm(elem)), compiled(operators.layer_norm_backward(elem))
    for R, C, form, most in cases(FORWARD, 256, elem):
        assert selected(f, norm_tensors(elem, R, C)) == {"tca_" + f.name + form: most}, (R, C)
    for R, C, form, most in cases(BACKWARD, 512, elem):
        t = [desc(elem, R, C), desc(elem, R, C), desc(elem, C), desc("f32", R), desc("f32", R), desc(elem, R, C), desc(elem, C), desc(elem, C)]
        assert selected(b, t)["tca_" + b.name + form] == most, (R, C)


@pytest.mark.gpu
@pytest.mark.parametrize("elem", ["f32", "bf16", "f16"])
def test_layer_norm_walks_rows(gpu, elem):
    for R, C, form, _ in cases(FORWARD, 256, elem):
        print("walk", elem, R, C, form, flush=True)
        g = gen_of("walk", R, C)
        x = rand(g, (R, C), elem, 1.5, 0.75)
        gamma, beta = rand(g, (C,), elem, 0.3, 1.0), rand(g, (C,), elem, 0.5)
        y, mean, rstd = empty((R, C), elem), empty((R,), "f32"), empty((R,), "f32")
        program(operators.layer_norm, elem, stats=True).launch([x, gamma, beta, y, mean, rstd], scalars=(EPS,))
        args = [t.double() for t in (x, gamma, beta)]
        for got, w, b, what in zip((y, mean, rstd), ref.layer_norm(*args, EPS), ref.layer_norm_bounds(*args, EPS, ref.DTYPES[elem]),
                                   ("y", "mean", "rstd")):
            close(got, w, b, what)


@pytest.mark.gpu
@pytest.mark.parametrize("elem", ["f32", "bf16", "f16"])
def test_layer_norm_backward_walks_rows(gpu, elem):
    t = ref.DTYPES[elem]
    long = [(2300, 16400, "_long", 32)]  # rows read twice, 32 chunks of 72 rows of the columns' pass
    for R, C, form, _ in list(cases(BACKWARD, 512, elem)) + long:
        print("walk back", elem, R, C, form, flush=True)
        g = gen_of("walkb", R, C)
        x, dy, dres = rand(g, (R, C), elem, 1.5, 0.75), rand(g, (R, C), elem), rand(g, (R, C), elem)
        gamma = rand(g, (C,), elem, 0.3, 1.0)
        mean = x.float().mean(1)
        rstd = (x.float().var(1, unbiased=False) + EPS).rsqrt()
        dx, dg, db = empty((R, C), elem), empty((C,), elem), empty((C,), elem)
        program(operators.layer_norm_backward, elem, residual=True).launch([dy, x, gamma, mean, rstd, dres, dx, dg, db])
        args = [v.double() for v in (dy, x, gamma, mean, rstd, dres)]
        for got, w, b, what in zip((dx, dg, db), ref.layer_norm_backward(*args), ref.layer_norm_backward_bounds(*args, t, t),
                                   ("dx", "dgamma", "dbeta")):
            close(got, w, b, what)
