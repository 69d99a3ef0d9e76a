"""Operator programs: layer norm, projections with an epilogue and gated
projections, forward and backward (include/tca_op.h has the mathematics, the
tensors of each and what may overlap).

A function here names an operator and its attributes and returns an
``Operator``, which compiles and launches like a built DSL program:

    from tcacomp_amd import compiler, operators

    up = compiler.compile_program(operators.gated("bf16", save=True))
    up.launch([x, wg, wu, h, g, u])                       # x [M, K], w [K, N], h [M, N]

    norm = compiler.compile_program(operators.layer_norm("bf16", stats=True))
    norm.launch([x, gamma, beta, y, mean, rstd], scalars=(1e-5,))

Tensors are row-major, 16-byte aligned at their start, and of any extents; a
call's tensors are its inputs in order, then its outputs. ``elem`` is a name
("f32", "bf16", "f16") or an element type of ``pkg``. An attribute that the
operator does not take is refused with ``BuildError`` when it is made. There
is no counterpart in the reference: its DSL has no backward pass and stores
contractions in f32.
"""
import ctypes

from . import _lib
from .pkg import ELEM_NAMES, BuildError, _take_result


class Operator:
    """An operator and its attributes: what compiler.compile_program takes."""

    def __init__(self, op, attributes):
        self.op, self.attributes = op, attributes
        self.name = None
        self.emit()

    def emit(self, kernel_name=None, target=None, flags=0):
        """The emitted program (pkg.EmitResult). Operators take no emit
        flags, and their symbols carry the program's own name."""
        if flags or kernel_name:
            raise BuildError("operator %s takes no emit flags and no kernel name" % self.op)
        L = _lib.lib()
        out = ctypes.c_void_p()
        rc = L.tca_op_emit(self.op.encode(), self.attributes.encode(), target.encode() if target else None,
                           ctypes.byref(out))
        if rc != 0:
            raise BuildError(L.tca_op_last_error().decode())
        self.name = L.tca_op_program_name(out).decode()
        return _take_result(out)

    def __repr__(self):
        return "Operator(%s %s)" % (self.op, self.attributes)


def _elem(elem):
    return ELEM_NAMES[elem] if isinstance(elem, int) else str(elem)


def _make(op, elem, act=None, weight=None, **flags):
    words = ["elem=" + _elem(elem)]
    if weight is not None:
        words.append("weight=" + _elem(weight))
    if act is not None:
        words.append("act=" + act)
    return Operator(op, " ".join(words + [f for f, on in flags.items() if on]))


def layer_norm(elem, weight=None, bias=True, stats=False):
    """x [R, C], gamma [C], (beta [C]) -> y [R, C], (mean [R], rstd [R]);
    scalars (eps,). `weight` f32 keeps gamma and beta in f32 beside 16-bit
    rows; `stats` stores what the backward pass reads."""
    return _make("layer_norm", elem, weight=_weight(elem, weight), nobias=not bias, stats=stats)


def layer_norm_backward(elem, weight=None, bias=True, residual=False):
    """dy, x [R, C], gamma [C], mean, rstd [R], (dres [R, C]) -> dx [R, C],
    dgamma [C], (dbeta [C]). `residual` adds dres, the gradient that reaches
    x past the norm; dx may be dres."""
    return _make("layer_norm_backward", elem, weight=_weight(elem, weight), nobias=not bias, residual=residual)


def _weight(elem, weight):
    return None if weight is None or _elem(weight) == _elem(elem) else weight


def linear(elem, act="none", bias=False, residual=False, save=False):
    """x [M, K], w [K, N], (b [N]), (res [M, N]) -> y [M, N], (z [M, N]) with
    y = res + act(z), z = x w + b. `save` stores z for the backward pass;
    y may be res."""
    return _make("linear", elem, act=act, bias=bias, residual=residual, save=save)


def linear_backward(elem, act="none", bias=False):
    """dy [M, N], x [M, K], w [K, N], (z [M, N]) -> (dz [M, N]), dx [M, K],
    dw [K, N], (db [N]); z and dz with an activation. The residual's gradient
    is dy itself."""
    return _make("linear_backward", elem, act=act, bias=bias)


def gated(elem, act="silu", bias=False, save=False):
    """x [M, K], wg, wu [K, N], (bg, bu [N]) -> h [M, N], (g, u [M, N]) with
    h = act(g) u, g = x wg + bg, u = x wu + bu."""
    return _make("gated", elem, act=act, bias=bias, save=save)


def gated_backward(elem, act="silu", bias=False):
    """dh [M, N], x [M, K], wg, wu [K, N], g, u [M, N] -> dg, du [M, N],
    dx [M, K], dwg, dwu [K, N], (dbg, dbu [N])."""
    return _make("gated_backward", elem, act=act, bias=bias)


def list_operators():
    """{operator: the attributes it takes} as the library lists them."""
    lines = _lib.lib().tca_op_list().decode().splitlines()
    return {l.split(" ", 1)[0]: l.split(" ", 1)[1] for l in lines}


def all_builds():
    """(name, factory, emit flags) of every operator program that build()
    compiles: forward and backward of each element type as models use them,
    and one program of each attribute and activation for the tests."""
    out = []

    def add(f, *a, **k):
        out.append(("op_%s_%d" % (f.__name__, len(out)), lambda: f(*a, **k), 0))

    for e in ("f32", "bf16", "f16"):
        add(layer_norm, e)
        add(layer_norm, e, stats=True)
        add(layer_norm_backward, e, residual=True)
    add(layer_norm, "bf16", weight="f32", stats=True)
    add(layer_norm, "f16", bias=False)
    add(layer_norm_backward, "bf16", weight="f32")
    add(layer_norm_backward, "f16", bias=False)
    for e in ("bf16", "f16"):
        add(linear, e, bias=True, residual=True)
        add(linear, e, act="gelu", bias=True)
        add(linear, e, act="gelu", bias=True, save=True)
        add(linear, e, act="gelu", bias=True, residual=True)
        add(linear_backward, e, act="gelu", bias=True)
        add(linear_backward, e, bias=True)
        add(gated, e)
        add(gated, e, save=True)
        add(gated_backward, e)
    add(linear, "bf16")
    add(linear, "bf16", act="relu", save=True)
    add(linear, "bf16", act="gelu_tanh", bias=True, save=True)
    add(linear, "f16", act="silu", residual=True, save=True)
    add(linear_backward, "bf16")
    add(linear_backward, "bf16", act="relu")
    add(linear_backward, "f16", act="silu")
    add(gated, "f16", act="gelu", bias=True, save=True)
    add(gated, "bf16", act="gelu_tanh", bias=True, save=True)
    add(gated, "bf16", act="none")
    add(gated, "bf16", act="relu", bias=True)
    add(gated_backward, "f16", act="gelu", bias=True)
    add(gated_backward, "bf16", act="gelu_tanh", bias=True)
    add(gated_backward, "bf16", act="none")
    return out
