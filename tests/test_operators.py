"""The operator programs without a GPU: the definitions the GPU tests use
against differences and autograd, the emitted programs, which kernel a size
takes, and the refusals of the C ABI."""
import ctypes
import itertools
import subprocess

import pytest
import torch

import operators_ref as ref
from tcacomp_amd import _lib, build, compiler, operators
from tcacomp_amd.compiler import TensorDesc
from tcacomp_amd.pkg import TBF16, BuildError

ELEM_CODES = {"f32": 0, "f16": 1, "bf16": 2}


def desc(elem, *shape):
    return TensorDesc(16, shape, ELEM_CODES[elem])


def compiled(op):
    """Emission and plan only: no code object is needed."""
    return compiler.CompiledProgram(op.name, op.emit(), "")


# ------------------------------------------------------------ definitions

@pytest.mark.parametrize("name", ["none", "relu", "silu", "gelu", "gelu_tanh"])
def test_slopes_against_differences(name):
    z = torch.linspace(-6, 6, 241, dtype=torch.float64) + 0.0125  # no point at relu's corner
    d = 1e-6
    diff = (ref.act(name, z + d) - ref.act(name, z - d)) / (2 * d)
    # the difference's own error: d^2 / 6 of a third derivative below 3, and its cancellation
    assert (ref.slope(name, z) - diff).abs().max() <= d * d + 8 * 2.0 ** -53 / d * 7


def test_layer_norm_gradients_against_differences_and_autograd():
    torch.manual_seed(0)
    x, gamma, beta, dy, dres = (torch.randn(s, dtype=torch.float64) for s in ((3, 5), (5,), (5,), (3, 5), (3, 5)))
    _, mean, rstd = ref.layer_norm(x, gamma, beta, 1e-5)
    dx, dg, db = ref.layer_norm_backward(dy, x, gamma, mean, rstd, dres)
    leaves = [t.clone().requires_grad_() for t in (x, gamma, beta)]
    ((ref.layer_norm(*leaves, 1e-5)[0] * dy).sum() + (leaves[0] * dres).sum()).backward()
    for got, leaf in zip((dx, dg, db), leaves):
        assert torch.allclose(got, leaf.grad, rtol=1e-10, atol=1e-10)
    f = lambda v: (ref.layer_norm(v, gamma, beta, 1e-5)[0] * dy).sum() + (v * dres).sum()  # noqa: E731
    for i, j in itertools.product(range(3), range(5)):
        e = torch.zeros_like(x)
        e[i, j] = 1e-5
        assert abs(float((f(x + e) - f(x - e)) / 2e-5 - dx[i, j])) < 1e-6


# --------------------------------------------------------------- emission

def test_attributes_in_any_order_are_one_program():
    L = _lib.lib()
    seen = set()
    for words in itertools.permutations(["elem=bf16", "act=gelu", "bias", "save"]):
        out = ctypes.c_void_p()
        assert L.tca_op_emit(b"linear", " ".join(words).encode(), None, ctypes.byref(out)) == 0
        seen.add((L.tca_op_program_name(out), L.tca_emit_plan(out), L.tca_emit_source(out)))
        L.tca_emit_free(out)
    assert len(seen) == 1


def test_elements_by_name_or_type():
    assert operators.gated(TBF16).name == operators.gated("bf16").name == "gated_bf16_silu"
    assert operators.layer_norm("bf16", weight="bf16").name == operators.layer_norm("bf16").name


def test_every_operator_is_listed_and_built():
    listed = operators.list_operators()
    assert set(listed) == {"layer_norm", "layer_norm_backward", "linear", "linear_backward", "gated", "gated_backward"}
    built = [f() for _, f, _ in operators.all_builds()]
    assert {o.op for o in built} == set(listed)
    assert len({o.name for o in built}) == len(built)


@pytest.mark.parametrize("op,attributes,word", [
    ("linear", "elem=f32", "elem=f32"), ("linear", "", "no elem"), ("linear", "elem=bf16 act=swish", "act=swish"),
    ("linear", "elem=bf16 stats", "stats"), ("linear", "elem=bf16 bias=1", "bias=1"), ("linear", "elem=bf16 elem=f16", "twice"),
    ("gated", "elem=bf16 residual", "residual"), ("gated_backward", "elem=bf16 save", "save"), ("linear", "elem=bf16 act", "act"),
    ("layer_norm", "elem=bf16 act=gelu", "act=gelu"), ("layer_norm", "elem=bf16 weight=f16", "weight=f16"), ("layer_norm", "elem=bf16 weight=elem", "weight=elem"),
    ("layer_norm", "elem=u8", "elem=u8"), ("linear_backward", "elem=bf16 residual", "residual")])
def test_refused_attributes(op, attributes, word):
    with pytest.raises(BuildError, match=word):
        operators.Operator(op, attributes)


def test_refusals_of_the_c_entry():
    L = _lib.lib()
    out = ctypes.c_void_p(7)
    assert L.tca_op_emit(None, b"elem=bf16", None, ctypes.byref(out)) == _lib.TCA_ERR_INVALID
    assert L.tca_op_emit(b"linear", b"elem=bf16", None, None) == _lib.TCA_ERR_INVALID
    assert L.tca_op_emit(b"conv", b"elem=bf16", None, ctypes.byref(out)) == _lib.TCA_ERR_NOT_FOUND
    assert out.value is None and b"no operator conv" in L.tca_op_last_error()
    assert L.tca_op_emit(b"linear", b"elem=bf16", b"gfx942", ctypes.byref(out)) == _lib.TCA_ERR_UNSUPPORTED
    assert b"gfx942" in L.tca_op_last_error()
    assert L.tca_op_emit(b"linear", None, None, ctypes.byref(out)) == _lib.TCA_ERR_UNSUPPORTED
    assert L.tca_op_program_name(None) is None
    with pytest.raises(BuildError, match="emit flags"):
        operators.linear("bf16").emit(flags=1)


# ------------------------------------------- which kernels a size takes

def norm_tensors(elem, R, C):
    return [desc(elem, R, C), desc(elem, C), desc(elem, C), desc(elem, R, C)]


@pytest.mark.parametrize("elem", ["f32", "bf16"])
def test_every_row_length_takes_one_norm_kernel(elem):
    p = compiled(operators.layer_norm(elem))
    lengths = sorted({c + d for e in range(3, 18) for c in (1 << e,) for d in (-1, 0, 1)} | {0, 1, 2, 100001})
    for C in lengths:
        assert len(p.selected_symbols(norm_tensors(elem, 3, C))) == 1, C


@pytest.mark.parametrize("elem", ["f32", "bf16"])
def test_every_row_length_takes_one_norm_backward_kernel(elem):
    p = compiled(operators.layer_norm_backward(elem))
    for C in sorted({c + d for e in range(3, 18) for c in (1 << e,) for d in (-1, 0, 1)} | {1, 2, 100001}):
        for R in (1, 5, 4000):
            t = [desc(elem, R, C), desc(elem, R, C), desc(elem, C), desc("f32", R), desc("f32", R), desc(elem, R, C),
                 desc(elem, C), desc(elem, C)]
            names = p.selected_symbols(t)
            assert [n.endswith("join") for n in names].count(True) == 1 and len(names) in (2, 3), (R, C, names)


def selected(p, tensors):
    """{symbol: grid} of the kernels a launch with these tensors runs."""
    L = _lib.lib()
    syms = p.kernel_symbols()
    out, grids = (ctypes.c_uint8 * len(syms))(), (ctypes.c_uint64 * len(syms))()
    fd = (ctypes.c_uint32 * 1)()
    _lib.check(L.tca_program_selected(p.parsed(), compiler._descriptors(tensors), len(tensors), fd, 0, out, grids, None, len(syms)))
    return {s: g for s, f, g in zip(syms, out, grids) if f and g}


def test_partial_rows_are_as_many_as_the_join_adds():
    """partial_rows on the device restates the grid of the kernel that writes
    the partial rows."""
    p = compiled(operators.layer_norm_backward("bf16"))
    for R, C in itertools.product((1, 3, 4, 5, 63, 64, 65, 255, 256, 257, 1023, 1024, 1025, 100000), (64, 300, 1000, 2000, 4000, 8000, 16000, 20000)):
        t = [desc("bf16", R, C), desc("bf16", R, C), desc("bf16", C), desc("f32", R), desc("f32", R), desc("bf16", R, C),
             desc("bf16", C), desc("bf16", C)]
        grids = selected(p, t)
        if C > 8192:
            parts = min(-(-R // 64), 32)
            assert grids["tca_" + p.name + "_columns"] == -(-C // 512) * parts
        else:
            (lanes, grid), = [(int(s.rsplit("_", 1)[1].split("x")[0]), g) for s, g in grids.items() if not s.endswith("join")]
            assert grid == min(-(-R // (512 // lanes)), 256)


def product_kernels(M, N, K, few, odd, half=1):
    """{suffix: workgroups} of one product of M x K by K x N (half 2: of two),
    by the rules restated, each as it is launched."""
    up = lambda a, b: -(-a // b)  # noqa: E731

    def shared(suffix, blocks, least):
        P = max(1, min(up(K, least), 256 // blocks))
        return {suffix: blocks * P, **({suffix.rstrip("0123456789") + "join": M * up(N, 256)} if P > 1 else {})}

    def tiles(rows, cols):
        return up(M, rows) * up(N, cols // half)

    if few and M <= 64:
        return shared("_few%d" % (16 if M <= 16 else 32 if M <= 32 else 64), up(N, 64), 256)
    if M * N <= 1 << 20:
        return shared("_o", tiles(64, 128), 512) if odd else shared("_k", tiles(128, 128), 512)
    if odd:
        return {"_a": tiles(128, 128)} if tiles(128, 128) >= 128 else {"": tiles(64, 128)}
    for form, rows, cols, least, of in (("_l", 256, 256, 385, (256, 256)), ("_m", 256, 128, 257, (256, 256)),
                                        ("_l", 256, 256, 257, (256, 128)), ("_m", 256, 128, 192, (256, 128)),
                                        ("_s", 128, 128, 257, (128, 128)), ("_r", 128, 128, 129, (128, 128))):
        if tiles(*of) >= least:
            return {form: tiles(rows, cols)}
    return {"_r": tiles(128, 128)} if half == 2 else {"_t": tiles(64, 128)}


def launched(p, plan, tensors, dims):
    """{suffix: workgroups} of a launch: the selected kernels, or the first of
    their forms whose bounds hold (plan: its kernel and form lines)."""
    out = {}
    for symbol, grid in selected(p, tensors).items():
        for name, bounds in plan[symbol]:
            counts = [(least, [dims[t.split("/")[0]] for t in terms], [int(t.split("/")[1]) for t in terms]) for least, terms in bounds]
            sizes = [-(-d[0] // q[0]) * -(-d[1] // q[1]) for _, d, q in counts]
            if all(size >= least for size, (least, _, _) in zip(sizes, counts)):
                symbol, grid = name, sizes[0]
                break
        out[symbol[len("tca_" + p.name):]] = grid
    return out


def forms(op):
    """{kernel: [(form, [(least, terms)])]} and all names of an operator's plan."""
    plan, last = {}, None
    for line in op.emit().plan.splitlines():
        w = line.split()
        if w and w[0] == "kernel":
            last = w[1]
            plan[last] = []
        elif w and w[0] == "form":
            assert w[2:4] == ["0", "2"] and w[5] == w[9] == "2" and len(w) == 12, line
            plan[last].append((w[1], [(int(w[4]), w[6:8]), (int(w[8]), w[10:12])]))
    return plan


SIZES = [1, 7, 8, 16, 17, 64, 65, 72, 128, 255, 512, 1000, 1024, 1032, 2048, 3600, 4096, 7297, 8192, 20000]


@pytest.mark.parametrize("gated", [False, True])
def test_every_product_takes_one_kernel(gated):
    """Forward and backward: one kernel for each product, with its join where
    k is split and only there, and as many workgroups as the kernel counts."""
    fop = (operators.gated if gated else operators.linear)("bf16", act="silu")
    bop = (operators.gated_backward if gated else operators.linear_backward)("bf16", act="silu")
    fwd, bwd, fplan, bplan = compiled(fop), compiled(bop), forms(fop), forms(bop)
    n = 2 if gated else 1
    seen = set()
    for M, K, N in itertools.product(SIZES, SIZES, SIZES):
        x, w, y, dims = desc("bf16", M, K), desc("bf16", K, N), desc("bf16", M, N), dict(M=M, K=K, N=N)
        got = launched(fwd, fplan, [x] + [w] * n + [y], dims)
        assert got == product_kernels(M, N, K, True, K % 8 or N % 8, half=n), dims
        seen |= {fwd.name + s for s in got}
        got = launched(bwd, bplan, [y, x] + [w] * n + [y] * n + [y] * n + [x] + [w] * n, dims)
        want = {"_slope": -(-M * N // 2048)}
        want.update({"_dx" + s: g for s, g in product_kernels(M, K, N, False, N % 8).items()})
        want.update({"_dw" + s: g for s, g in product_kernels(K, N, M, False, K % 8 or N % 8, half=n).items()})
        assert got == want, dims
        seen |= {bwd.name + s for s in got}
    # nothing in the programs that no size takes
    for plan in (fplan, bplan):
        assert {s[4:] for s in plan} | {f[0][4:] for of in plan.values() for f in of} <= seen


def test_shape_contract():
    p = compiled(operators.gated("bf16", save=True))
    good = [desc("bf16", 4, 8), desc("bf16", 8, 16), desc("bf16", 8, 16)] + [desc("bf16", 4, 16)] * 3
    assert p.check(good) == 0
    for i, bad in ((1, desc("bf16", 9, 16)), (2, desc("bf16", 8, 17)), (3, desc("bf16", 5, 16)), (4, desc("f16", 4, 16)),
                   (0, desc("bf16", 4, 8, 1))):
        t = list(good)
        t[i] = bad
        assert p.check(t) == _lib.TCA_ERR_SHAPE
    assert p.check(good[:-1]) == _lib.TCA_ERR_INVALID
    assert p.check([TensorDesc(8, (4, 8), 2)] + good[1:]) == _lib.TCA_ERR_INVALID


def test_the_driver_emits_operators(tmp_path):
    """tcacomp operator: the files of the program, word for word, with a Makefile
    of its own hipcc line; the list; refusals."""
    cli = lambda *a: subprocess.run([build.CLI] + list(a), capture_output=True, text=True)  # noqa: E731
    r = cli("operator")
    assert r.returncode == 0 and r.stdout == _lib.lib().tca_op_list().decode()
    op = operators.linear("bf16", act="gelu", bias=True)
    r = cli("operator", "-o", str(tmp_path), "linear", "elem=bf16", "act=gelu", "bias")
    assert r.returncode == 0 and r.stdout == "tcacomp: compiled %s -> %s\n" % (op.name, tmp_path), r.stderr
    e = op.emit()
    assert (tmp_path / (op.name + ".hip")).read_text() == e.source and (tmp_path / (op.name + ".plan")).read_text() == e.plan
    r = subprocess.run(["make", "-n", "-C", str(tmp_path)], capture_output=True, text=True)
    assert r.returncode == 0 and all(f in r.stdout for f in e.hipcc) and op.name + ".hip" in r.stdout
    for args, code, word in ((("nothing", "elem=bf16"), 1, "nothing"), (("linear", "elem=f32"), 1, "elem=f32"),
                             (("-target", "sm_86", "linear", "elem=bf16"), 1, "sm_86"), (("-x", "linear"), 2, "-x"), (("-o",), 2, "-o")):
        r = cli("operator", *args)
        assert r.returncode == code and word in r.stderr and not r.stdout, (args, r.stderr)
