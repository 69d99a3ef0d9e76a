"""What the GPU tests of long products (test_gpu_products.py) would notice: the
bound of a random walk against models of the sums on the CPU, and the kernels
that their sizes take."""
import re

import pytest
import torch

import operators_ref as ref
from products_cases import FEW, ODD_PLANES, REDUCTION_ODD, REDUCTION_WHOLE, WHOLE_PLANES
from tcacomp_amd import operators
from test_operators import compiled, desc, forms, launched


def model(a, b, parts, keep):
    """a b in f32, 32 values of k at a time, in `parts` runs of k, whose sums
    are rounded to `keep` and added in it."""
    total = None
    for run in torch.arange(a.shape[1]).chunk(parts):
        s = torch.zeros(a.shape[0], b.shape[1])
        for k in run.split(32):
            s = s + a[:, k].float() @ b[k].float()
        s = s.to(keep)
        total = s if total is None else (total + s).to(keep)
    return total


@pytest.mark.parametrize("elem", ["bf16", "f16"])
@pytest.mark.parametrize("M,K,N,parts", [(130, 1003, 150, 2), (64, 4099, 131, 17), (72, 3608, 400, 8), (200, 1096, 264, 3),
                                         (257, 515, 300, 2)])
def test_the_bound_tells_16_bit_partial_sums(M, K, N, parts, elem):
    torch.manual_seed(0)
    t = ref.DTYPES[elem]
    a, b = torch.randn(M, K).to(t), (torch.randn(K, N) * K ** -0.5).to(t)
    want = a.double() @ b.double()
    bound = ref.walk_bound(a.double(), b.double()) + ref.half_step(t, want)
    off = lambda keep: float(((model(a, b, parts, keep).to(t).double() - want).abs() / bound).max())  # noqa: E731
    assert off(torch.float32) <= 1.0 < off(t), (off(torch.float32), off(t))


def rows_of(f, elem, attrs, M, K, N):
    """{symbol: (k of its product, segments of it, P)} of a launch."""
    op = f(elem, **attrs)
    p, plan = compiled(op), forms(op)
    x, w, y, b, dims = desc(elem, M, K), desc(elem, K, N), desc(elem, M, N), desc(elem, N), dict(M=M, K=K, N=N)
    n = 2 if "gated" in op.op else 1
    has, acts = ([b] * n if attrs.get("bias") else []), n == 2 or attrs.get("act", "none") != "none"
    if "backward" in op.op:
        pre = [y] * n if acts else []
        t = [y, x] + [w] * n + pre + pre + [x] + [w] * n + has
    else:
        t = [x] + [w] * n + has + [y] * (1 + bool(attrs.get("residual")) + (n if attrs.get("save") else 0))
    out, up = {}, lambda a, b: -(-a // b)  # noqa: E731
    for suffix, grid in launched(p, plan, t, dims).items():
        if suffix.endswith("join") or suffix in ("_slope", "_bias"):
            continue
        dx, dw = suffix.startswith("_dx"), suffix.startswith("_dw")
        rows, cols, k = (M, K, N) if dx else (K, N, M) if dw else (M, N, K)
        half = 2 if n == 2 and not dx else 1
        tail = suffix[3:] if dx or dw else suffix
        blocks = up(cols, 64) if tail.startswith("_few") else up(rows, 64 if tail == "_o" else 128) * up(cols, 128 // half)
        P = grid // blocks if tail in ("_k", "_o") or tail.startswith("_few") else 1
        out["tca_" + p.name + suffix] = (k, 2 if dx and n == 2 else 1, P)
    return out


def launches():
    for M, K, N in FEW:
        yield operators.linear, "bf16", dict(bias=True, residual=True), M, K, N
        yield operators.gated, "f16", {}, M, K, N
    for planes, K in ((ODD_PLANES, REDUCTION_ODD), (WHOLE_PLANES, REDUCTION_WHOLE)):
        for M, N in planes:
            yield operators.linear, "bf16", dict(bias=True, residual=True), M, K, N
            yield operators.gated, "f16", {}, M, K, N
            yield operators.linear_backward, "bf16", dict(act="gelu", bias=True), K, M, N
            yield operators.linear_backward, "bf16", dict(act="gelu", bias=True), M, N, K
            yield operators.gated_backward, "f16", {}, K, M, N
            yield operators.gated_backward, "f16", {}, M, N, K


def test_every_kernel_reaches_its_steady_state():
    """Every product kernel and form of the four programs: a ring, more turns
    than twice its slots; rows of any shape, more than four slices; few rows,
    more steps a wave than its registers hold; where k may be split, P > 1 too."""
    loops, parts, split = {}, {}, set()
    for f, elem, attrs, M, K, N in launches():
        op = f(elem, **attrs)
        bodies = dict(re.findall(r"(tca_\w+)\([^{]*\{(.*?)\n\}", op.emit().source, re.S))
        for s, body in bodies.items():
            if "join_" in body or "product_" not in body:
                continue
            loops.setdefault(s, False)
            if "product_few" in body or "split_store" in body:
                split.add(s)
        for s, (k, segs, P) in rows_of(f, elem, attrs, M, K, N).items():
            ring = re.search(r"product_ring<[^>]*, (\d+), (\d+)>", bodies[s])
            few = re.search(r"product_few<\w+, (\w+), (\d+)>", bodies[s])
            if ring:
                ok = s in split or k // 64 * segs > 2 * int(ring.group(1))
            elif few:
                held = 2 if (2 if few.group(1) == "true" else 1) * int(few.group(2)) > 4 else 4
                ok = -(-k // 32) // P // 8 > held
            else:
                ok = k // 64 * segs // P > 4
            loops[s] = loops[s] or ok
            parts.setdefault(s, set()).add(P)
    assert all(loops.values()), sorted(s for s, ok in loops.items() if not ok)
    assert split and all(max(parts[s]) > 1 for s in split), {s: parts.get(s) for s in split}
