"""The workspace of attention over pages: what a launch allocates is what the largest
batch at its width needs, and which batches the allocation-free launch has room for."""
import pytest

from tcacomp_amd import attention
from test_attention import args, attend_tensors
from test_operators import compiled

SCRATCH = 32 << 20  # of the allocation-free launch


def up(n):
    return -(-n // 256) * 256


def locals_of(plan, D):
    """(name, declared bytes) of the locals that the kernels for heads of D take, in the plan's order."""
    dims, declared, kernels = {}, [], []
    for line in plan.splitlines():
        w = line.split()
        if w[0] == "dim":
            dims[w[1]] = int(w[2])
        elif w[0] == "tensor" and w[3] == "local":
            n = 4
            for d in w[5:]:
                n *= D if d == "D" else dims[d]
            declared.append((w[1], n))
        elif w[0] == "kernel":
            kernels.append([set(), None])
        elif w[:2] == ["arg", "ptr"]:
            kernels[-1][0].add(w[2])
        elif w[:2] == ["when", "D"]:
            kernels[-1][1] = int(w[2]) <= D <= int(w[3])
    used = set().union(*(names for names, runs in kernels if runs))
    return [(n, b) for n, b in declared if n in used]


def need(p, names, **shape):
    """Bytes that a launch uses: where its locals lie in a workspace at address 0, and the last one's size."""
    D = shape["D"]
    kernel = 2 * (-(-D // 64) - 1)
    a = args(p, attend_tensors(**shape), kernel)
    at = [int.from_bytes(a[8 * i:8 * i + 8], "little") for i in range(7, 7 + len(names))]
    assert at == sorted(at) and at[0] == 0
    return at[-1] + up(256 * 8 * 4)


@pytest.mark.parametrize("D", [8, 64, 72, 128, 136, 192, 200, 256])
def test_no_more_is_allocated_than_can_be_used(D):
    op = attention.paged_attention("bf16")
    found = locals_of(op.emit().plan, D)
    assert len(found) == 6
    allocated = sum(up(b) for _, b in found)
    rows = 256 if D <= 128 else 128  # of a tile
    assert need(compiled(op), found, T=4000, G=4, D=D) == allocated == 512 * (32 + rows) * (4 * D + 8) + 2 * 256 * 8 * 4


def test_the_largest_and_what_fits_the_allocation_free_launch():
    """The figures of include/tca_op.h."""
    op = attention.paged_attention("f16")
    p, plan = compiled(op), op.emit().plan
    most = {D: sum(up(b) for _, b in locals_of(plan, D)) for D in range(8, 257, 8)}
    assert max(most.values()) == most[256] and round(most[256] / 1e6) == 85 and round(most[128] / 1e6) == 77
    names = locals_of(plan, 128)
    assert need(p, names, T=93, G=1, D=128, elem="f16") <= SCRATCH < need(p, names, T=94, G=1, D=128, elem="f16")
