"""The workspaces of operator programs: what a launch needs is what its kernels
write at its sizes, not the most that they could (the plan's scratch records);
the allocation-free launch and a captured one ask for no more."""
import ctypes
import itertools
import re
import threading

import pytest
import torch

import operators_ref as ref
from tcacomp_amd import _lib, compiler, operators
from test_gpu_operators import EPS, close, empty, gen_of, rand
from test_operators import compiled, desc, selected

PLAN = """tca-plan 1
program p
dim M 0
dim N 0
dim most 100
tensor x f32 in 2 M N
tensor y f32 out 2 M N
tensor a f32 local 1 most
tensor b f32 local 1 most
kernel k0 256 0 1 M*N/256
arg ptr x
arg ptr a
arg ptr b
%s
kernel k1 256 0 1 M*N/256
arg ptr b
arg ptr y
end
"""


def parse(text):
    h = ctypes.c_void_p()
    return _lib.lib().tca_program_parse(text.encode(), ctypes.byref(h)), h


def pointers(h, tensors, n_tensors, kernel):
    """The pointer arguments of a kernel: a local's is its offset in the workspace."""
    buf, size = (ctypes.c_uint8 * 512)(), ctypes.c_size_t()
    rc = _lib.lib().tca_program_kernel_args(h, compiler._descriptors(tensors), n_tensors, None, 0, None, 0, kernel, buf, 512, ctypes.byref(size))
    assert rc == 0, _lib.last_error()
    return lambda i: int.from_bytes(bytes(buf[8 * i:8 * i + 8]), "little")


@pytest.mark.parametrize("record,ok", [("scratch a 1 M/16:4", True), ("scratch a 2 M/16 N/1\nscratch b 1 N/1", True), ("scratch a", False),
                                       ("scratch a 0", False), ("scratch x 1 M/1", False), ("scratch c 1 M/1", False), ("scratch a 2 M/1", False),
                                       ("scratch a 1 M", False), ("scratch a 1 M/pack", False), ("scratch a 1 Q/1", False)])
def test_scratch_record(record, ok):
    rc, h = parse(PLAN % record)
    assert (rc == 0) == ok
    if ok:
        assert record in _lib.lib().tca_program_plan_text(h).decode()
    assert parse((PLAN % "").replace("kernel k0", record + "\nkernel k0"))[0] != 0  # before any kernel


@pytest.mark.parametrize("record,elems", [("", 100), ("scratch a 2 M/16:4 N/1", 36), ("scratch a 1 M/1\nscratch a 1 N/1", 70),
                                          ("split M 32 64 0 1 N/9\nscratch a 1 N/1", 27), ("split M 128 64 0 1 N/9\nscratch a 1 N/1", 0)])
def test_scratch_sizes(record, elems):
    """Local b lies behind what a needs (256-byte steps): M = 70, N = 9; split in three, then not."""
    rc, h = parse(PLAN % record)
    assert rc == 0, _lib.last_error()
    t = [desc("f32", 70, 9), desc("f32", 70, 9)]
    at = pointers(h, t, 2, 0)
    assert at(1) == 0 and at(2) == (4 * elems + 255) // 256 * 256


def test_scratch_that_overflows():
    rc, h = parse(PLAN % "scratch a 3 M*N/1 M*N/1 M*N/1")
    assert rc == 0
    buf, size = (ctypes.c_uint8 * 512)(), ctypes.c_size_t()
    arr = compiler._descriptors([desc("f32", 1 << 16, 60000)] * 2)
    assert _lib.lib().tca_program_kernel_args(h, arr, 2, None, 0, None, 0, 0, buf, 512, ctypes.byref(size)) == _lib.TCA_ERR_INVALID
    assert "address space" in _lib.last_error()


def needs(op, tensors, dims):
    """{local: elements} by the plan's scratch records and split records of the selected kernels."""
    p = compiled(op)
    grids, out, last, split = selected(p, tensors), {}, None, None
    up = lambda a, b: -(-a // b)  # noqa: E731

    def value(term):
        f, d = term.split("/")
        d, _, cap = d.partition(":")
        n = 1
        for x in f.split("*"):
            n *= dims[x] if x in dims else int(x)
        return min(up(n, int(d)), int(cap) if cap else 1 << 60)

    for line in op.emit().plan.splitlines():
        w = line.split()
        if not w:
            continue
        if w[0] == "kernel":
            last, split = w[1], None
        elif w[0] == "split":
            blocks = 1
            for t in w[6:]:
                blocks *= value(t)
            split = max(1, min(up(dims[w[1]], int(w[2])), int(w[3]) // blocks)) if blocks and dims[w[1]] else 1
        elif w[0] == "scratch" and last in grids:
            n = 1 if split is None else split if split > 1 else 0
            for t in w[3:]:
                n *= value(t)
            out[w[1]] = max(out.get(w[1], 0), n)
    return out, grids


def test_workspaces_hold_what_the_kernels_write():
    """Partial rows and partial sums, by the kernels' grids: every workgroup of a
    norm's rows and every chunk of columns writes one row of each gradient;
    every part of k a plane."""
    up = lambda a, b: -(-a // b)  # noqa: E731
    op = operators.layer_norm_backward("bf16")
    for R, C in itertools.product((1, 7, 64, 500, 5000), (64, 300, 4000, 8192, 20000)):
        t = [desc("bf16", R, C), desc("bf16", R, C), desc("bf16", C), desc("f32", R), desc("f32", R), desc("bf16", R, C), desc("bf16", C),
             desc("bf16", C)]
        got, grids = needs(op, t, dict(R=R, C=C))
        (part, elems), = got.items()
        rows = [g for s, g in grids.items() if re.search(r"_\d+x\d+$", s)]
        rows = rows[0] if rows else grids["tca_" + op.name + "_columns"] // up(C, 512)
        assert elems == rows * 2 * C, (R, C)
    for f, halves in ((operators.linear, 1), (operators.gated, 2)):
        op = f("bf16")
        for M, K, N in itertools.product((1, 16, 64, 65, 300, 1024), (64, 257, 1000, 4096), (64, 333, 1000, 20000)):
            y = [desc("bf16", M, N)]
            got, grids = needs(op, [desc("bf16", M, K)] + [desc("bf16", K, N)] * halves + y, dict(M=M, K=K, N=N))
            joined = any(s.endswith("join") for s in grids)
            assert bool(got.get("part")) == joined, (M, K, N)
            if joined:
                s, g = next((s, g) for s, g in grids.items() if not s.endswith("join"))
                rows, cols = (M, 64) if "_few" in s else (64, 128 // halves) if s.endswith("_o") else (128, 128 // halves)
                assert got["part"] == g // (up(M, rows) * up(N, cols)) * M * N * halves <= 256 * 128 * 128


def gated_backward_tensors(M, K, N, make):
    return [make(M, N), make(M, K), make(K, N), make(K, N), make(M, N), make(M, N), make(M, N), make(M, N), make(M, K), make(K, N), make(K, N),
            make(N), make(N)]


def test_few_tokens_need_few_partial_rows():
    """16 tokens have one partial row of a bias' gradient, not 256: `part` lies right behind it."""
    op = operators.gated_backward("f16", act="gelu", bias=True)
    p = compiled(op)
    M, K, N = 16, 1000, 10000
    t = gated_backward_tensors(M, K, N, lambda *s: desc("f16", *s))
    kernel = next(i for i, s in enumerate(p.kernel_symbols()) if s.endswith("_dx_k"))
    at = pointers(p.parsed(), t, len(t), kernel)
    assert at(7) == (4 * 2 * N + 255) // 256 * 256  # dg du wg wu dx, M K N (padded to 16 bytes), part


@pytest.mark.gpu
def test_noalloc_launch_of_few_tokens(gpu):
    """Wide layers and long rows without an allocation: refused while a workspace
    was sized for 4096 tokens."""
    M, K, N = 16, 1000, 10000
    g = gen_of("na")
    p = compiler.compile_program(operators.gated_backward("f16", act="gelu", bias=True))
    ins = [rand(g, s, "f16") for s in ((M, N), (M, K), (K, N), (K, N), (M, N), (M, N))]
    runs = []
    for noalloc in (True, False):
        outs = [empty(s, "f16") for s in ((M, N), (M, N), (M, K), (K, N), (K, N), (N,), (N,))]
        p.launch(ins + outs, noalloc=noalloc)
        runs.append(outs)
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    R, C = 3, 140000
    p = compiler.compile_program(operators.layer_norm_backward("bf16", residual=True))
    x, dy, dres, gamma = (rand(g, s, "bf16") for s in ((R, C), (R, C), (R, C), (C,)))
    mean, rstd = x.float().mean(1), (x.float().var(1, unbiased=False) + EPS).rsqrt()
    runs = []
    for noalloc in (True, False):
        outs = [empty(s, "bf16") for s in ((R, C), (C,), (C,))]
        p.launch([dy, x, gamma, mean, rstd, dres] + outs, noalloc=noalloc)
        runs.append(outs)
    assert all(torch.equal(a, b) for a, b in zip(*runs))
    args = [v.double() for v in (dy, x, gamma, mean, rstd, dres)]
    for got, w, b in zip(runs[0], ref.layer_norm_backward(*args), ref.layer_norm_backward_bounds(*args, torch.bfloat16, torch.bfloat16)):
        close(got, w, b, "long rows")


@pytest.mark.gpu
@pytest.mark.parametrize("mode", ["global", "thread_local", "relaxed"])
def test_a_refused_launch_leaves_the_capture(gpu, mode):
    """A launch that would allocate while its stream is captured, also after one
    on another stream: refused in every mode, and the capture goes on, with the
    allocation-free launch in its place."""
    g = gen_of("refused")
    p = compiler.compile_program(operators.linear("bf16"))
    M, K, N = 5, 1000, 90
    x, w, y, want = rand(g, (M, K), "bf16"), rand(g, (K, N), "bf16"), empty((M, N), "bf16"), empty((M, N), "bf16")
    p.launch([x, w, want])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream(), capture_error_mode=mode):
        with pytest.raises(_lib.TcaError, match="being captured"):
            p.launch([x, w, y])
        p.launch([x, w, y], noalloc=True)
    for _ in range(3):
        y.fill_(-1.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)


@pytest.mark.gpu
def test_a_launch_that_needs_no_workspace_is_captured_at_once(gpu):
    """K in one part writes no partial sums: a first launch may be captured, and
    replayed between eager launches."""
    g = gen_of("first")
    for M, K, N in ((5, 200, 90), (130, 264, 200)):
        p = compiler.compile_program(operators.linear("bf16"))
        x, w, y = rand(g, (M, K), "bf16"), rand(g, (K, N), "bf16"), empty((M, N), "bf16")
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            p.launch([x, w, y])
        for _ in range(3):
            x.copy_(rand(g, (M, K), "bf16"))
            want = empty((M, N), "bf16")
            p.launch([x, w, want])
            torch.cuda.synchronize()
            y.fill_(-1.0)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, want)


@pytest.mark.gpu
@pytest.mark.parametrize("shared", [False, True], ids=["two_streams", "one_stream"])
def test_two_threads_launch_one_program(gpu, shared):
    """Each thread its own sizes, of which one outgrows the other's workspace; on
    streams of their own, or on one, where the launches take turns."""
    g = gen_of("threads")
    p = compiler.compile_program(operators.layer_norm_backward("bf16", residual=True))

    def make(R, C):
        x, dy, dres = (rand(g, (R, C), "bf16") for _ in range(3))
        ins = [dy, x, rand(g, (C,), "bf16"), x.float().mean(1), x.float().std(1).reciprocal(), dres]
        want = [empty((R, C), "bf16"), empty((C,), "bf16"), empty((C,), "bf16")]
        compiler.compile_program(operators.layer_norm_backward("bf16", residual=True)).launch(ins + want)
        return ins, want

    work = [make(500, 300), make(700, 3000)]
    runs = [[[torch.full_like(w, -1.0) for w in want] for _ in range(30)] for _, want in work]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    if shared:
        streams[1] = streams[0]
    torch.cuda.synchronize()
    failed = []

    def run(i):
        try:
            for outs in runs[i]:
                p.launch(work[i][0] + outs, stream=streams[i].cuda_stream)
        except Exception as e:  # noqa: BLE001 (reported below)
            failed.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failed, failed
    for (_, want), outs in zip(work, runs):
        assert all(torch.equal(a, w) for o in outs for a, w in zip(o, want))
