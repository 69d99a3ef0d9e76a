"""The products of the operator programs past their first step, slice or turn
(products_cases.py), against 64 bits, with the bound of a random walk in place
of the framework's bar for contractions: a partial sum kept in 16 bits fails it
(test_product_bounds.py)."""
import pytest
import torch

import operators_ref as ref
import test_gpu_operators as base
from products_cases import FEW, ODD_PLANES, REDUCTION_ODD, REDUCTION_WHOLE, WHOLE_PLANES
from tcacomp_amd import operators

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def walk(monkeypatch):
    monkeypatch.setattr(ref, "product_bound", ref.walk_bound)


@pytest.mark.parametrize("M,K,N", FEW)
def test_few_rows(gpu, M, K, N):
    print("few rows", M, K, N, flush=True)
    base.check_linear("bf16", M, K, N, bias=True, residual=True)
    base.check_linear("f16", M, K, N, act="gelu", bias=True, residual=True)
    base.check_linear("bf16", M, K, N, act="gelu", bias=True, save=True)
    base.check_gated("bf16", M, K, N, save=True)
    base.check_gated("f16", M, K, N)
    base.check_gated("f16", M, K, N, act="gelu", bias=True, save=True)


def test_the_repeated_product_is_right(gpu):
    base.check_linear("bf16", 7, 3000, 640, bias=True, residual=True)  # what base.test_runs_repeat_bit_for_bit compares with itself


def check_plane(M, N, K):
    """Results of M x N with a reduction of K: forward, as dw and as dx."""
    base.check_linear("bf16", M, K, N, act="gelu", bias=True, residual=True)
    base.check_linear("f16", M, K, N, act="gelu", bias=True, save=True)
    base.check_gated("f16", M, K, N, save=True)
    base.check_gated("bf16", M, K, N)
    base.check_linear_backward("bf16", K, M, N, act="gelu", bias=True)
    base.check_gated_backward("f16", K, M, N)
    base.check_linear_backward("f16", M, N, K, bias=True)
    base.check_gated_backward("bf16", M, N, K)


@pytest.mark.parametrize("M,N", ODD_PLANES)
def test_odd_rows(gpu, M, N):
    print("odd rows", M, N, flush=True)
    check_plane(M, N, REDUCTION_ODD)


@pytest.mark.parametrize("M,N", WHOLE_PLANES)
def test_whole_chunks(gpu, M, N):
    print("whole chunks", M, N, flush=True)
    check_plane(M, N, REDUCTION_WHOLE)


def test_gradients_repeat_bit_for_bit(gpu):
    """The gradients, split over k: right, and five runs alike."""
    base.check_gated_backward("f16", 500, 769, 2049)
    g = base.gen_of("rep2")
    for f, elem, M, K, N in ((operators.linear_backward, "bf16", 600, 264, 520), (operators.linear_backward, "f16", 601, 265, 521)):
        dy, x, w, z = (base.rand(g, s, elem) for s in ((M, N), (M, K), (K, N), (M, N)))
        p = base.program(f, elem, act="gelu", bias=True)
        runs = []
        for _ in range(5):
            runs.append([base.empty(s, elem) for s in ((M, N), (M, K), (K, N), (N,))])
            p.launch([dy, x, w, z] + runs[-1])
        assert all(torch.equal(a, b) for r in runs for a, b in zip(runs[0], r))


@pytest.mark.parametrize("M,K,N", [(70, 0, 91), (3, 0, 21), (0, 41, 63), (30, 0, 63), (30, 41, 0), (1200, 0, 1000), (0, 1200, 1000),
                                   (1101, 0, 1001), (0, 1101, 1001), (1200, 1000, 0), (1101, 1001, 0)])
def test_empty_extents(gpu, M, K, N):
    """No reduction leaves the bias and the residual, no tokens zero gradients of
    the weights, in every kind of kernel."""
    print("empty", M, K, N, flush=True)
    base.check_linear("bf16", M, K, N, bias=True, residual=True)
    base.check_gated("f16", M, K, N, act="gelu", bias=True, save=True)
    base.check_linear_backward("bf16", M, K, N, act="gelu", bias=True)
    base.check_gated_backward("f16", M, K, N)


@pytest.mark.parametrize("M,K,N", [(20000, 24, 40), (9001, 17, 1027)])
def test_bias_gradients_of_many_rows(gpu, M, K, N):
    """More than 16 rows a partial row of the bias' gradient: a wave of it walks rows, two at a time."""
    print("many rows", M, K, N, flush=True)
    base.check_linear_backward("bf16", M, K, N, act="gelu", bias=True)
    base.check_linear_backward("f16", M, K, N, bias=True)
    base.check_gated_backward("f16", M, K, N, act="gelu", bias=True)
