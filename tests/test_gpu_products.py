"""The products of the operator programs past their first step, slice or turn
(products_cases.py), against 64 bits, with the bound of a random walk in place
of the framework's bar for contractions: a partial sum kept in 16 bits fails it
(test_product_bounds.py)."""
import pytest

import operators_ref as ref
import test_gpu_operators as base
from products_cases import FEW

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
