"""What a test of the operator programs' products would notice: the
bound of a random walk against models of the sums on the CPU."""
import pytest
import torch

import operators_ref as ref


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
