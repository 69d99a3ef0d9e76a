"""A dispatch counts its lanes in 32 bits: launches of more are refused, where they ran
the lanes left modulo 2^32 without a word."""
import pytest

from tcacomp_amd import _lib


@pytest.mark.parametrize("block", [64, 256, 512, 1024])
def test_lanes_fit_32_bits(block):
    L = _lib.lib()
    most = (1 << 32) // block
    assert L.tca_rt_validate_launch(most - 1, block, 0) == 0
    for grid in (most, most + 1, (1 << 31) - 1):
        assert L.tca_rt_validate_launch(grid, block, 0) == _lib.TCA_ERR_LAUNCH
        assert "lanes" in _lib.last_error()


@pytest.mark.gpu
def test_rotary_of_too_many_tokens(gpu):
    """2^26 tokens of 16 features are 2^24 workgroups of 256 lanes; one group less of four runs."""
    import torch

    from tcacomp_amd import attention
    from test_gpu_operators import program
    x = torch.arange(1 << 15, device="cuda", dtype=torch.float32).to(torch.bfloat16).repeat(1 << 15).view(1 << 26, 1, 16)
    pos, freq = torch.zeros(1 << 26, device="cuda", dtype=torch.int32), torch.ones(4, device="cuda")
    y = torch.zeros_like(x)
    p = program(attention.rotary, "bf16")
    with pytest.raises(_lib.TcaError, match="lanes"):
        p.launch([x, pos, freq, y], scalars=(1.0,))
    n = (1 << 26) - 4
    p.launch([x[:n], pos[:n], freq, y[:n]], scalars=(1.0,))
    assert torch.equal(y[:n], x[:n]) and not y[n:].any()
