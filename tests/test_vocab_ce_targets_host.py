"""The bounds of test_gpu_vocab_ce_targets tell a remainder that is carried from one that is dropped or subtracted (planted
in an emulation of the sums, on the CPU)."""
import pytest
import torch

from test_gpu_vocab_ce_targets import U, holds


@pytest.mark.parametrize("dt", list(U))
@pytest.mark.parametrize("M", [1, 30, 200])
def test_bounds_see_the_remainder(M, dt):
    g = torch.Generator().manual_seed(M)
    G = -(torch.rand(M, generator=g, dtype=torch.float64) * 0.5 + 0.4)
    row = (torch.randn(64, generator=g) * 0.3).to(dt).double()
    known = 4e-5 * (1 + G)
    Gf = G.float()                                            # the kernels' fp32 entry, rounded, and what that takes off
    G16 = Gf.to(dt).float()
    rest = Gf - G16

    def result(carried):
        return ((G16.double() + carried.double())[:, None] * row).float().to(dt)
    want = G[:, None] * row
    holds(result(rest), want, known[:, None] * row.abs(), dt, 0.0)
    holds(result(rest.to(dt)), want, known[:, None] * row.abs(), dt, U[dt] ** 2)
    for wrong in (0 * rest, -rest, rest.roll(1) if M > 1 else -rest):
        with pytest.raises(AssertionError):
            holds(result(wrong), want, known[:, None] * row.abs(), dt, U[dt] ** 2)
