"""Orthogonalised updates of 16-bit matrices: what the iteration gives in float32, rounded once, for every spectrum, number
of steps, size and batch; float32 against the definition on the same inputs."""
import pytest
import torch

from test_gpu_muon import COEFFS, definition, gradient_like, near

pytestmark = pytest.mark.gpu

HALF = [torch.bfloat16, torch.float16]


def spectrum(kind, m, n):
    g = torch.Generator("cuda").manual_seed(m + n)
    r = min(m, n)
    u, _ = torch.linalg.qr(torch.randn(m, r, device="cuda", generator=g))
    v, _ = torch.linalg.qr(torch.randn(n, r, device="cuda", generator=g))
    s = {"flat": torch.ones(r), "few": torch.cat([torch.ones(16), torch.full((r - 16,), 1e-3)]), "one": torch.cat([torch.ones(1), torch.full((r - 1,), 1e-2)]),
         "log": torch.logspace(0, -3, r)}[kind].cuda()
    return (u * s) @ v.T


@pytest.mark.parametrize("dt", HALF)
@pytest.mark.parametrize("kind", ["flat", "few", "one", "log"])
@pytest.mark.parametrize("steps,coeffs", [(1, COEFFS), (2, COEFFS), (3, COEFFS), (5, COEFFS), (7, COEFFS), (2, (4.0, -6.0, 3.0)),
                                          (5, (2.0, 0.0, -1.0)), (8, (1.5, -0.5, 0.0))])
def test_rounded_once_for_every_spectrum(kind, steps, coeffs, dt):
    from capdec import ops
    for shape in ((256, 384), (300, 128)):
        G = spectrum(kind, *shape).to(dt)
        want = ops.orthogonalize(G.float(), steps=steps, coeffs=coeffs)
        assert torch.equal(ops.orthogonalize(G, steps=steps, coeffs=coeffs), want.to(dt))
        near(want, definition(G, steps, coeffs), torch.float32)


@pytest.mark.parametrize("dt", HALF)
@pytest.mark.parametrize("shape", [(1, 1), (7, 5), (77, 130), (3, 1333, 517), (1, 2048, 1024), (1, 1024, 3000), (1, 2500, 1100), (1, 800, 5000),
                                   (1, 2048, 6000), (6, 640, 640), (20, 300, 700), (40, 64, 96)])
def test_rounded_once_at_every_size(shape, dt):
    """Every tile, the triangles with their parts, tall and wide, one matrix and batches."""
    from capdec import ops
    G = gradient_like(shape).to(dt)
    want = ops.orthogonalize(G.float())
    assert torch.equal(ops.orthogonalize(G), want.to(dt))
    near(want, definition(G), torch.float32)
