"""Batches of matrices in any layout: what is written arrives in the caller's tensor."""
import pytest
import torch

from test_gpu_muon import gradient_like

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("order", [(0, 1, 2), (1, 0, 2), (2, 0, 1)])
def test_results_in_a_permuted_batch(order):
    """Batch dimensions whose strides no single one replaces."""
    from capdec import ops
    shape = (2, 3, 4)
    G = gradient_like((24, 40, 56)).view(*shape, 40, 56)
    want = ops.orthogonalize(G)
    G, want = G.permute(*order, 3, 4), want.permute(*order, 3, 4)
    out = torch.full_like(G, float("nan"))                   # (keeps the strides)
    assert out.stride() == G.stride() and ops.orthogonalize(G, out=out) is out and torch.equal(out, want)
    assert torch.equal(ops.orthogonalize(G), want)
    H = G.clone()
    assert H.stride() == G.stride() and ops.orthogonalize(H, out=H) is H and torch.equal(H, want)


def test_updates_of_a_permuted_batch():
    from capdec import ops
    p, g, m = (gradient_like((6, 48, 32), k).view(2, 3, 48, 32) for k in range(3))
    a = [t.transpose(0, 1).clone() for t in (p, g, m)]
    b = [[t[i, j].clone() for i in range(3) for j in range(2)] for t in a]
    assert not a[0].is_contiguous()
    ops.muon_step(*a, lr=0.1)
    ops.muon_step(*b, lr=0.1)
    for t, want in zip((a[0], a[2]), (b[0], b[2])):
        assert all(torch.equal(t[i, j], want[2 * i + j]) for i in range(3) for j in range(2))


def test_empty_batches():
    from capdec import ops
    for shape in ((0, 4, 5), (2, 0, 4, 5)):
        assert ops.orthogonalize(torch.empty(shape, device="cuda")).shape == shape
    assert ops.orthogonalize([]) == []
    ops.muon_step([], [], [], lr=0.1)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("scale", [1e-33, 1e-36, 1e36])
def test_norms_at_the_ends_of_the_range(scale, dt):
    """Without eps: matrices whose norm has no reciprocal in fp32, and large ones; on their own (rounded) values."""
    from capdec import ops
    from test_gpu_muon import definition, near
    G = (gradient_like((60, 90)) * scale).to(dt)
    near(ops.orthogonalize(G, eps=0.0), definition(G, eps=0.0), dt)
    m, p = torch.zeros(60, 90, device="cuda"), torch.zeros(60, 90, device="cuda")
    ops.muon_step([p], [G.float()], [m], lr=1.0, momentum=0.0, nesterov=False, eps=0.0, update_scale=1.0)
    near(-p, definition(G, eps=0.0), torch.float32)
