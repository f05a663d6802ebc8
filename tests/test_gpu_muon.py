"""Orthogonalised updates against the iteration in 64 bits.

Tolerance.  A step maps each singular value s to s (a + b s^2 + c s^4); over [0, 1.3] the slope is at most |a| = 3.4445 for
the default coefficients, so an error made with r steps to go grows by at most a^r.  A step's own error is at most
12 * 2^-22 of the iterate: the values are kept to 2^-22 (X twice, A, B), three products leave 2^-22 each out and their fp32
sums round.  Over five steps, in the spectral norm and so in the Frobenius norm of a result of full rank to within the
same factor:  (a^5 - 1) / (a - 1) * 12 * 2^-22 = 5.7e-4 at most; half a step of the result's type comes on top.  Errors of
single entries are random and far smaller, so the Frobenius norm is held to a twentieth of that, 3e-5.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
COEFFS = (3.4445, -4.7750, 2.0315)


def gradient_like(shape, seed=0, rank=None):
    g = torch.Generator("cuda").manual_seed(seed + sum(shape))
    rows, cols = shape[-2:]
    r = rank or max(1, min(rows, cols) // 8)
    u = torch.randn(*shape[:-1], r, device="cuda", generator=g) / torch.arange(1, r + 1, device="cuda").sqrt()
    v = torch.randn(*shape[:-2], r, cols, device="cuda", generator=g)
    return (u @ v + 0.3 * torch.randn(shape, device="cuda", generator=g)) * 1e-3


def definition(G, steps=5, coeffs=COEFFS, eps=1e-7):
    a, b, c = coeffs
    X = G.double()
    X = X / (X.square().sum((-2, -1), keepdim=True).sqrt() + eps)
    for _ in range(steps):
        if X.shape[-2] <= X.shape[-1]:
            A = X @ X.mT
            X = a * X + (b * A + c * (A @ A)) @ X
        else:
            A = X.mT @ X
            X = a * X + X @ (b * A + c * (A @ A))
    return X


def near(got, want, dt, tol=3e-5):
    assert got.dtype == dt and got.shape == want.shape
    err = float((got.double() - want).norm() / want.norm())
    assert err <= tol + U[dt], f"relative error {err:.2e}"


SHAPES = [(1, 1), (1, 100), (100, 1), (7, 5), (31, 32), (32, 33), (64, 64), (130, 77), (77, 130), (128, 512), (513, 129),
          (512, 512), (1000, 333), (333, 2000)]


@pytest.mark.parametrize("dt", list(U))
@pytest.mark.parametrize("shape", SHAPES)
def test_orthogonalize(shape, dt):
    from capdec import ops
    G = gradient_like(shape).to(dt)
    near(ops.orthogonalize(G), definition(G), dt)


@pytest.mark.parametrize("shape", [(1, 2048, 1024), (1, 1024, 3000), (1, 900, 1000), (2, 2500, 1100), (1, 800, 5000), (1, 2048, 6000), (6, 640, 640), (20, 300, 700), (40, 64, 96)])
def test_batches_and_larger_tiles(shape):
    from capdec import ops
    for dt in (torch.float32, torch.bfloat16):
        G = gradient_like(shape).to(dt)
        near(ops.orthogonalize(G), definition(G), dt)


def test_batch_dimensions_lists_and_in_place():
    from capdec import ops
    G = gradient_like((2, 3, 40, 60))
    want = ops.orthogonalize(G)
    near(want, definition(G), torch.float32)
    mats = [G[0, 0], G[1, 2], gradient_like((70, 20)), G[0, 1]]
    got = ops.orthogonalize(mats)
    assert torch.equal(got[0], want[0, 0]) and torch.equal(got[1], want[1, 2]) and torch.equal(got[3], want[0, 1])
    near(got[2], definition(mats[2]), torch.float32)
    H = G.clone()
    assert ops.orthogonalize(H, out=H) is H and torch.equal(H, want)


def test_strided_matrices():
    from capdec import ops
    wide = torch.full((50, 90), float("nan"), device="cuda")
    wide[:, 3:73] = gradient_like((50, 70))
    out = torch.full((50, 80), 7.0, device="cuda")
    ops.orthogonalize([wide[:, 3:73]], out=[out[:, 1:71]])
    assert torch.equal(out[:, 1:71], ops.orthogonalize(wide[:, 3:73].contiguous()))
    assert bool((out[:, 0] == 7).all()) and bool((out[:, 71:] == 7).all())


def test_columns_of_one_wider_matrix():
    """Three projections side by side in one matrix, updated in place."""
    from capdec import ops
    w = gradient_like((64, 150)) * 1e3
    parts, want = [w[:, 50 * k:50 * k + 50] for k in range(3)], [w[:, 50 * k:50 * k + 50].contiguous() for k in range(3)]
    g, m = [gradient_like((64, 50), k) for k in range(3)], [torch.zeros(64, 50, device="cuda") for _ in range(6)]
    ops.muon_step(parts, g, m[:3], lr=0.1)
    ops.muon_step(want, g, m[3:], lr=0.1)
    assert all(torch.equal(a, b) for a, b in zip(parts, want))


def test_steps_coefficients_and_spectra():
    """Other iterations, and spectra from one direction to six orders of magnitude."""
    from capdec import ops
    G = gradient_like((200, 300))
    for steps in (1, 2, 7):
        # slope growth of the docstring for `steps` steps, relative to a result whose norm is at least that of X_0 = 1
        near(ops.orthogonalize(G, steps=steps), definition(G, steps), torch.float32, tol=3e-5 * max(1.0, 3.4445 ** (steps - 5)))
    for co in ((1.5, -0.5, 0.0), (1.875, -1.25, 0.375), (2.0, 0.0, -1.0)):
        near(ops.orthogonalize(G, steps=9, coeffs=co), definition(G, 9, co), torch.float32)
    near(ops.orthogonalize(gradient_like((128, 128), rank=1)), definition(gradient_like((128, 128), rank=1)), torch.float32)
    u, _ = torch.linalg.qr(torch.randn(96, 96, device="cuda"))
    G = (u * torch.logspace(0, -6, 96, device="cuda")) @ u.flip(1).T
    near(ops.orthogonalize(G), definition(G), torch.float32)


def test_scale_does_not_matter_and_zero_stays_zero():
    from capdec import ops
    G = gradient_like((60, 90))
    want = definition(G, eps=0.0)
    for s in (1e-25, 1e-10, 1e10, 1e30):
        near(ops.orthogonalize(G * s, eps=0.0), want, torch.float32)
    for eps in (1e-7, 0.0):
        assert int(ops.orthogonalize(torch.zeros(3, 40, 50, device="cuda"), eps=eps).count_nonzero()) == 0
    out = ops.orthogonalize(G, coeffs=(1e-9, 0.0, 0.0))            # an iterate that shrinks away
    assert bool(out.isfinite().all()) and float(out.norm()) < 1e-30
    bad = torch.stack([G, G, G])
    bad[1, 5, 5] = float("nan")
    out = ops.orthogonalize(bad)
    assert bool(out[1].isnan().any()) and torch.equal(out[0], ops.orthogonalize(G)) and torch.equal(out[2], out[0])


@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("shapes", [[(64, 64)], [(200, 100), (33, 65), (200, 100), (100, 200)], [(48, 80)] * 40])
def test_muon_step(shapes, nesterov):
    from capdec import ops
    g = torch.Generator("cuda").manual_seed(4)
    p = [torch.randn(s, device="cuda", generator=g) for s in shapes]
    gr = [gradient_like(s, 1) for s in shapes]
    m = [gradient_like(s, 2) * 5 for s in shapes]
    p0, m0 = [t.clone() for t in p], [t.clone() for t in m]
    ops.muon_step(p, gr, m, lr=0.03, momentum=0.9, nesterov=nesterov, weight_decay=0.1, grad_scale=0.5)
    for s, a, b, c, d, e in zip(shapes, p, gr, m, p0, m0):
        mom = 0.9 * e.double() + 0.5 * b.double()
        u = 0.5 * b.double() + 0.9 * mom if nesterov else mom
        # momentum: two roundings of fp32 and the fp32 value of 0.9 (2^-25)
        assert bool(((c.double() - mom).abs() <= 2.0 ** -23 * (mom.abs() + 0.9 * e.abs())).all())
        x = definition(u)
        want = d.double() * (1 - 0.03 * 0.1) - 0.03 * math.sqrt(max(1, s[0] / s[1])) * x
        step = 0.03 * math.sqrt(max(1, s[0] / s[1]))
        assert float((a.double() - want).norm()) <= 3e-5 * step * float(x.norm()) + 2.0 ** -22 * float(d.norm())


def test_learning_rate_on_the_device_and_graph_replays():
    """A captured step reads the learning rate at every replay; two captured steps share no memory."""
    from capdec import ops
    state = ops.TrainState("cuda", 0.01, 1)
    sets = []
    for n in range(2):
        p, g, m = gradient_like((96, 160), n) * 1e3, gradient_like((96, 160), 10 + n), torch.zeros(96, 160, device="cuda")
        ops.muon_step([p.clone()], [g], [m.clone()], state=state)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.muon_step([p], [g], [m], state=state)
        sets.append((graph, p, g, m, p.clone(), m.clone()))
    for r in range(3):
        state.set(lr=0.01 * (r + 1))
        for n, (graph, p, g, m, q, k) in enumerate(sets):
            g.copy_(gradient_like((96, 160), 50 + 2 * r + n))
        for graph, *_ in sets:
            graph.replay()
        for _, p, g, m, q, k in sets:
            ops.muon_step([q], [g], [k], lr=0.01 * (r + 1))
            assert torch.equal(p, q) and torch.equal(m, k)


def test_repeats_bit_for_bit_and_on_another_stream():
    from capdec import ops
    G = gradient_like((4, 300, 500))
    want = ops.orthogonalize(G)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = ops.orthogonalize(G)
    s.synchronize()
    assert torch.equal(got, want) and torch.equal(ops.orthogonalize(G), want)


def test_refusals_on_the_gpu():
    from capdec import ops
    G = gradient_like((40, 60))
    with pytest.raises(RuntimeError, match="capdec"):
        ops.orthogonalize(G, coeffs=(100.0, 0.0, 0.0))
    with pytest.raises(RuntimeError, match="capdec"):
        ops.orthogonalize(G, steps=0)
    with pytest.raises(RuntimeError, match="overlap"):
        ops.muon_step([G, G], [G, G], [G.clone(), G.clone()], lr=0.1)
    with pytest.raises(RuntimeError, match="overlap"):
        ops.muon_step([G], [G.clone()], [G], lr=0.1)
    with pytest.raises(RuntimeError, match="overlap"):
        ops.muon_step([G.clone()], [G], [G], lr=0.1)
    with pytest.raises(RuntimeError, match="overlap"):
        ops.orthogonalize([G, G.clone()], out=[G.clone(), G])
    with pytest.raises(RuntimeError, match="2-D|rows"):
        ops.orthogonalize(G.t())
    with pytest.raises(RuntimeError, match="type"):
        ops.orthogonalize(G.double())
