"""What rounding takes off the targets' entries of the logits' gradient, which 16-bit operands carry beside it.

Every checked sum has one term, the target's: G = (p - 1) w times a row of W or of x, whose product with G is the exact
result.  So the result may be off by half of ITS last place and by what p is known to, and by nothing for G's own rounding
to 16 bits, which would take it up to half a place further.

p is known to dp = 2 dz + (3 Z + 200) 2^-23 of itself, with dz = (K + 1) 2^-24 S and S, Z the largest sum of magnitudes and logit
(exact products, sums in fp32, three rounded exponents, 200 additions).  What is carried is itself rounded to 16 bits (dW, db:
u^2 of G; dx: fp32), and three fp32 roundings follow (expm1's 4 steps, the sum, the factor): 8 * 2^-24."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def half_place(v, dt):
    """Half a unit in the last place of v in the type (of its smallest normal numbers below them)."""
    low = -126 if dt == torch.bfloat16 else -14
    e = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** low)))
    return torch.exp2(e) * U[dt]


def gradients(x, W, b, t, w):
    from capdec import functional as F
    x, W = x.detach().requires_grad_(), W.detach().requires_grad_()
    b = b.detach().requires_grad_() if b is not None else None
    loss = F.vocab_cross_entropy(x, W, b, t, ignore_index=-1, reduction="none")
    return torch.autograd.grad(loss, [v for v in (x, W, b) if v is not None], w)


def target_entries(x, W, b, t, w):
    """(p - 1) w of each row in 64 bits, and what p w is known to."""
    z, S = [], 0.0
    for i in range(0, len(W), 200000):
        wd = W[i:i + 200000].double()
        z.append(x.double() @ wd.T + (0 if b is None else b[i:i + 200000].double()))
        S = max(S, float((x.double().abs() @ wd.abs().T + (0 if b is None else b[i:i + 200000].double().abs())).max()))
    z = torch.cat(z, 1)
    nll = torch.logsumexp(z, 1) - z.gather(1, t[:, None])[:, 0]
    p = torch.exp(-nll)
    dp = 2 * (x.shape[1] + 1) * 2.0 ** -24 * S + (3 * 1.4427 * float(z.abs().max()) + 200) * 2.0 ** -23
    return torch.expm1(-nll) * w.double(), dp * p * w.double()


def holds(got, want, known, dt, carried):
    """known: what the target's entry is known to, times the other factor; carried: rounding of what is carried"""
    tol = half_place(want, dt) * (1 + 2.0 ** -10) + known + (8 * 2.0 ** -24 + carried) * want.abs()
    over = (got.double() - want).abs() - tol
    assert bool((over <= 0).all()), f"{float((over / tol).max()):.2f} of the bound over it"


@pytest.mark.parametrize("dt", list(U))
@pytest.mark.parametrize("M,V", [(1, 300), (30, 300), (64, 1000), (200, 700), (2000, 9000)])
def test_dx(M, V, dt):
    """W is zero but for the one word that is every row's target."""
    g = torch.Generator("cuda").manual_seed(M + V)
    K = 32
    x = torch.randn(M, K, device="cuda", generator=g).to(dt)
    W = torch.zeros(V, K, device="cuda", dtype=dt)
    W[V // 2] = (torch.randn(K, device="cuda", generator=g) * 0.3).to(dt)
    b = torch.zeros(V, device="cuda", dtype=dt)
    b[V // 2] = 6.0
    t = torch.full((M,), V // 2, device="cuda")
    w = torch.rand(M, device="cuda", generator=g) * 0.5 + 0.5
    dx, _, _ = gradients(x, W, b, t, w)
    G, known = target_entries(x, W, b, t, w)
    row = W[V // 2].double()
    holds(dx, G[:, None] * row, known[:, None] * row.abs(), dt, 0.0)


def own_columns(M, K, V, dt, g):
    """Rows of x on columns of their own, targets of their own."""
    c = K // M
    x = torch.zeros(M, K, device="cuda")
    cols = torch.arange(M, device="cuda")[:, None] * c + torch.arange(c, device="cuda")
    x.scatter_(1, cols, torch.randn(M, c, device="cuda", generator=g))
    t = torch.randperm(V, device="cuda", generator=g)[:M]
    return x.to(dt), cols, t


@pytest.mark.parametrize("dt", list(U))
@pytest.mark.parametrize("M,V,K", [(1, 300, 40), (30, 300, 240), (64, 1000, 512), (64, 40000, 512)])
def test_dW_and_db(M, V, K, dt):
    g = torch.Generator("cuda").manual_seed(M + V + K)
    x, cols, t = own_columns(M, K, V, dt, g)
    W = (torch.randn(V, K, device="cuda", generator=g) * 0.2).to(dt)
    b = torch.zeros(V, device="cuda", dtype=dt)
    b[t] = 4.0
    w = torch.rand(M, device="cuda", generator=g) * 0.5 + 0.5
    _, dW, db = gradients(x, W, b, t, w)
    G, known = target_entries(x, W, b, t, w)
    xs = x.double().gather(1, cols)
    holds(dW[t].gather(1, cols), G[:, None] * xs, known[:, None] * xs.abs(), dt, U[dt] ** 2)
    # db: every row's entry of the word, none rounded to 16 bits alone
    z = x.double() @ W.double().T + b.double()
    P = torch.softmax(z, 1) * w.double()[:, None]
    P[torch.arange(M), t] = G
    want = P.sum(0)
    dp = float((known / (w.double() + G)).max())              # known = dp p w, w + G = p w
    tol = half_place(want, dt) * (1 + 2.0 ** -10) + (dp + U[dt] ** 2 + (M + 8) * 2.0 ** -24) * (P.abs() + (P == G[:, None]) * w.double()[:, None]).sum(0)
    if dt == torch.float16:
        tol = tol + M * 2.0 ** -38
    assert bool(((db.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("dt", list(U))
def test_targets_in_a_later_piece(dt):
    """A vocabulary of more than one piece (512 MiB of gradient): targets in the first and in the second."""
    g = torch.Generator("cuda").manual_seed(9)
    M, V, K = 40, 1100000, 320
    x, cols, t = own_columns(M, K, V, dt, g)
    t[:20] = torch.randperm(2000, device="cuda", generator=g)[:20]
    t[20:] = V - 1 - torch.randperm(2000, device="cuda", generator=g)[:20]
    W = torch.zeros(V, K, device="cuda", dtype=dt)
    # (a target's row of W lies on its own columns too: dx has one term)
    W[t] = torch.zeros(M, K, device="cuda").scatter_(1, cols, torch.randn(M, K // M, device="cuda", generator=g) * 0.3).to(dt)
    w = torch.rand(M, device="cuda", generator=g) * 0.5 + 0.5
    dx, dW = gradients(x, W, None, t, w)
    G, known = target_entries(x, W, None, t, w)
    xs, ws = x.double().gather(1, cols), W[t].double().gather(1, cols)
    holds(dW[t].gather(1, cols), G[:, None] * xs, known[:, None] * xs.abs(), dt, U[dt] ** 2)
    holds(dx.gather(1, cols), G[:, None] * ws, known[:, None] * ws.abs(), dt, 0.0)
