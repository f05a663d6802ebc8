"""Vocabulary cross entropy without kept logits: loss and gradients against the definition in 64 bits.

Tolerances.  Let u be half a step of the operands' type (2^-24, 2^-8 for bfloat16, 2^-11 for float16).
  logits: every product of the split fp32 operands is off by at most 3 * 2^-22 of itself (both low parts rounded, their
  product left out; 16-bit products are exact) and a sum of K + 1 terms in fp32 by at most (K + 1) 2^-24 of the sum of
  magnitudes S = |x| |W|^T + |b|: dz = (3 * 2^-22 + (K + 1) 2^-24) S.
  softmax: exp2 in fp32 of a number of size Z = max |z| log2(e), rounded three times, over a sum of V terms added in a tree of
  depth < 200:  dp / p <= 2 dz + (3 Z + 200) 2^-23.
  gradients: G is rounded once to the operands' type (fp32: to 22 bits), its contraction's sum again in fp32 and the result
  to the type:  |d| <= (dp/p + g + n 2^-24) sum |G| |other| + u |result|, with g = u (fp32: 2^-22) and n the length of the sum.
  expm1 at the target adds 4 * 2^-24 + dz, which the bound of dp / p covers.  There G is p - 1, and an error dp of p (or of
  log p) stays dp while the difference may vanish (a vocabulary of one word): the dp term is of p, not of |G|, so it is
  taken over  H = p + [v = t] >= |G|:  |d| <= (dp/p) sum H |other| + (g + n 2^-24) sum |G| |other| + u |result|.
  fp16 numbers (also the pairs that fp32 takes) end in steps of 2^-24: G, stored times at least 2^13 / max |w|, is off by
  half a step, 2^-38 max |w|, however small it is; over a sum that is 2^-38 max |w| sum |other|.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TYPES = list(U)


def make(M, V, K, dt, seed=0, bias=True, ignored=0.25, ignore=0):
    g = torch.Generator("cuda").manual_seed(1000 * seed + M + V + K)
    x = torch.randn(M, K, device="cuda", generator=g).to(dt)
    W = (torch.randn(V, K, device="cuda", generator=g) * 1.5 / math.sqrt(K)).to(dt)
    b = torch.randn(V, device="cuda", generator=g).to(dt) if bias else None
    t = torch.randint(0, V, (M,), device="cuda", generator=g)
    if ignored:
        t[torch.rand(M, device="cuda", generator=g) < ignored] = ignore
    return x, W, b, t


def definition(x, W, b, t, w, ignore=0):
    """nll, dx, dW, db for the upstream gradients ``w`` of the rows, and the error bounds of the module's docstring."""
    K, V = x.shape[1], W.shape[0]
    u = U[x.dtype]
    x, W = x.double(), W.double()
    bb = torch.zeros(V, device=x.device, dtype=torch.float64) if b is None else b.double()
    live = t != ignore
    z = x @ W.T + bb
    lse = torch.logsumexp(z, 1)
    at = torch.where(live, t, 0)
    nll = torch.where(live, lse - z.gather(1, at[:, None])[:, 0], 0.0)
    G = torch.softmax(z, 1)
    H = G.clone()
    G[torch.arange(len(t), device=t.device), at] -= 1.0
    H[torch.arange(len(t), device=t.device), at] += 1.0
    G, H = G * (w.double() * live)[:, None], H * (w.double().abs() * live)[:, None]
    S = x.abs() @ W.abs().T + torch.where(bb.isfinite(), bb.abs(), 0.0)
    S, Z = S[live].max().item() if live.any() else 0.0, z[live][z[live].isfinite()].abs().max().item() if live.any() else 0.0
    dz = (3 * 2.0 ** -22 + (K + 1) * 2.0 ** -24) * S
    dp = 2 * dz + (3 * Z * 1.4427 + 200) * 2.0 ** -23
    g = 2.0 ** -22 if u == 2.0 ** -24 else u

    floor = 0.0 if u == 2.0 ** -8 else 2.0 ** -38 * float(w.abs().max())

    def bound(A, H, B, n):
        return floor * B.abs().sum(0) + dp * (H @ B.abs()) + (g + n * 2.0 ** -24) * (A.abs() @ B.abs()) + u * (A @ B).abs()
    n_live = int(live.sum())
    res = [nll, G @ W, G.T @ x, G.sum(0)]
    tol = [dz * 2 + (3 * Z + 200) * 2.0 ** -23, bound(G, H, W, V), bound(G.T, H.T, x, n_live),
           floor * n_live + dp * H.sum(0) + (g + n_live * 2.0 ** -24) * G.abs().sum(0) + u * G.sum(0).abs()]
    return res, tol


def near(got, want, tol, what, subnormal=0.0):
    err = (got.double() - want).abs()
    assert got.shape == want.shape, what
    assert bool((err <= tol + subnormal).all()), f"{what}: {float((err - tol).max()):.3e} over the bound, error {float(err.max()):.3e}"


def run(x, W, b, t, reduction, w, ignore=0):
    from capdec import functional as F
    x, W = x.detach().requires_grad_(), W.detach().requires_grad_()
    b = None if b is None else b.detach().requires_grad_()
    loss = F.vocab_cross_entropy(x, W, b, t, ignore_index=ignore, reduction=reduction)
    ins = [v for v in (x, W, b) if v is not None]
    grads = torch.autograd.grad(loss, ins, w if reduction == "none" else None)
    return loss.detach(), grads


def check(x, W, b, t, reduction="mean", ignore=0, w=None):
    n = max(1, int((t != ignore).sum()))
    if reduction == "none":
        w = torch.rand(len(t), device=x.device) + 0.1 if w is None else w
        rows = w
    else:
        rows = torch.full((len(t),), 1.0 / n if reduction == "mean" else 1.0, device=x.device)
    loss, grads = run(x, W, b, t, reduction, w, ignore)
    (nll, *want), (tn, *tol) = definition(x, W, b, t, rows, ignore)
    if reduction == "none":
        near(loss, nll, torch.full_like(nll, tn), "loss")
    else:
        total = nll.sum() / (n if reduction == "mean" else 1)
        near(loss, total, (tn * n + 2.0 ** -22 * nll.abs().sum()) / (n if reduction == "mean" else 1), "loss")
    sub = 2.0 ** -25 if x.dtype == torch.float16 else 0.0          # half a step of fp16's smallest numbers
    for got, ref, bound, name in zip(grads, want, tol, ("dx", "dW", "db")):
        assert got.dtype == x.dtype
        near(got, ref, bound, name, sub)
    return loss, grads


SIZES = [(1, 1, 1), (1, 2, 3), (1, 5, 32), (3, 257, 33), (31, 300, 40), (64, 255, 64), (65, 256, 31), (128, 1000, 96),
         (129, 513, 333), (500, 2049, 128), (1030, 777, 512), (2000, 5000, 65)]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("size", SIZES)
def test_loss_and_gradients(size, dt):
    x, W, b, t = make(*size, dt)
    t[0] = size[1] - 1 if size[1] > 1 else 0
    check(x, W, b if size[0] % 2 else None, t, "mean", ignore=0 if size[1] > 1 else -100)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_reductions_and_ignored_rows(reduction, dt):
    for ignored in (0.0, 0.5, 0.95):
        x, W, b, t = make(300, 1100, 96, dt, seed=1, ignored=ignored, ignore=-100)
        check(x, W, b, t, reduction, ignore=-100)


def test_row_weights_of_any_size():
    """Upstream gradients of the rows over many orders of magnitude, zero among them."""
    x, W, b, t = make(200, 600, 64, torch.float32, seed=2)
    w = torch.rand(200, device="cuda") * 1e-12
    w[3] = 0.0
    check(x, W, b, t, "none", w=w)
    w[5] = 1.0
    check(x, W, b, t, "none", w=w * 1e20)


@pytest.mark.parametrize("dt", TYPES)
def test_no_counted_row(dt):
    x, W, b, t = make(70, 300, 64, dt)
    t[:] = 0
    loss, grads = run(x, W, b, t, "mean", None)
    assert math.isnan(loss.item()) and all(int(g.count_nonzero()) == 0 for g in grads)
    loss, grads = run(x, W, b, t, "sum", None)
    assert loss.item() == 0.0 and all(int(g.count_nonzero()) == 0 for g in grads)


def test_empty_batch():
    x, W, b, t = make(4, 300, 64, torch.float32)
    loss, grads = run(x[:0], W, b, t[:0], "mean", None)
    assert math.isnan(loss.item()) and grads[0].shape == (0, 64) and all(int(g.count_nonzero()) == 0 for g in grads)
    assert run(x[:0], W, b, t[:0], "sum", None)[0].item() == 0.0


def test_ignored_rows_are_not_read():
    """Rows behind an ignored target may hold anything: infinities, NaN, uninitialised memory."""
    x, W, b, t = make(300, 500, 64, torch.float32, seed=3)
    want = run(x, W, b, t, "mean", None)
    y = x.clone()
    y[t == 0] = float("nan")
    y[(t == 0).nonzero()[0]] = float("inf")
    got = run(y, W, b, t, "mean", None)
    assert torch.equal(got[0], want[0]) and all(torch.equal(a, c) for a, c in zip(got[1], want[1]))


@pytest.mark.parametrize("dt", TYPES)
def test_masked_words(dt):
    """Words masked by a bias of -inf or of the type's lowest value: whole tiles of them, and all but one."""
    x, W, b, t = make(100, 700, 64, dt, seed=4, ignored=0.0)
    b[:300] = float("-inf")
    b[300:400] = torch.finfo(dt).min
    t[:] = torch.randint(400, 700, (100,), device="cuda")
    loss, grads = check(x, W, b, t, "mean", ignore=-1)
    assert int(grads[1][:400].count_nonzero()) == 0 and int(grads[2][:400].count_nonzero()) == 0
    b[:] = float("-inf")
    b[650] = 0.5
    t[:] = 650
    loss, grads = run(x, W, b, t, "mean", None, ignore=-1)
    assert abs(loss.item()) < 1e-5 and all(bool(g.isfinite().all()) for g in grads)


def test_nan_stays_in_its_row():
    x, W, b, t = make(200, 400, 64, torch.float32, seed=5, ignored=0.0)
    want, _ = run(x, W, b, t, "none", torch.ones(200, device="cuda"), ignore=-1)
    x[7, 3] = float("nan")
    x[11, 3] = float("inf")
    got, grads = run(x, W, b, t, "none", torch.ones(200, device="cuda"), ignore=-1)
    bad = torch.zeros(200, dtype=torch.bool, device="cuda")
    bad[[7, 11]] = True
    assert bool(got[7].isnan()) and not bool(got[11].isfinite()) and torch.equal(got[~bad], want[~bad])
    assert bool(grads[0][7].isnan().all()) and bool(grads[0][~bad].isfinite().all())


def test_target_outside_the_vocabulary_is_nan():
    for bad in (-5, 400, 2 ** 40):
        x, W, b, t = make(50, 400, 64, torch.float32, seed=6)
        t[9] = bad
        loss, grads = run(x, W, b, t, "mean", None)
        assert math.isnan(loss.item()) and bool(grads[0][9].isnan().all())
        assert bool(grads[0][torch.arange(50) != 9].isfinite().all())


@pytest.mark.parametrize("dt", TYPES)
def test_strides_and_alignment(dt):
    x, W, b, t = make(130, 520, 96, dt, seed=7)
    want = run(x, W, b, t, "sum", None)
    for off in (1, 8):
        wide_x = torch.full((130, 120), float("nan"), device="cuda", dtype=dt)
        wide_w = torch.full((520, 130), float("nan"), device="cuda", dtype=dt)
        wide_x[:, off:off + 96], wide_w[:, off:off + 96] = x, W
        got = run(wide_x[:, off:off + 96], wide_w[:, off:off + 96], b, t, "sum", None)
        assert torch.equal(got[0], want[0]) and all(torch.equal(a, c) for a, c in zip(got[1], want[1]))
    # x whose columns are not contiguous is copied by the call; targets of any shape
    from capdec import functional as F
    got = F.vocab_cross_entropy(x.t().contiguous().t().view(10, 13, 96), W, b, t.view(10, 13), reduction="none")
    assert got.shape == (10, 13) and torch.equal(got.sum(), F.vocab_cross_entropy(x, W, b, t, reduction="none").view(10, 13).sum())


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("M,V,K,bias", [(1, 5000, 512, True), (7, 70001, 100, False), (100, 300, 33, True), (192, 1000, 64, True),
                                         (193, 1000, 64, False), (700, 2000, 128, True)])
def test_loss_alone(M, V, K, bias, dt):
    """The loss where nothing asks for gradients."""
    from capdec import functional as F
    x, W, b, t = make(M, V, K, dt, seed=15, bias=bias, ignored=0.3)
    t[0] = V - 1
    (nll, *_), (tol, *_) = definition(x, W, b, t, torch.zeros(M, device="cuda"))
    got = F.vocab_cross_entropy(x, W, b, t, reduction="none")
    near(got, nll, torch.full_like(nll, tol), "loss")
    n = int((t != 0).sum())
    for red, want in (("sum", nll.sum()), ("mean", nll.sum() / n)):
        got = F.vocab_cross_entropy(x, W, b, t, reduction=red)
        near(got, want, (tol * n + 2.0 ** -22 * nll.sum()) / (n if red == "mean" else 1), red)
        assert torch.equal(got, F.vocab_cross_entropy(x, W, b, t, reduction=red))
    if M > 2:
        y = x.clone()
        y[t == 0] = float("nan")
        assert torch.equal(F.vocab_cross_entropy(y, W, b, t, reduction="sum"), F.vocab_cross_entropy(x, W, b, t, reduction="sum"))
        t[1] = V
        assert math.isnan(F.vocab_cross_entropy(x, W, b, t).item())
        t[:] = 0
        assert math.isnan(F.vocab_cross_entropy(x, W, b, t).item()) and F.vocab_cross_entropy(x, W, b, t, reduction="sum").item() == 0
    if bias:
        b[:V // 2] = float("-inf")
        t[:] = torch.randint(V // 2, V, (M,), device="cuda")
        (nll, *_), (tol, *_) = definition(x, W, b, t, torch.zeros(M, device="cuda"), ignore=-1)
        near(F.vocab_cross_entropy(x, W, b, t, ignore_index=-1, reduction="none"), nll, torch.full_like(nll, tol), "loss")


def test_broadcast_inputs():
    """Rows of x that are one row: its gradient is the sum of theirs."""
    from capdec import functional as F
    x, W, b, t = make(40, 300, 64, torch.float32, seed=13, ignored=0.3)
    row = x[:1].detach().requires_grad_()
    g, = torch.autograd.grad(F.vocab_cross_entropy(row.expand(40, 64), W, b, t), (row,))
    (nll, dx, _, _), (_, tol, _, _) = definition(row.detach().expand(40, 64), W, b, t, torch.full((40,), 1 / int((t != 0).sum()), device="cuda"))
    near(g, dx.sum(0, keepdim=True), tol.sum(0, keepdim=True) + 40 * 2.0 ** -24 * dx.abs().sum(0, keepdim=True), "dx")


def test_operands_changed_in_between_are_noticed():
    from capdec import functional as F
    x, W, b, t = make(40, 300, 64, torch.float32, seed=14)
    W.requires_grad_()
    loss = F.vocab_cross_entropy(x, W, b, t)
    with torch.no_grad():
        W += 1
    with pytest.raises(RuntimeError, match="modified"):
        loss.backward()


def test_gradients_written_into_given_buffers_with_strides():
    from capdec import ops
    x, W, b, t = make(130, 520, 96, torch.float32, seed=8)
    nll, loss, saved = ops.vocab_ce_forward(x, W, b, t)
    one = torch.ones(1, device="cuda")
    want = ops.vocab_ce_backward(saved, grad=one)
    bx, bw = torch.full((130, 100), 7.0, device="cuda"), torch.full((520, 101), 7.0, device="cuda")
    got = ops.vocab_ce_backward(saved, grad=one, dx=bx[:, :96], dW=bw[:, :96])
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    assert bool((bx[:, 96:] == 7).all()) and bool((bw[:, 96:] == 7).all())
    assert all(torch.equal(a, c) for a, c in zip(ops.vocab_ce_backward(saved), want))        # no upstream gradient: 1
    only = ops.vocab_ce_backward(saved, grad=one, need=(False, False, True))
    assert only[0] is None and only[1] is None and torch.equal(only[2], want[2])
    only = ops.vocab_ce_backward(saved, grad=one, need=(False, True, False))
    assert torch.equal(only[1], want[1])


@pytest.mark.parametrize("dt", TYPES)
def test_large_and_tiny_values(dt):
    """Logits of hundreds, and operands at the ends of the type's range (fp32 operands are scaled by their largest)."""
    x, W, b, t = make(100, 300, 64, dt, seed=9)
    check((x.float() * 12).to(dt), W, b, t, "mean")
    if dt == torch.float32:
        check(x * 1e-18, W * 1e18, b, t, "mean")
        check(x * 1e15, W * 1e-15, None, t, "mean")
        check(x * 0, W, b, t, "mean")


def test_gradient_against_differences():
    """Central differences of the fp32 loss along random directions.  The loss of size L is known to about 2^-22 L, so a
    step h leaves 2^-22 L / h of noise and h^2 / 6 of the third derivative (below |d|^3, |d| = the logits' change)."""
    from capdec import functional as F
    x, W, b, t = make(60, 200, 32, torch.float32, seed=10)
    loss, (dx, dW, db) = run(x, W, b, t, "mean", None)
    g = torch.Generator("cuda").manual_seed(3)
    for k, (v, dv) in enumerate(((x, dx), (W, dW), (b, db))):
        d = torch.randn(v.shape, device="cuda", generator=g)
        d /= d.norm()
        h = 0.02
        ins = [x, W, b]

        def at(s):
            ins[k] = v + s * d
            return F.vocab_cross_entropy(*ins, t).double().item()
        diff = (at(h) - at(-h)) / (2 * h)
        reach = max(1.0, float(W.norm(dim=1).max()), float(x.norm(dim=1).max()))
        assert abs(diff - float((dv * d).sum())) <= 2.0 ** -20 * float(loss) / h + h * h * min(reach, 8.0) ** 3 / 6


@pytest.mark.parametrize("dt", TYPES)
def test_repeats_bit_for_bit_and_on_another_stream(dt):
    x, W, b, t = make(700, 3000, 160, dt, seed=11)
    want = run(x, W, b, t, "mean", None)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = run(x, W, b, t, "mean", None)
    s.synchronize()
    again = run(x, W, b, t, "mean", None)
    for r in (got, again):
        assert torch.equal(r[0], want[0]) and all(torch.equal(a, c) for a, c in zip(r[1], want[1]))


def test_captured_and_replayed():
    """Forward and backward in one HIP graph, replayed with new inputs, other work in between; two graphs side by side."""
    from capdec import ops
    graphs = []
    one = torch.ones(1, device="cuda")
    for n in range(2):
        x, W, b, t = make(260, 900, 96, torch.float32, seed=20 + n)

        def step(x=x, W=W, b=b, t=t):
            nll, loss, saved = ops.vocab_ce_forward(x, W, b, t)
            return (loss,) + ops.vocab_ce_backward(saved, grad=one)
        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        graphs.append((graph, outs, (x, W, b, t), step))
    for r in range(3):
        for n, (graph, outs, ins, step) in enumerate(graphs):
            fresh = make(260, 900, 96, torch.float32, seed=30 + 2 * r + n, ignored=0.2 * r)
            for dst, src in zip(ins, fresh):
                dst.copy_(src)
        for graph, *_ in graphs:
            graph.replay()
        got = [[o.clone() for o in outs] for _, outs, _, _ in graphs]
        torch.cuda.synchronize()
        for have, (_, _, _, step) in zip(got, graphs):
            assert all(torch.equal(a, c) for a, c in zip(have, step()))


def test_pieces_of_the_vocabulary():
    """A batch and vocabulary whose gradient matrix takes more than one piece (512 MiB each)."""
    M, V, K = 30000, 10007, 32
    for dt in (torch.bfloat16, torch.float32):
        x, W, b, t = make(M, V, K, dt, seed=12)
        check(x, W, b, t, "mean")


def test_offsets_past_32_bits():
    """A vocabulary matrix of more than 2^31 elements: loss, and the gradients of the words at its end."""
    V, K, M = 1100001, 2048, 40
    g = torch.Generator("cuda").manual_seed(5)
    W = torch.empty(V, K, device="cuda", dtype=torch.bfloat16)
    for i in range(0, V, 100000):
        W[i:i + 100000] = torch.randn(min(100000, V - i), K, device="cuda", generator=g) * 0.03
    x = torch.randn(M, K, device="cuda", generator=g).bfloat16()
    t = torch.randint(V - 1000, V, (M,), device="cuda", generator=g)
    loss, (dx, dW) = run(x, W, None, t, "mean", None)
    z = torch.cat([x.double() @ W[i:i + 100000].double().T for i in range(0, V, 100000)], 1)
    lse = torch.logsumexp(z, 1)
    want = (lse - z.gather(1, t[:, None])[:, 0]).mean()
    assert abs(loss.item() - want.item()) <= 1e-5 * abs(want.item())
    G = torch.softmax(z, 1)
    G[torch.arange(M), t] -= 1
    G /= M
    u = U[torch.bfloat16]
    end = G[:, -1000:].T @ x.double()
    # twice u: G's rounding and the result's, plus a sixteenth for the fp32 sums
    near(dW[-1000:], end, (1 + 1 / 16) * u * (G[:, -1000:].abs().T @ x.double().abs() + end.abs()), "dW")
    ref, mag = torch.zeros(M, K, device="cuda", dtype=torch.float64), torch.zeros(M, K, device="cuda", dtype=torch.float64)
    for i in range(0, V, 100000):
        w = W[i:i + 100000].double()
        ref += G[:, i:i + 100000] @ w
        mag += G[:, i:i + 100000].abs() @ w.abs()
    near(dx, ref, (1 + 1 / 16) * u * (mag + ref.abs()), "dx")


@pytest.mark.parametrize("M,V,K", [(1, 300, 512), (2, 1, 4), (16, 1000, 36), (17, 4097, 30), (32, 515, 65), (33, 2000, 200), (48, 30, 1),
                                   (63, 6000, 515), (64, 777, 96), (64, 70000, 64), (20, 40000, 52)])
@pytest.mark.parametrize("reduction", ["mean", "none"])
def test_few_rows(M, V, K, reduction):
    """Batches of at most 64 rows of fp32, in groups of 16 slots: counted rows below and at the ends of the groups."""
    for ignored in (0.0, 0.4):
        x, W, b, t = make(M, V, K, torch.float32, seed=21, ignored=ignored, ignore=-100)
        if reduction == "mean" and bool((t == -100).all()):          # (one row, ignored: the mean over none)
            assert run(x, W, b, t, "mean", None, -100)[0].isnan()
            continue
        check(x, W, b if M % 3 else None, t, reduction, ignore=-100)


def test_few_rows_upstream_gradients_far_apart():
    """Rows whose upstream gradient is 1e-12 of the largest keep their accuracy in dx: bound of the row alone."""
    x, W, b, t = make(40, 900, 72, torch.float32, seed=22, ignored=0.0, ignore=-100)
    w = torch.logspace(0, -12, 40, device="cuda")
    _, (dx, *_) = run(x, W, b, t, "none", w, -100)
    (_, want, *_), (_, tol, *_) = definition(x, W, b, t, w, -100)
    floor = 2.0 ** -38 * W.double().abs().sum(0)              # of the largest gradient, which these rows need not allow for
    near(dx, want, tol - floor, "dx")


@pytest.mark.parametrize("M", [5, 24, 64])
def test_few_rows_layouts(M):
    """Rows of x, W and the gradients at any stride and offset; what lies beside and behind them stays; a second backward."""
    from capdec import ops
    V, K = 530, 100
    x, W, b, t = make(M, V, K, torch.float32, seed=23, ignored=0.3)
    t[M - 1] = V - 1
    one = torch.ones((), device="cuda")
    want = None
    for off in (0, 1, 4):
        xs, ws, gx, gw = (torch.full((r + 2, K + 30 + off), 7.0, device="cuda") for r in (M, V, M, V))
        xv, wv, dx, dW = (a[1:-1, off:off + K] for a in (xs, ws, gx, gw))
        xv.copy_(x), wv.copy_(W)
        nll, loss, state = ops.vocab_ce_forward(xv, wv, b, t)
        xs.fill_(float("nan"))                                # the backward call has a copy of x, and reads W again
        for _ in range(2):
            dx.zero_(), dW.zero_()
            db = torch.zeros_like(b)
            ops.vocab_ce_backward(state, grad=one, mean=True, dx=dx, dW=dW, db=db)
            got = [v.clone() for v in (nll, loss, dx, dW, db)]
            want = got if want is None else want
            assert all(torch.equal(p, q) for p, q in zip(got, want))
        for a, v in ((gx, dx), (gw, dW)):
            v.fill_(7.0)
            assert bool((a == 7.0).all())


def test_few_rows_masked_and_out_of_range():
    from capdec import functional as F
    x, W, b, t = make(20, 700, 64, torch.float32, seed=24, ignored=0.0)
    t[:] = 650
    b[:600] = float("-inf")
    loss, (dx, dW, db) = check(x, W, b, t, "sum", ignore=-100)
    assert bool((dW[:600] == 0).all()) and bool((db[:600] == 0).all())
    t[3:] = -100
    y = x.clone()
    y[3:] = float("nan")                                      # rows that are not counted are not read
    _, grads = run(y, W, b, t, "mean", None, -100)
    assert bool(grads[0][:3].isfinite().all()) and bool((grads[0][3:] == 0).all()) and bool(grads[1].isfinite().all())
    t[:] = -100
    _, grads = run(y, W, b, t, "sum", None, -100)
    assert all(bool((g == 0).all()) for g in grads)
    t[1] = 700
    assert math.isnan(F.vocab_cross_entropy(x, W, b, t, ignore_index=-100).item())


def test_few_rows_captured():
    """Loss and gradients in a graph, replayed with other values between eager calls."""
    from capdec import ops
    x, W, b, t = make(30, 3000, 128, torch.float32, seed=25)
    dx, dW, db = torch.empty_like(x), torch.empty_like(W), torch.empty_like(b)

    def step():
        nll, loss, state = ops.vocab_ce_forward(x, W, b, t)
        ops.vocab_ce_backward(state, grad=None, mean=True, dx=dx, dW=dW, db=db)
        return loss
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = step()
    for k in range(4):
        x.copy_(torch.randn_like(x) * (k + 1))
        t.copy_(torch.randint(0, 3000, t.shape, device="cuda"))
        graph.replay()
        got = [v.clone() for v in (loss, dx, dW, db)]
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, (want, dx, dW, db)))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("M", [12, 150])
def test_rows_sure_of_their_target(M, dt):
    """Logits far above the others at the targets.  The target's logit and the sum have the same roundings, which cancel as
    its probability goes to 1: the loss is off by 2 (1 - p) dz, by what up to 200 additions to a sum near 1 round off (half
    a step of 2^-23 each, and no more than the 1 - p that is added) and by the roundings of the sum, its logarithm and one
    product, 4 * 2^-23 - not by dz, here (K + 1) 2^-24 times some hundred.  No loss below -4 * 2^-23."""
    K, V = 128, 700
    g = torch.Generator("cuda").manual_seed(31)
    W = torch.randn(V, K, device="cuda", generator=g).to(dt)
    t = torch.randint(0, V, (M,), device="cuda", generator=g)
    x = (W[t].float() * torch.linspace(0.02, 1.5, M, device="cuda")[:, None]).to(dt)
    b = torch.randn(V, device="cuda", generator=g).to(dt)
    w = torch.ones(M, device="cuda")
    loss, _ = run(x, W, b, t, "none", w, -100)
    z = x.double() @ W.double().T + b.double()
    nll = torch.logsumexp(z, 1) - z.gather(1, t[:, None])[:, 0]
    rest = -torch.expm1(-nll)                                 # 1 - p
    S = x.double().abs() @ W.double().abs().T + b.double().abs()
    dz = (3 * 2.0 ** -22 + (K + 1) * 2.0 ** -24) * S.max()
    Z = z.abs().max() * 1.4427
    tol = 2 * dz * rest + (3 * Z + 200) * 2.0 ** -23 * rest + rest.clamp(max=200 * 2.0 ** -24) + 4 * 2.0 ** -23
    near(loss, nll, tol, "loss")
    assert float(loss.min()) >= -4 * 2.0 ** -23 and float(nll.min()) < 1e-12 and float(nll.max()) > 1e-3


def test_gradients_in_shared_memory():
    """Gradients written over W or over one another are refused; dx in x's own memory is right."""
    from capdec import ops
    for M, dt in ((40, torch.float32), (100, torch.float32), (100, torch.bfloat16)):
        x, W, b, t = make(M, 300, 64, dt, seed=41)
        _, _, state = ops.vocab_ce_forward(x, W, b, t)
        both = torch.empty(300 + M, 64, device="cuda", dtype=dt)
        for bad in (dict(dW=W), dict(dx=W[:M]), dict(dx=both[:M], dW=both[M - 1:M + 299]), dict(db=W.view(-1)[64:364])):
            with pytest.raises(RuntimeError, match="overlaps"):
                ops.vocab_ce_backward(state, **bad)
        want = ops.vocab_ce_backward(state)
        got = ops.vocab_ce_backward(state, dx=x, dW=both[M:])
        assert all(torch.equal(p, q) for p, q in zip(got, want)) and got[0] is x


@pytest.mark.parametrize("M,V,K", [(65, 500, 33), (70, 1000, 64), (200, 3000, 130), (700, 40000, 300), (600, 9000, 1540), (4200, 20000, 2048)])
def test_loss_alone_of_float32_rows_of_any_size(M, V, K):
    """Without gradients every row of x and W has a scale of its own: rows 1e-12 and 1e12 times the others keep their digits.
    Bound of a row's logits from that row's own sums of magnitudes; no state that gradients could be taken from."""
    from capdec import functional as F, ops
    x, W, b, t = make(M, V, K, torch.float32, seed=51, ignored=0.2)
    t[0] = V - 1
    x[1:3] *= 1e-12
    W[V // 2:V // 2 + 40] *= 1e-12
    W[5] *= 1e12
    x[:, :] = torch.where(torch.arange(K, device="cuda") < K // 2, x, -x.abs() * W[5].sign())      # (word 5 far below the others)
    b[5] = -1e30
    x[4] = 0
    live = t != 0
    z = x.double() @ W.double().T + b.double()
    S = x.double().abs() @ W.double().abs().T + b.double().abs()
    keep = [v for v in range(V) if v != 5]
    z, S = z[:, keep], S[:, keep]
    t2 = torch.where(t > 5, t - 1, t)
    ok = live & (t != 5)
    nll = torch.logsumexp(z, 1) - z.gather(1, t2[:, None])[:, 0]
    dz = (3 * 2.0 ** -22 + (K + 1) * 2.0 ** -24) * S.max(1).values
    tol = 2 * dz + (3 * z.abs().max(1).values * 1.4427 + 200) * 2.0 ** -23
    got = F.vocab_cross_entropy(x, W, b, t, reduction="none")
    assert bool((got[~live] == 0).all())
    near(got[ok], nll[ok], tol[ok], "loss")
    _, _, state = ops.vocab_ce_forward(x, W, b, t, loss_only=True)
    with pytest.raises(RuntimeError, match="loss alone"):
        ops.vocab_ce_backward(state)
