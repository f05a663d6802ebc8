"""The vocabulary cross entropy of float32 operands over fp32's range: rows far apart, very small and large ones.

Bounds are those of test_gpu_vocab_ce.definition, taken of the rows and words that count: a word whose bias is -inf, or a row
whose upstream gradient is zero, is left out of the definition, since it enters nothing."""
import pytest
import torch

from test_gpu_vocab_ce import definition, make, near, run

pytestmark = pytest.mark.gpu

# rows, words, width: with 128 x 128, 256 x 128 and 256 x 256 tiles of the logits, odd sizes, parts of the contractions
SIZES = [(70, 1000, 64), (100, 500, 33), (200, 3000, 130), (700, 40000, 96), (1024, 13000, 1024), (1700, 16500, 768)]


@pytest.mark.parametrize("scale", [(1e-30, 1), (1, 1e-30), (1e-30, 1e30), (1e30, 1e-30)])
@pytest.mark.parametrize("M", [40, 100])
def test_very_small_and_large_operands(M, scale):
    """Gradients relative to their own size, each operand at an end of the range."""
    x, W, b, t = make(M, 300, 64, torch.float32, seed=60)
    x, W = x * scale[0], W * scale[1]
    w = torch.rand(M, device="cuda") + 0.1
    loss, grads = run(x, W, b, t, "none", w)
    (nll, *want), (tn, *tol) = definition(x, W, b, t, w)
    near(loss, nll, torch.full_like(nll, tn), "loss")
    for got, ref, bound, name in zip(grads, want, tol, ("dx", "dW", "db")):
        # half a step of fp32's smallest numbers, twice (a factor, the result)
        near(got, ref, bound, name, 2.0 ** -149)
    from capdec import functional as F
    near(F.vocab_cross_entropy(x, W, b, t, reduction="none"), nll, torch.full_like(nll, tn), "loss alone")


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("far", [1e6, 1e9, 1e30])
def test_a_masked_word_far_larger_than_the_others(size, far):
    """It may not cost the other words digits, with gradients as without."""
    from capdec import functional as F
    M, V, K = size
    x, W, b, t = make(M, V, K, torch.float32, seed=61)
    W[5] *= far
    b[5] = float("-inf")
    t[t == 5] = 6
    keep = torch.arange(V, device="cuda") != 5
    w = torch.rand(M, device="cuda") + 0.1
    loss, (dx, dW, db) = run(x, W, b, t, "none", w)
    (nll, *want), (tn, *tol) = definition(x, W[keep], b[keep], torch.where(t > 5, t - 1, t), w)
    for got, ref, bound, name in zip((dx, dW[keep], db[keep]), want, tol, ("dx", "dW", "db")):
        near(got, ref, bound, name)
    assert int(dW[5].count_nonzero()) == 0 and float(db[5]) == 0.0
    near(loss, nll, torch.full_like(nll, tn), "loss")
    near(F.vocab_cross_entropy(x, W, b, t, reduction="none"), nll, torch.full_like(nll, tn), "loss alone")


@pytest.mark.parametrize("size", SIZES)
def test_rows_far_apart(size):
    """Rows 1e-12 times the others, and one 1e9 times the others without an upstream gradient."""
    M, V, K = size
    x, W, b, t = make(M, V, K, torch.float32, seed=62)
    x[1:4] *= 1e-12
    t[1:4] = V - 1
    x[7] *= 1e9
    t[7] = 1
    w = torch.rand(M, device="cuda") + 0.1
    w[7] = 0.0
    loss, (dx, dW, db) = run(x, W, b, t, "none", w)
    keep = torch.arange(M, device="cuda") != 7
    (nll, ref, *want), (tn, bound, *tol) = definition(x[keep], W, b, t[keep], w[keep])
    near(loss[keep], nll, torch.full_like(nll, tn), "loss")
    near(dx[keep], ref, bound, "dx")
    assert int(dx[7].count_nonzero()) == 0
    for got, r, bd, name in zip((dW, db), want, tol, ("dW", "db")):
        near(got, r, bd, name)
    # the small rows by their own sums of magnitudes: their logits are the bias
    (nll, *_), (tn, *_) = definition(x[1:4], W, b, t[1:4], w[1:4])
    near(loss[1:4], nll, torch.full_like(nll, tn), "loss of the small rows")


def test_rows_far_apart_captured():
    """One graph, replayed with operands that are far apart and with ones that are not."""
    from capdec import ops
    x, W, b, t = make(150, 900, 96, torch.float32, seed=63)
    ins = [v.clone() for v in (x, W, b)]

    def step():
        _, loss, state = ops.vocab_ce_forward(*ins, t)
        return (loss,) + ops.vocab_ce_backward(state)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for k in range(5):
        for dst, src in zip(ins, make(150, 900, 96, torch.float32, seed=64 + k)):
            dst.copy_(src)
        if k % 2:
            ins[1][17] *= 1e8
            ins[2][17] = float("-inf")
            t[t == 17] = 18
        graph.replay()
        got = [o.clone() for o in outs]
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, step())) and all(bool(p.isfinite().all()) for p in got)


def test_zero_rows_are_not_far_apart():
    """Rows of zeros (a padding word) leave the operands as pairs: the same bits as without them."""
    x, W, b, t = make(100, 600, 64, torch.float32, seed=65, ignored=0.0, ignore=-1)
    t[t >= 590] = 3
    W[590:] = 0
    b[590:] = float("-inf")
    want = run(x, W[:590], b[:590], t, "sum", None, -1)
    got = run(x, W, b, t, "sum", None, -1)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1][1][:590], want[1][1])


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,V,K", [(20, 700, 64), (100, 700, 64), (300, 9000, 800)])
def test_a_word_of_infinite_distance(M, V, K, dt):
    """A weight of -inf against positive entries of x: the word's logits are -inf, the others as if it were not there.  In
    dx its column is 0 * inf."""
    from capdec import functional as F
    x, W, b, t = make(M, V, K, dt, seed=66)
    x[:, 3] = x[:, 3].abs() + 0.5
    W[5, 3] = float("-inf")
    t[t == 5] = 6
    keep = torch.arange(V, device="cuda") != 5
    w = torch.rand(M, device="cuda") + 0.1
    loss, (dx, dW, db) = run(x, W, b, t, "none", w)
    (nll, ref, *want), (tn, bound, *tol) = definition(x, W[keep], b[keep], torch.where(t > 5, t - 1, t), w)
    sub = 2.0 ** -25 if dt == torch.float16 else 0.0
    near(loss, nll, torch.full_like(nll, tn), "loss")
    cols = torch.arange(K, device="cuda") != 3
    near(dx[:, cols], ref[:, cols], bound[:, cols], "dx", sub)
    assert bool(dx[t != 0, 3].isnan().all())
    for got, r, bd, name in zip((dW, db), want, tol, ("dW", "db")):
        near(got[keep], r, bd, name, sub)
    assert int(dW[5].count_nonzero()) == 0
    near(F.vocab_cross_entropy(x, W, b, t, reduction="none"), nll, torch.full_like(nll, tn), "loss alone")


@pytest.mark.parametrize("reduction", ["mean", "none"])
@pytest.mark.parametrize("M,dt,far", [(40, torch.float32, False), (100, torch.float32, False), (100, torch.float32, True),
                                      (100, torch.bfloat16, False)])
def test_weights_near_the_end_of_the_range(M, dt, far, reduction):
    """W up to 1e36 and more against an x of 1e-36: the gradient of the logits carries no factor that its products could overflow by
    before it is undone."""
    x, W, b, t = make(M, 300, 64, dt, seed=67)
    x, W = (x.float() * 1e-36).to(dt), (W.float() * 1e36).to(dt)
    if far:
        W[7] = W[7] * 1e-30
    w = torch.rand(M, device="cuda") + 0.1 if reduction == "none" else torch.full((M,), 1 / int((t != 0).sum()), device="cuda")
    loss, grads = run(x, W, b, t, reduction, w if reduction == "none" else None)
    (_, *want), (_, *tol) = definition(x, W, b, t, w)
    assert bool(loss.isfinite().all())
    near(grads[0], want[0], tol[0], "dx")
    # x has fewer digits at its small end, and its products with G may leave the range: steps of 2^-149 each
    near(grads[1], want[1], tol[1] + M * 2.0 ** -149, "dW", 2.0 ** -134 if dt == torch.bfloat16 else 0.0)
    near(grads[2], want[2], tol[2], "db")


def test_far_rows_in_pieces_and_at_odd_strides():
    """More than one piece of the vocabulary, operands and gradients inside wider matrices at odd offsets."""
    from capdec import ops
    M, V, K = 30000, 10007, 37
    x, W, b, t = make(M, V, K, torch.float32, seed=68)
    W[5] *= 1e8
    b[5] = float("-inf")
    t[t == 5] = 6
    xs, ws, gx, gw = (torch.full((r, K + 6), 7.0, device="cuda") for r in (M, V, M, V))
    xv, wv, dx, dW = (v[:, 1:1 + K] for v in (xs, ws, gx, gw))
    xv.copy_(x), wv.copy_(W)
    _, loss, state = ops.vocab_ce_forward(xv, wv, b, t)
    xs.fill_(float("nan"))
    _, _, db = ops.vocab_ce_backward(state, dx=dx, dW=dW)
    keep = torch.arange(V, device="cuda") != 5
    w = torch.full((M,), 1 / int((t != 0).sum()), device="cuda")
    (nll, *want), (tn, *tol) = definition(x, W[keep], b[keep], torch.where(t > 5, t - 1, t), w)
    near(loss[0], nll.sum() * float(w[0]), tn + 2.0 ** -22 * nll.sum() * float(w[0]), "loss")
    for got, ref, bound, name in zip((dx, dW[keep], db[keep]), want, tol, ("dx", "dW", "db")):
        near(got, ref, bound, name)
    assert int(dW[5].count_nonzero()) == 0
    for wide in (gx, gw):
        assert bool((wide[:, 0] == 7).all()) and bool((wide[:, 1 + K:] == 7).all())
