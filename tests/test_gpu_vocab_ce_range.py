"""The vocabulary cross entropy of float32 operands over fp32's range."""
import pytest
import torch

from test_gpu_vocab_ce import definition, make, near, run

pytestmark = pytest.mark.gpu


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
