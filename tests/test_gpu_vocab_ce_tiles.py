"""The vocabulary cross entropy at the sizes that select each of its tiles, against the definition in 64 bits."""
import ctypes

import pytest
import torch

from test_gpu_vocab_ce import check, make

pytestmark = pytest.mark.gpu

MID, BIG, WIDE = 128 * 128, 256 * 128, 256 * 256


def tiles_of(M, V, K, dt, loss_only=False):
    from capdec import _lib
    at = 1 << 20
    code = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}[dt]
    t = (ctypes.c_int32 * 3)()
    assert _lib.load().capdec_vocab_ce_tiles(_lib.VocabCE(at, at, at, at, K, K, 0, M, V, K, code, loss_only), t) == 0
    return tuple(t)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,V,K,want", [
    (300, 2000, 96, (MID, BIG, BIG)),
    (2000, 9000, 64, (BIG, BIG, BIG)),              # parts of dx and of dW, joined afterwards
    (2000, 16500, 2048, (WIDE, WIDE, WIDE)),        # dx in parts
    (8100, 2000, 2048, (WIDE, WIDE, WIDE)),         # dW in parts
    (1700, 16500, 1536, (WIDE, BIG, WIDE))])
def test_gradients_with_every_tile(M, V, K, want, dt):
    """With a bias and ignored rows; a retuned rule that leaves a tile without a test shows here."""
    assert tiles_of(M, V, K, dt) == want
    x, W, b, t = make(M, V, K, dt, seed=70)
    t[-1] = V - 1
    check(x, W, b, t, "mean")


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,V,K,want", [(300, 2000, 96, MID), (2000, 9000, 64, BIG), (2000, 16500, 2048, WIDE)])
def test_loss_alone_with_every_tile(M, V, K, want, dt):
    from capdec import functional as F
    from test_gpu_vocab_ce import definition, near
    assert tiles_of(M, V, K, dt, True) == (want, 0, 0)
    x, W, b, t = make(M, V, K, dt, seed=71)
    t[-1] = V - 1
    (nll, *_), (tol, *_) = definition(x, W, b, t, torch.zeros(M, device="cuda"))
    near(F.vocab_cross_entropy(x, W, b, t, reduction="none"), nll, torch.full_like(nll, tol), "loss")


def test_largest_number_of_logits():
    """2^20 rows over 2^19 - 512 words, 2^29 logits short of the accepted 2^39; sampled rows, the last among them."""
    from capdec import functional as F
    M, V, K = 1 << 20, (1 << 19) - 512, 32
    g = torch.Generator("cuda").manual_seed(1)
    x = torch.randn(M, K, device="cuda", generator=g).bfloat16()
    W = (torch.randn(V, K, device="cuda", generator=g) * 0.3).bfloat16()
    t = torch.randint(0, V, (M,), device="cuda", generator=g)
    t[-1] = V - 1
    nll = F.vocab_cross_entropy(x, W, None, t, ignore_index=-1, reduction="none")
    rows = torch.cat([torch.arange(8), torch.randint(0, M, (48,), generator=torch.Generator().manual_seed(2)), torch.arange(M - 8, M)]).cuda()
    z = x[rows].double() @ W.double().T
    want = torch.logsumexp(z, 1) - z.gather(1, t[rows, None])[:, 0]
    # exact products, K + 1 fp32 sums of at most S; 200 additions and three roundings of exponents up to Z
    S, Z = float((x[rows].double().abs() @ W.double().abs().T).max()), float(z.abs().max()) * 1.4427
    assert float((nll[rows].double() - want).abs().max()) <= 2 * (K + 1) * 2.0 ** -24 * S + (3 * Z + 200) * 2.0 ** -23
    assert bool(nll.isfinite().all())
