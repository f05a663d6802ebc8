"""The vocabulary cross entropy at the sizes that select each of its tiles, against the definition in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu


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
