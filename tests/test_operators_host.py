"""Host side of the vocabulary cross entropy and of the orthogonalised update: sizes and refusals, on a machine without
a GPU (every call is turned down before anything is launched)."""
import ctypes

import pytest
import torch

EINVAL, ENOMEM, EALIGN = -22, -12, -14
BASE = 1 << 20                # stands for device memory: only the address is looked at


def ce(**kw):
    from capdec import _lib
    d = dict(x=BASE, W=BASE, bias=None, targets=BASE, ldx=64, ldw=64, ignore_index=0, M=100, V=1000, K=64, dtype=0)
    d.update(kw)
    return _lib.VocabCE(**d)


def test_vocab_ce_sizes():
    from capdec import _lib
    lib = _lib.load()
    for dtype, packed in ((0, 1000 * 64 * 4), (1, 0), (2, 0)):
        a = ce(dtype=dtype)
        assert packed <= lib.capdec_vocab_ce_saved_bytes(a) < packed + 256 * 64 * 4 + 16384
        # G of at most 512 MiB, the gradient's partial sums, never a logits matrix of 32 bits
        big = ce(dtype=dtype, M=100000, V=200000)
        assert lib.capdec_vocab_ce_backward_workspace_bytes(big) < (512 << 20) + 17 * 100096 * 64 * 4 + 17 * 200192 * 64 * 4
    assert lib.capdec_vocab_ce_saved_bytes(ce(dtype=1, K=50, ldw=50)) > 1000 * 64 * 2      # odd widths are packed
    for bad in (dict(M=0), dict(V=0), dict(K=0), dict(dtype=3), dict(dtype=-1), dict(M=1 << 25), dict(V=1 << 25), dict(K=1 << 21),
                dict(M=1 << 24, V=1 << 19)):
        a = ce(**bad)
        assert lib.capdec_vocab_ce_saved_bytes(a) == 0 and lib.capdec_vocab_ce_backward_workspace_bytes(a) == 0
    assert lib.capdec_vocab_ce_saved_bytes(None) == 0


def test_vocab_ce_refusals():
    from capdec import _lib
    lib = _lib.load()
    n = 1 << 30

    def fwd(a, saved=BASE, ns=n, ws=BASE, nw=n, nll=BASE):
        return lib.capdec_vocab_ce_forward(a, saved, ns, ws, nw, nll, None, None)

    def bwd(a, saved=BASE, ns=n, ws=BASE, nw=n, row=None, g=BASE, dx=BASE, ldx=64, dW=BASE, ldw=64, db=None):
        return lib.capdec_vocab_ce_backward(a, saved, ns, ws, nw, row, g, 1, dx, ldx, dW, ldw, db, None)
    for bad in (dict(x=None), dict(W=None), dict(targets=None), dict(M=0), dict(V=-1), dict(K=0), dict(dtype=7),
                dict(ldx=63), dict(ldw=63)):
        assert fwd(ce(**bad)) == EINVAL and bwd(ce(**bad)) == EINVAL
    a = ce()
    assert fwd(None) == EINVAL and fwd(a, nll=None) == EINVAL and fwd(a, saved=None) == EINVAL and fwd(a, ws=None) == EINVAL
    assert fwd(a, saved=BASE + 4) == EALIGN and fwd(a, ws=BASE + 8) == EALIGN
    assert fwd(a, ns=lib.capdec_vocab_ce_saved_bytes(a) - 1) == ENOMEM
    assert fwd(a, nw=lib.capdec_vocab_ce_forward_workspace_bytes(a) - 1) == ENOMEM
    assert bwd(a, row=BASE) == EINVAL and bwd(a, ldx=63) == EINVAL and bwd(a, ldw=60) == EINVAL
    assert bwd(a, db=BASE) == EINVAL                                       # a bias gradient without a bias
    assert bwd(a, ns=100) == ENOMEM and bwd(a, nw=lib.capdec_vocab_ce_backward_workspace_bytes(a) - 1) == ENOMEM
    assert bwd(a, ws=BASE + 4) == EALIGN
    assert bwd(a, dx=None, dW=None) == 0                                   # nothing wanted, nothing launched


def test_orthogonalize_and_muon_refusals():
    from capdec import _lib
    lib = _lib.load()
    co = (ctypes.c_float * 3)(3.4445, -4.7750, 2.0315)
    n = 1 << 40

    def ortho(rows=40, cols=60, count=1, dtype=0, steps=5, c=co, eps=1e-7, ws=BASE, nw=n, **m):
        d = dict(src=BASE, dst=BASE, ld_src=60, ld_dst=60)
        d.update(m)
        return lib.capdec_orthogonalize((_lib.Matrix * 1)(_lib.Matrix(**d)), count, rows, cols, dtype, steps, c, eps, ws, nw, None)
    for bad in (dict(rows=0), dict(cols=-1), dict(count=0), dict(dtype=3), dict(steps=0), dict(steps=33), dict(c=None),
                dict(src=None), dict(dst=None), dict(ld_src=59), dict(ld_dst=59), dict(ws=None), dict(eps=-1.0),
                dict(eps=float("nan")), dict(c=(ctypes.c_float * 3)(9.0, 0.0, 0.0)), dict(rows=1 << 20, cols=1 << 12),
                dict(c=(ctypes.c_float * 3)(float("nan"), 0.0, 0.0)), dict(c=(ctypes.c_float * 3)(2.0, float("inf"), 0.0))):
        assert ortho(**bad) == EINVAL, bad
    assert ortho(ws=BASE + 4) == EALIGN
    assert ortho(nw=lib.capdec_orthogonalize_workspace_bytes(1, 40, 60) - 1) == ENOMEM
    assert lib.capdec_orthogonalize_workspace_bytes(0, 4, 4) == 0 and lib.capdec_orthogonalize_workspace_bytes(1, 0, 4) == 0
    # many matrices go through in batches: the workspace stops growing
    assert lib.capdec_orthogonalize_workspace_bytes(500, 64, 64) == lib.capdec_orthogonalize_workspace_bytes(32, 64, 64)

    def muon(count=1, rows=40, cols=60, steps=5, c=co, ws=BASE, nw=n, **m):
        d = dict(p=BASE, g=BASE, m=BASE, ldp=60, ldg=60, ldm=60)
        d.update(m)
        return lib.capdec_muon_step((_lib.MuonParam * 1)(_lib.MuonParam(**d)), count, rows, cols, 0.1, None, 0.9, 1, 0.0, 1.0, 1.0,
                                    steps, c, 1e-7, ws, nw, None)
    for bad in (dict(p=None), dict(g=None), dict(m=None), dict(ldp=59), dict(ldg=59), dict(ldm=59), dict(count=-1),
                dict(steps=-1), dict(ws=None), dict(c=None)):
        assert muon(**bad) == EINVAL, bad
    assert muon(ws=BASE + 4) == EALIGN and muon(nw=16) == ENOMEM


def test_overlapping_matrices_are_told_apart():
    """Rows of one matrix, columns of one wider matrix and separate ones do not overlap; anything shared does."""
    from capdec import ops
    w = torch.zeros(20, 60)
    ops._check_overlap("t", [w[:10], w[10:]])
    ops._check_overlap("t", [w[:, :20], w[:, 20:40], w[:, 40:], torch.zeros(20, 60)])
    ops._check_overlap("t", [w[3:9, 40:50]], [w[3:9, 50:]])
    ops._check_overlap("t", [torch.zeros(4, 4)], [w, w, w[:5]])            # what is only read may be the same twice
    for written, read in (([w, w], []), ([w[:11], w[10:]], []), ([w[:, :21], w[:, 20:40]], []), ([w], [w]),
                          ([w[:, 10:30]], [w[5:6, 29:35]]), ([w[:10]], [w[9:, :1]]), ([w[2:4]], [w]), ([w[0:1], w[0:1]], [])):
        with pytest.raises(RuntimeError, match="overlap"):
            ops._check_overlap("t", written, read)


def test_python_wrappers_refuse_what_they_cannot_take():
    from capdec import functional as F
    from capdec import ops
    x, W, t = torch.zeros(4, 8), torch.zeros(10, 8), torch.zeros(4, dtype=torch.long)
    with pytest.raises(RuntimeError, match="GPU"):
        F.vocab_cross_entropy(x, W, None, t)
    with pytest.raises(ValueError, match="reduction"):
        F.vocab_cross_entropy(x, W, None, t, reduction="max")
    with pytest.raises(RuntimeError, match="fit"):
        F.vocab_cross_entropy(x, W, None, t[:3])
    with pytest.raises(RuntimeError, match="GPU"):
        ops.orthogonalize(torch.zeros(4, 4))
    with pytest.raises(RuntimeError, match="matrix"):
        ops.orthogonalize(torch.zeros(4))
    with pytest.raises(RuntimeError, match="lr"):
        ops.muon_step([], [], [])
    with pytest.raises(RuntimeError, match="GPU"):
        ops.muon_step([x], [x], [x], lr=0.1)
