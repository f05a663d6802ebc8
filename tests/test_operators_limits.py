"""Largest sizes of the vocabulary cross entropy: what the size queries accept, a launch can hold."""
import pytest

BASE = 1 << 20


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("M,V", [(1 << 20, 1 << 19), (1 << 24, 1 << 15), (1 << 15, 1 << 24), (3 << 18, 699051), (100000, 5497558)])
def test_logits_launches_stay_below_2_32_work_items(M, V, dtype):
    from capdec import _lib
    lib = _lib.load()

    def accepted(m, v):
        a = _lib.VocabCE(BASE, BASE, None, BASE, 64, 64, 0, m, v, 64, dtype, 0)
        sizes = [f(a) for f in (lib.capdec_vocab_ce_saved_bytes, lib.capdec_vocab_ce_forward_workspace_bytes,
                                lib.capdec_vocab_ce_backward_workspace_bytes)]
        assert all(sizes) or not any(sizes)
        return bool(sizes[0])

    def work_items(m, v):
        """Of 256 x 256 tiles with 512 threads and of 256 x 128 ones with 256, their number rounded up to 8."""
        mp, vp = -(-m // 256) * 256, -(-v // 256) * 256
        return max(-(-(mp // 256 * (vp // 256)) // 8) * 8 * 512, -(-(mp // 128 * (vp // 256)) // 8) * 8 * 256)
    assert not accepted(M, V)                                    # 2^39 or just above
    below = V
    while not accepted(M, below):
        below -= 256
        assert V - below <= 1 << 16
    assert work_items(M, below) < 1 << 32 and M * below > (1 << 39) - (1 << 33)
    for m, v in ((M // 2, V), (M, V // 2), (M // 2, V // 3)):
        assert accepted(m, v) and work_items(m, v) < 1 << 32


def test_forward_refuses_what_cannot_be_launched():
    from capdec import _lib
    lib = _lib.load()
    a = _lib.VocabCE(BASE, BASE, None, BASE, 64, 64, 0, 1 << 20, 1 << 19, 64, 1, 0)
    n = 1 << 40
    assert lib.capdec_vocab_ce_forward(a, BASE, n, BASE, n, BASE, None, None) == -22
    assert lib.capdec_vocab_ce_backward(a, BASE, n, BASE, n, None, None, 1, BASE, 64, BASE, 64, None, None) == -22


def test_tiles_of_sizes():
    import ctypes

    from capdec import _lib
    lib = _lib.load()
    t = (ctypes.c_int32 * 3)(7, 7, 7)

    def a(M, dtype=0, loss_only=0, V=1000):
        return _lib.VocabCE(BASE, BASE, None, BASE, 64, 64, 0, M, V, 64, dtype, loss_only)
    assert lib.capdec_vocab_ce_tiles(None, t) == -22 and lib.capdec_vocab_ce_tiles(a(100), None) == -22
    assert lib.capdec_vocab_ce_tiles(a(0), t) == -22 and tuple(t) == (7, 7, 7)
    assert lib.capdec_vocab_ce_tiles(a(64), t) == 0 and tuple(t) == (0, 0, 0)            # float32: kernels without tiles
    for dtype in (0, 1, 2):
        assert lib.capdec_vocab_ce_tiles(a(65, dtype), t) == 0 and tuple(t) == (128 * 128, 256 * 128, 256 * 128)
        assert lib.capdec_vocab_ce_tiles(a(65, dtype, 1), t) == 0 and tuple(t) == (128 * 128, 0, 0)
