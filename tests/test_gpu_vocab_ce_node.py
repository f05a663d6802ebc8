"""The vocabulary cross entropy as a node of autograd's graph: what it keeps, for how long, and whose memory it reads."""
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def make(M, V, K, dt, seed=0):
    g = torch.Generator("cuda").manual_seed(seed + M + V + K)
    x = torch.randn(M, K, device="cuda", generator=g).to(dt).requires_grad_()
    W = torch.nn.Parameter((torch.randn(V, K, device="cuda", generator=g) / K ** 0.5).to(dt))
    b = torch.randn(V, device="cuda", generator=g).to(dt).requires_grad_()
    t = torch.randint(1, V, (M,), device="cuda", generator=g)
    t[::5] = 0
    return x, W, b, t


def loss_of(x, W, b, t, reduction="mean"):
    from capdec import functional as F
    return F.vocab_cross_entropy(x, W, b, t, reduction=reduction)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("M", [20, 100])
def test_data_exchanged_in_between(M, dt):
    """A parameter whose ``data`` is exchanged after the forward pass: the gradients are of the values that it read."""
    x, W, b, t = make(M, 500, 64, dt)
    want = torch.autograd.grad(loss_of(x, W, b, t), (x, W, b))
    loss = loss_of(x, W, b, t)
    W.data = torch.full_like(W, float("nan"))
    more = [torch.full_like(W, float("nan")) for _ in range(8)]           # takes the memory of the old values if it is free
    got = torch.autograd.grad(loss, (x, W, b))
    assert len(more) == 8 and all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("dt", TYPES)
def test_what_the_node_keeps_goes_with_its_backward_pass(dt):
    x, W, b, t = make(3000, 2000, 64, dt)
    loss = loss_of(x, W, b, t)
    torch.autograd.grad(loss, (x, W, b))
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    kept = loss_of(x, W, b, t)
    held = torch.cuda.memory_allocated() - before
    assert held >= 3000 * 64 * x.element_size()                           # (the packed rows of x)
    grads = torch.autograd.grad(kept, (x, W, b))
    size = sum((g.numel() * g.element_size() + 511) // 512 * 512 for g in grads)
    # the loss (with the rows' losses beside it) is what stays of it
    assert torch.cuda.memory_allocated() - before - size <= 4 * 3003 + 1024
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(kept, (x, W, b))
    again = loss_of(x, W, b, t)
    for _ in range(2):
        got = torch.autograd.grad(again, (x, W, b), retain_graph=True)
        assert all(torch.equal(p, q) for p, q in zip(got, grads))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("M,K,off", [(100, 64, 0), (100, 64, 1), (20, 64, 1), (100, 33, 0)])
def test_saved_tensor_hooks(M, K, off, dt):
    """W and the node's buffer taken to the host and back in between, to other addresses and strides; W in place where it
    was packed and unaligned where it was in place."""
    _, W, b, t = make(M, 500, K, dt)
    wide = torch.zeros(500, K + 8, device="cuda", dtype=dt)
    wide[:, off:off + K] = W.detach()
    view = wide[:, off:off + K].requires_grad_()
    x = make(M, 500, K, dt)[0]
    want = torch.autograd.grad(loss_of(x, view, b, t), (x, view, b))
    seen = []

    def pack(v):
        seen.append(v.shape)
        return v.cpu(), v.shape == view.shape

    def to(shift):
        def unpack(p):
            v, is_w = p
            if not is_w:
                return v.cuda()
            buf = torch.full((500, K + 8), float("nan"), device="cuda", dtype=dt)
            buf[:, shift:shift + K] = v.cuda()
            return buf[:, shift:shift + K]
        return unpack
    for shift in (0, 1):
        with torch.autograd.graph.saved_tensors_hooks(pack, to(shift)):
            loss = loss_of(x, view, b, t)
        for _ in range(2):
            got = torch.autograd.grad(loss, (x, view, b), retain_graph=True)
            assert all(torch.equal(p, q) for p, q in zip(got, want))
    assert view.shape in seen and len(seen) == 4
    with torch.autograd.graph.save_on_cpu():
        loss = loss_of(x, view, b, t)
    got = torch.autograd.grad(loss, (x, view, b))
    assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("M", [0, 20, 100])
def test_loss_changed_in_place(M, reduction):
    """``loss /= n`` and the like, as on any other loss."""
    x, W, b, t = make(max(M, 1), 300, 64, torch.float32)
    x = x[:M]
    one = loss_of(x, W, b, t[:M], reduction)
    out = torch.ones_like(one)
    want = torch.autograd.grad(one, (W, b), out * 0.25)
    loss = loss_of(x, W, b, t[:M], reduction)
    loss /= 4
    got = torch.autograd.grad(loss, (W, b), out)
    assert torch.equal(loss, one / 4) or M == 0
    assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("M", [20, 100])
@pytest.mark.parametrize("which", [0, 1, 2])
def test_tangents_are_refused(which, M):
    """Forward-mode differentiation is not offered: an input's tangent is refused, not dropped, with and without gradients."""
    from torch.autograd import forward_ad as fw
    x, W, b, t = make(M, 300, 64, torch.float32)
    for grads in (False, True):
        ins = [v.detach().requires_grad_(grads) for v in (x, W, b)]
        with fw.dual_level():
            ins[which] = fw.make_dual(ins[which], torch.ones_like(ins[which]))
            with pytest.raises(RuntimeError, match="jvp|forward"):
                loss_of(*ins, t)
            with torch.no_grad(), pytest.raises(RuntimeError, match="jvp|forward"):
                loss_of(*ins, t)
    assert bool(loss_of(*(v.detach() for v in (x, W, b)), t).isfinite())


def test_recomputed_in_the_backward_pass():
    """Under torch's activation checkpointing, which runs the forward pass again."""
    from torch.utils.checkpoint import checkpoint
    x, W, b, t = make(100, 500, 64, torch.bfloat16)
    want = torch.autograd.grad(loss_of(x, W, b, t), (x, W, b))
    for reentrant in (False, True):
        ins = [v.detach().requires_grad_() for v in (x, W, b)]
        checkpoint(loss_of, *ins, t, use_reentrant=reentrant).backward()
        assert all(torch.equal(p.grad, q) for p, q in zip(ins, want))
