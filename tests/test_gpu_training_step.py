"""The training step with the vocabulary loss that keeps no logits and with orthogonalised updates: against the step it
replaces, against a plain loop in 64 bits, captured in a HIP graph, saved and resumed."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def model(E=64, V=150, L=2, seed=11):
    from models.vitattn_model import VITAttentionModel
    torch.manual_seed(seed)
    return VITAttentionModel(E, V, 4, L, dropout=0.0).cuda()


def batch(B=24, T=11, V=150, seed=0, dim=1000):
    g = torch.Generator().manual_seed(seed)
    feats = torch.rand(B, dim, generator=g).cuda()
    caps = torch.randint(4, V, (B, T + 1), generator=g)
    caps[:, 0] = 1
    for r in range(B):
        n = int(torch.randint(3, T, (1,), generator=g))
        caps[r, n] = 2
        caps[r, n + 1:] = 0
    return feats, caps.cuda()


def trainer(m, **kw):
    from capdec.trainer import CaptionTrainer
    torch.manual_seed(5)
    return CaptionTrainer(m, lr=1e-3, **kw)


def rnn_model():
    from models.cnnrnn_model import CNNtoRNN
    torch.manual_seed(12)
    m = CNNtoRNN(48, 80, 150).cuda()
    m.decoderRNN.dropout.p = 0.0
    return m


@pytest.mark.parametrize("skip_dead_rows", [True, False])
@pytest.mark.parametrize("kind", ["transformer", "lstm"])
def test_loss_in_pieces_gives_the_step_of_the_materialised_loss(kind, skip_dead_rows):
    """Same loss and gradients within the package's tolerance for fp32 paths, 1e-4 of the largest entry."""
    make = model if kind == "transformer" else rnn_model
    feats, caps = batch(dim=1000 if kind == "transformer" else 2048)
    got = []
    for how in ("logits", "pieces"):
        tr = trainer(make(), vocab_loss=how, skip_dead_rows=skip_dead_rows)
        loss = tr.step(feats, caps)
        got.append((loss, {n: g.clone() for n, g in tr.grads.items()}))
    assert got[1][0].shape == got[0][0].shape
    assert abs(float(got[0][0]) - float(got[1][0])) <= 1e-5 * float(got[0][0])
    top = max(float(g.abs().max()) for g in got[0][1].values())
    for n, g in got[0][1].items():
        assert float((g - got[1][1][n]).abs().max()) <= 1e-4 * max(float(g.abs().max()), 1e-3 * top), n


def newton_schulz(u):
    a, b, c = 3.4445, -4.7750, 2.0315
    x = u / (u.norm() + 1e-7)
    for _ in range(5):
        if x.shape[0] <= x.shape[1]:
            s = x @ x.T
            x = a * x + (b * s + c * s @ s) @ x
        else:
            s = x.T @ x
            x = a * x + x @ (b * s + c * s @ s)
    return x


@pytest.mark.parametrize("kind", ["transformer", "lstm"])
def test_muon_steps_the_matrices_and_adam_the_rest(kind):
    """Two steps; each parameter against its own rule in 64 bits, from the gradients the trainer left."""
    m = model() if kind == "transformer" else rnn_model()
    core = m if kind == "transformer" else m.decoderRNN
    tr = trainer(m, optimizer="muon", vocab_loss="pieces", muon_weight_decay=0.1)
    want = {n for n, p in core.named_parameters() if p.dim() == 2 and n.startswith(("decoder_layers.", "lstm."))}
    assert set(tr.muon_names) == want and len(want) == (20 if kind == "transformer" else 2)
    mom = {n: torch.zeros_like(p, dtype=torch.float64) for n, p in core.named_parameters()}
    sq = {n: torch.zeros_like(p, dtype=torch.float64) for n, p in core.named_parameters()}
    for t in (1, 2):
        feats, caps = batch(seed=t, dim=1000 if kind == "transformer" else 2048)
        before = {n: p.detach().double() for n, p in core.named_parameters()}
        tr.step(feats, caps)
        for n, p in core.named_parameters():
            g = tr.grads[n].double()
            if n in want:
                mom[n] = 0.95 * mom[n] + g
                if float(g.norm()) < 1e-6:
                    continue                    # (cross-attention over one memory row: no gradient reaches W_q and W_k)
                step = 1e-3 * 0.2 * max(p.shape) ** 0.5 * newton_schulz(g + 0.95 * mom[n])
                ref = before[n] * (1 - 1e-3 * 0.1) - step
            else:
                mom[n], sq[n] = 0.9 * mom[n] + 0.1 * g, 0.999 * sq[n] + 0.001 * g * g
                step = 1e-3 / (1 - 0.9 ** t) * mom[n] / (sq[n].sqrt() / (1 - 0.999 ** t) ** 0.5 + 1e-8)
                ref = before[n] - step
            # the update to 1e-4 of itself (entries far below the gradient's noise move freely under Adam), the sum to fp32
            assert float((p.detach().double() - ref).norm()) <= 1e-4 * float(step.norm()) + 2.0 ** -22 * float(ref.norm()) + 1e-7, n


@pytest.mark.parametrize("kw", [dict(vocab_loss="pieces"), dict(optimizer="muon"), dict(vocab_loss="pieces", optimizer="muon")])
def test_captured_steps_follow_launched_ones(kw):
    a, b = model(), model()
    ta, tb = trainer(a, **kw), trainer(b, graph=True, **kw)
    for t in range(5):
        feats, caps = batch(seed=t % 3)
        if t == 3:
            ta.scheduler_step(4)
            tb.scheduler_step(4)
        la, lb = float(ta.step(feats, caps)), float(tb.step(feats, caps))
        assert abs(la - lb) <= 2e-5 * abs(la), t
        torch.cuda.synchronize()
    for (k, va), (_, vb) in zip(a.state_dict().items(), b.state_dict().items()):
        # a bias in front of the BatchNorm and the keys' bias shift what is subtracted again: their gradient is zero but for
        # rounding, and Adam's step is the sign of that (the batch means hold the first of the two)
        if va.is_floating_point() and k not in ("fc_vit.bias", "batchnorm.running_mean") and not k.endswith("W_k.bias"):
            assert float((va - vb).abs().max()) <= 2.2 * 1e-3 * 5 * 1e-2 + 1e-6, k


def test_checkpoint_with_muon_resumes(tmp_path):
    from capdec.checkpoint import load_reference_checkpoint, save_reference_checkpoint
    a = model()
    ta = trainer(a, optimizer="muon")
    for t in range(2):
        ta.step(*batch(seed=t))
    path = str(tmp_path / "ck.pth.tar")
    out = save_reference_checkpoint(path, a, ta, step=2)
    assert set(out["muon"]) == set(ta.muon_names) and len(out["optimizer"]["state"]) == len(ta.grads) - len(ta.muon_names)
    b = model(seed=99)
    tb = trainer(b, optimizer="muon")
    assert load_reference_checkpoint(path, b, tb) == 2
    assert torch.equal(ta.m, tb.m) and torch.equal(ta.v, tb.v) and tb.t == 2
    assert all(torch.equal(x, y) for x, y in zip(a.state_dict().values(), b.state_dict().values()))
    la, lb = ta.step(*batch(seed=7)), tb.step(*batch(seed=7))
    assert abs(float(la) - float(lb)) <= 1e-6 * float(la)
    # into a trainer with Adam: the matrices start without moments; and an Adam checkpoint into one with Muon likewise
    c = model(seed=98)
    tc = trainer(c)
    load_reference_checkpoint(path, c, tc)
    save_reference_checkpoint(path, c, tc)
    load_reference_checkpoint(path, b, tb)
    assert all(int(m.count_nonzero()) == 0 for _, _, ms in tb.muon_groups.values() for m in ms)


def test_the_trainer_refuses_unknown_choices():
    from capdec.trainer import CaptionTrainer
    for kw in (dict(vocab_loss="chunks"), dict(optimizer="sgd")):
        with pytest.raises(ValueError, match="capdec"):
            CaptionTrainer(model(), **kw)
