"""Checkpoints between trainers of different optimizers."""
import warnings

import pytest
import torch

pytestmark = pytest.mark.gpu


def model(seed):
    from models.vitattn_model import VITAttentionModel
    torch.manual_seed(seed)
    return VITAttentionModel(64, 150, 4, 2, dropout=0.0).cuda()


def batch(seed):
    g = torch.Generator().manual_seed(seed)
    caps = torch.randint(4, 150, (24, 12), generator=g)
    caps[:, 0], caps[:, -2], caps[:, -1] = 1, 2, 0
    return torch.rand(24, 1000, generator=g).cuda(), caps.cuda()


def trainer(m, **kw):
    from capdec.trainer import CaptionTrainer
    return CaptionTrainer(m, lr=1e-3, **kw)


@pytest.mark.parametrize("stepped", [0, 3])
def test_momentum_checkpoint_into_a_trainer_with_adam(tmp_path, stepped):
    """Adam starts afresh, whatever the trainer held: the first update is |g| / (|g| + eps) of the learning rate."""
    from capdec.checkpoint import load_reference_checkpoint, save_reference_checkpoint
    a = model(1)
    ta = trainer(a, optimizer="muon")
    for t in range(4):
        ta.step(*batch(t))
    path = str(tmp_path / "ck.pth.tar")
    save_reference_checkpoint(path, a, ta, step=4)
    b = model(2)
    tb = trainer(b)
    for t in range(stepped):
        tb.step(*batch(20 + t))
    with pytest.warns(UserWarning, match="afresh"):
        assert load_reference_checkpoint(path, b, tb) == 4
    assert all(torch.equal(x, y) for x, y in zip(a.state_dict().values(), b.state_dict().values()))
    assert tb.t == 0 and int(tb.m.count_nonzero()) == 0 and int(tb.v.count_nonzero()) == 0
    before = tb.flat_p.clone()
    tb.step(*batch(7))
    assert tb.t == 1
    step = (tb.flat_p - before).abs().double()
    # rounding: the update's own (lr, quotient, correction) and half a step of the parameter
    assert bool((step <= 1e-3 * (1 + 2.0 ** -20) + 2.0 ** -24 * before.abs().double().clamp(min=1e-3) * 2).all())
    assert float(step.max()) >= 0.9e-3


def test_checkpoints_of_one_optimizer_do_not_warn(tmp_path):
    from capdec.checkpoint import load_reference_checkpoint, save_reference_checkpoint
    for kw in (dict(), dict(optimizer="muon")):
        a, b = model(1), model(2)
        ta, tb = trainer(a, **kw), trainer(b, **kw)
        ta.step(*batch(0))
        tb.step(*batch(1))
        path = str(tmp_path / "ck.pth.tar")
        save_reference_checkpoint(path, a, ta)
        with warnings.catch_warnings():
            warnings.simplefilter("error")
            load_reference_checkpoint(path, b, tb)
        assert torch.equal(ta.m, tb.m) and torch.equal(ta.v, tb.v) and tb.t == 1
