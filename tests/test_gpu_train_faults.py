"""GPU: what a training step does with arguments and states that are wrong."""
import pytest
import torch

from diffsvc_amd import synth
from diffsvc_amd.train import DiffusionTrainerHip
from test_gpu_train_tables import ARCHS, cuda, rel, setup


@pytest.mark.gpu
def test_frame_energies_below_zero_are_reported_while_training():
    """They have no row in the energy table (nn.Embedding raises at once); the steps read the sticky flag every CHECK_EVERY steps, before they
    change a weight."""
    hp, sd, clips, batch, energy, seed = setup("tiny")
    tr = DiffusionTrainerHip(hp, sd)
    hub, m2p, f0, mels, t = cuda(batch)
    step = lambda e: tr.train_step(hub, m2p, f0.clone(), mels, t=t, seed=seed, energy=e)
    energy = energy.cuda()
    bad = energy.clone()
    bad[0, 3] = -0.5
    tr.global_step = tr.CHECK_EVERY - 2
    step(bad)
    before = tr.params.clone()
    with pytest.raises(IndexError):
        step(energy)
    assert tr.global_step == tr.CHECK_EVERY and torch.equal(tr.params, before)
    tr.global_step = tr.CHECK_EVERY - 1                    # the flag is read once
    step(energy)
    assert not torch.equal(tr.params, before)


@pytest.mark.gpu
def test_a_step_that_fails_says_why_and_leaves_no_phase_open(monkeypatch):
    """33 layers with pitch: the last phase refuses them (host-side), after the layers have run.  The error is that one, also where d loss / d cond was
    asked for, and the handle takes the next step."""
    hp = dict(synth.tiny_hparams(K=50), residual_layers=33)
    monkeypatch.setitem(ARCHS, "deep", (hp,) + ARCHS["tiny"][1:])
    hp, sd, clips, batch, energy, seed = setup("deep")
    tr = DiffusionTrainerHip(hp, sd)
    hub, m2p, f0, mels, t = cuda(batch)
    ret = tr.fs2(hub, m2p, None, None, f0.clone(), None, energy.cuda(), infer=True)
    cond, pitch = ret["decoder_inp"].transpose(1, 2).contiguous(), ret["pitch_pred"].squeeze(-1)
    out = torch.zeros(*mels.shape[:2], hp["hidden_size"], device="cuda")
    for g in (out, None):
        with pytest.raises(RuntimeError, match="exceed the scratch"):
            tr.h.step(mels, cond, t, pitch=pitch, mel2ph=m2p, seed=seed, cond_grad=g)
    loss = tr.h.step(mels, cond, t, seed=seed, cond_grad=out)
    assert torch.isfinite(loss).all() and out.any()


@pytest.mark.gpu
def test_a_step_that_was_not_ended_gives_way_to_the_next():
    """An exception between the phases of a step with d loss / d cond (a failed all-reduce) does not close the trainer."""
    hp, sd, clips, batch, energy, seed = setup("tiny")
    tr = DiffusionTrainerHip(hp, sd)
    hub, m2p, f0, mels, t = cuda(batch)
    ret = tr.fs2(hub, m2p, None, None, f0.clone(), None, energy.cuda(), infer=True)
    cond, kw = ret["decoder_inp"].transpose(1, 2).contiguous(), dict(pitch=ret["pitch_pred"].squeeze(-1), mel2ph=m2p, seed=seed)
    want, out, L = torch.zeros(*mels.shape[:2], hp["hidden_size"], device="cuda"), torch.zeros(*mels.shape[:2], hp["hidden_size"], device="cuda"), hp["residual_layers"]
    tr.h.step(mels, cond, t, cond_grad=want, **kw)
    for layers in (0, 1):
        tr.h.step_begin(mels, cond, t, cond_grad=torch.zeros_like(out), **kw)
        if layers:
            tr.h.step_layers(L, L - 1)
        out.zero_()
        tr.h.step(mels, cond, t, cond_grad=out, **kw)
        assert rel(out, want) < 1e-6
        tr.h.step_begin(mels, cond, t, cond_grad=torch.zeros_like(out), **kw)
        out.zero_()
        tr.h.step_begin(mels, cond, t, cond_grad=out, **kw)
        tr.h.step_layers(L, 0)
        tr.h.step_end()
        assert rel(out, want) < 1e-6
    loss = tr.forward_backward(hub, m2p, f0, mels, t, seed=seed, energy=energy.cuda())
    assert torch.isfinite(loss).all()


def test_abandon_refuses_a_null_handle():
    from diffsvc_amd import _lib
    assert _lib.lib().dsvc_trainer_abandon(None) != 0 and b"null" in _lib.lib().dsvc_last_error()
