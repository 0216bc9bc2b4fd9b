"""GPU: what a training step does with arguments and states that are wrong."""
import pytest
import torch

from diffsvc_amd.train import DiffusionTrainerHip
from test_gpu_train_tables import cuda, setup


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
