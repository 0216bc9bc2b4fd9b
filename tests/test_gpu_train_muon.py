"""GPU: the ``matrix_optimizer: muon`` step of the 44.1 kHz architecture -- seven groups of 384 x 384 up to 20 x 768 x 1152, whole tiles beside K slices --
against momentum, Newton-Schulz products and the weight step in float64 on the device, the rest of the tensors against torch.optim.AdamW."""
import pytest
import torch

from diffsvc_amd import muon
from diffsvc_amd.train import ENERGY, DiffusionTrainerHip, muon_groups
from test_gpu_muon import limit
from test_gpu_train_tables import setup


@pytest.mark.gpu
@pytest.mark.parametrize("precision", [None, "f16"])
def test_step_of_the_44k_architecture(precision):
    """Tolerance of an update: ``limit`` of test_gpu_muon.py, three times the distance of the formula with rounded operands from float64 and six standard
    deviations of an element, computed here for every matrix (it grows with the shape: a constant number of half steps is no bound), times the
    size of the step; the momentum's two and the weight's three float32 roundings of each step come to it."""
    hp, sd, _, _, _, _ = setup("44k", lr=1e-3, weight_decay=0.01, clip_grad_norm=1.0, matrix_optimizer="muon", muon_lr=2e-3, muon_precision=precision)
    tr = DiffusionTrainerHip(hp, sd)
    groups, _ = muon_groups(tr.layout, tr.shapes)
    at = {o: n for n, o, _ in tr.layout}
    inner = {at[off + i * stride]: (rows, cols) for off, b, stride, rows, cols in groups for i in range(b)}
    others = [n for n, _, _ in tr.layout if n not in inner]
    assert (20, 768, 1152) in [(b, r, c) for _, b, _, r, c in groups] and ENERGY in others
    ref = {n: sd[n].cuda().double() for n, _, _ in tr.layout}
    mom = {n: torch.zeros(inner[n], device="cuda", dtype=torch.float64) for n in inner}
    adam = [torch.nn.Parameter(sd[n].cuda().float()) for n in others]
    opt = torch.optim.AdamW(adam, lr=hp["lr"], betas=(0.9, 0.98), weight_decay=0.01)
    g = torch.Generator(device="cuda").manual_seed(4)
    lim = dict.fromkeys(inner, 0.0)
    for it in range(2):
        tr.grads.copy_(torch.randn(tr.n_floats, generator=g, device="cuda") * 0.02)
        grads = {n: tr.view(tr.grads, n).clone() for n, _, _ in tr.layout}
        coef = float(1.0 / (torch.stack([v.double().square().sum() for v in grads.values()]).sum().sqrt() + 1e-6))
        assert coef < 1
        tr.optimizer_step()
        for n, (rows, cols) in inner.items():
            gr = grads[n].double().reshape(rows, cols) * coef
            m = mom[n].mul_(0.95).add_(gr, alpha=0.05)
            with torch.device("cuda"):
                want, _, big = limit(0.05 * gr + 0.95 * m, torch.float32, 1 if precision else 2)
            size = 2e-3 * muon.rms_scale(rows, cols)
            ref[n] = ((1 - 2e-3 * 0.01) * ref[n].reshape(rows, cols) - size * want).reshape(ref[n].shape)
            # (the momentum's roundings are an input's, which the iteration passes on as it does the operands': 2^-22 of them are in `big`)
            lim[n] = lim[n] + size * big + 4 * 2.0 ** -24 * (ref[n].abs().max() + size * want.abs().max())
            e = (tr.view(tr.params, n).double() - ref[n]).reshape(rows, cols).abs() / lim[n]
            assert float(e.max()) <= 1, (n, it, float(e.max()))
        for p, n in zip(adam, others):
            p.grad = grads[n] * coef
        opt.step()
        for p, n in zip(adam, others):
            assert float((tr.view(tr.params, n) - p.detach()).abs().max()) < 1e-6, n
