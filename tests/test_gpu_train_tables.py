"""GPU: what the training step has beside its own tensors -- the energy table (``use_energy_embed``: lookup, d loss / d cond, gradient by sorted
tokens) and orthogonalised updates of the inner matrices (``matrix_optimizer: muon``) -- against torch autograd on the oracle and the
formulas in float64; both together in a training loop."""
import numpy as np
import pytest
import torch
import torch.nn.functional as F

import dsvc_oracle as O
from diffsvc_amd import muon, synth
from diffsvc_amd.train import ENERGY, DiffusionTrainerHip, muon_groups
from test_gpu_train import _batch

ARCHS = {"tiny": (synth.tiny_hparams(K=50), [0, 1, 2], 40, 23, 5), "44k": (synth.HPARAMS_44K, [4, 9], 64, 37, 6), "24k": (synth.HPARAMS_24K, [1, 2, 3], 51, 29, 7)}


def setup(arch, seed=11, **more):
    hp, clips, T, units, s = ARCHS[arch]
    hp = dict(hp, diff_loss_type="l2", use_energy_embed=True, **more)
    sd = dict(synth.acoustic_state(hp, 3))
    g = torch.Generator().manual_seed(seed)
    sd[ENERGY] = torch.randn(256, hp["hidden_size"], generator=g) * hp["hidden_size"] ** -0.5
    sd[ENERGY][0] = 0
    hub, m2p, f0, mels, t = _batch(hp, clips, T, units, s)
    m2p[0, T - 5:] = 0
    energy = torch.rand(len(clips), T, generator=g) * 4.4                  # some at and above the last bin, some in bin 0 (the padding row)
    energy[:, ::7] = 0.01
    return hp, sd, clips, (hub, m2p, f0, mels, t), energy, s


def reference(hp, sd, clips, batch, energy, seed):
    """Loss and gradients of every trained tensor by autograd (the oracle's own path, with the energy table in it)."""
    hub, m2p, f0, mels, t = batch
    names = [k for k in sd if k.startswith("denoise_fn.")] + ["fs2.pitch_embed.weight", ENERGY]
    p = dict(sd)
    for k in names:
        p[k] = sd[k].detach().clone().requires_grad_(True)
    cond, _, _ = O.build_cond(p, hub, m2p, f0.clone(), hp, energy=energy)
    noise = O.ddpm_noise_ref_layout(seed, clips, 0, mels.shape[1], hp["audio_num_mel_bins"], O.PURPOSE_TRAIN_NOISE)
    x0 = O.norm_spec(sd, mels).transpose(1, 2)[:, None, :, :]
    loss = O.p_losses(p, x0, t, cond.transpose(1, 2), noise, hp["dilation_cycle_length"], "l2")
    grads = torch.autograd.grad(loss, [p[k] for k in names] + [cond])
    ref = dict(zip(names, grads))
    ref[ENERGY][0] = 0                                                    # nn.Embedding's padding_idx (fs2.py:81-82)
    return loss.detach(), ref, grads[-1]


def rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm().clamp_min(1e-300))


def cuda(batch):
    return [v.cuda() for v in batch]


@pytest.mark.gpu
@pytest.mark.parametrize("arch", ["tiny", "44k", "24k"])
def test_energy_table_gradient_vs_autograd(arch):
    """Every gradient, the energy table's and d loss / d cond included, within 5e-5 of autograd's: the tolerance of the step's other gradients --
    three fp16 products per product (2^-22 each) through 20 layers."""
    hp, sd, clips, batch, energy, seed = setup(arch)
    ref_loss, ref, ref_cond = reference(hp, sd, clips, batch, energy, seed)
    tr = DiffusionTrainerHip(hp, sd)
    hub, m2p, f0, mels, t = cuda(batch)
    ids = torch.tensor(clips, dtype=torch.int32, device="cuda")
    loss = tr.forward_backward(hub, m2p, f0, mels, t, seed=seed, clip_ids=ids, energy=energy.cuda())
    assert abs(loss.item() - ref_loss.item()) <= 1e-5 * max(1.0, abs(ref_loss.item()))
    for name, _, _ in tr.layout:
        got = tr.view(tr.grads, name).cpu()
        assert rel(got, ref[name]) < 5e-5 if ref[name].any() else not got.any(), (name, rel(got, ref[name]))
    assert not tr.view(tr.grads, ENERGY)[0].any() and set(tr.state_dict()) == set(sd)
    # d loss / d cond itself; frames whose gradient the mask drops are part of it
    ret = tr.fs2(hub, m2p, None, None, f0.clone(), None, energy.cuda(), infer=True)
    out = torch.full((len(clips), mels.shape[1], hp["hidden_size"]), float("nan"), device="cuda")
    again = tr.h.step(mels, ret["decoder_inp"].transpose(1, 2), t, pitch=ret["pitch_pred"].squeeze(-1), mel2ph=m2p, seed=seed, clip_ids=ids, cond_grad=out)
    # (the loss is a float atomic sum of the blocks' parts: its last bits depend on their order, 2^-24 per addition of a part)
    assert abs(again.item() - loss.item()) <= 1e-6 * loss.item() and rel(out.cpu(), ref_cond) < 5e-5
    # the phases leave the same behind, and the buckets (the energy table's behind the handle's own) cover the flat buffer
    out2 = torch.full_like(out, float("nan"))
    L = hp["residual_layers"]
    tr.h.step_begin(mels, ret["decoder_inp"].transpose(1, 2), t, pitch=ret["pitch_pred"].squeeze(-1), mel2ph=m2p, seed=seed, clip_ids=ids, cond_grad=out2)
    with pytest.raises(RuntimeError, match="in flight"):
        tr.h._want_cond_grad(out, mels)
    tr.h.step_layers(L, L // 2)
    tr.h.step_layers(L // 2, 0)
    tr.h.step_end()
    assert rel(out2, out) < 1e-6


@pytest.mark.gpu
def test_cond_grad_is_bounded_by_its_rows_and_off_by_default():
    hp, sd, clips, batch, energy, seed = setup("tiny")
    tr = DiffusionTrainerHip(dict(hp, use_energy_embed=False), sd)
    hub, m2p, f0, mels, t = cuda(batch)
    assert tr.n_floats == tr.h.n_floats and torch.equal(tr.state_dict()[ENERGY], sd[ENERGY])
    loss = tr.forward_backward(hub, m2p, f0, mels, t, seed=seed)
    grads = tr.grads.clone()
    B, T = mels.shape[:2]
    buf = torch.full((B * T + 1, hp["hidden_size"]), 3.0, device="cuda")
    check = tr.h._ck
    check(tr.h._L.dsvc_trainer_set_cond_grad(tr.h._h, buf.data_ptr(), B * T - 1))
    with pytest.raises(RuntimeError, match="rows"):
        tr.forward_backward(hub, m2p, f0, mels, t, seed=seed)
    assert bool((buf == 3).all())
    check(tr.h._L.dsvc_trainer_set_cond_grad(tr.h._h, buf.data_ptr(), B * T))
    tr.forward_backward(hub, m2p, f0, mels, t, seed=seed)
    assert bool((buf[B * T:] == 3).all()) and not bool((buf[:B * T] == 3).any())
    check(tr.h._L.dsvc_trainer_set_cond_grad(tr.h._h, None, 0))
    buf.fill_(3.0)
    assert abs(tr.forward_backward(hub, m2p, f0, mels, t, seed=seed).item() - loss.item()) <= 1e-6 * loss.item() and bool((buf == 3).all())
    assert rel(tr.grads, grads) < 1e-6                                    # (bias gradients are float atomics)
    with pytest.raises(ValueError, match="cond_grad"):
        tr.h.step(mels, torch.zeros(B, hp["hidden_size"], T, device="cuda"), t, cond_grad=buf)
    with pytest.raises(ValueError, match="matrix_optimizer"):
        DiffusionTrainerHip(dict(hp, matrix_optimizer="sgd"), sd)


@pytest.mark.gpu
def test_energy_table_through_the_drop_in_module():
    """loss.backward() of GaussianDiffusionHip.forward(infer=False) fills the energy table's .grad as the flat trainer does; inference carries no
    graph; a frame energy below zero has no row (check_alignment)."""
    from diffsvc_amd.denoiser import DiffNetHip
    from diffsvc_amd.sampler import GaussianDiffusionHip
    hp, sd, clips, batch, energy, seed = setup("tiny")
    M = hp["audio_num_mel_bins"]
    model = GaussianDiffusionHip(None, M, DiffNetHip(M, hparams=hp), timesteps=50, K_step=50, loss_type="l2", spec_min=hp["spec_min"],
                                 spec_max=hp["spec_max"], hparams=hp)
    model.load_state_dict(sd, strict=True)
    model.cuda()
    hub, m2p, f0, mels, t = cuda(batch)
    loss = model(hub, mel2ph=m2p, ref_mels=mels, f0=f0.clone(), energy=energy.cuda(), infer=False, t=t, seed=7)["diff_loss"]
    (2.0 * loss).backward()
    tr = DiffusionTrainerHip(hp, sd)
    want = tr.forward_backward(hub, m2p, f0.clone(), mels, t, seed=7, energy=energy.cuda())
    assert abs(loss.item() - want.item()) <= 1e-6 * abs(want.item())
    named = dict(model.named_parameters())
    for name, _, _ in tr.layout:
        assert rel(named[name].grad, 2.0 * tr.view(tr.grads, name)) < 1e-6, name
    ret = model.fs2(hub, mel2ph=m2p, f0=f0.clone(), energy=energy.cuda(), infer=True)
    assert not ret["decoder_inp"].requires_grad and not ret["cond_bht"].requires_grad
    model.fs2.check_alignment()
    model.fs2(hub, mel2ph=m2p, f0=f0.clone(), energy=energy.cuda() - 1, infer=True)
    with pytest.raises(IndexError):
        model.fs2.check_alignment()


def newton_schulz(g, steps=5):
    a, b, c = muon.COEFFICIENTS
    x = g.double()
    tall = x.shape[0] > x.shape[1]
    x = x.t() if tall else x
    x = x / (x.norm() + 1e-7)
    for _ in range(steps):
        A = x @ x.t()
        x = a * x + (b * A + c * A @ A) @ x
    return x.t() if tall else x


@pytest.mark.gpu
@pytest.mark.parametrize("precision", [None, "f16"])
def test_muon_optimizer_step_vs_formulas(precision):
    """Two optimisation steps on given gradients: the inner matrices against momentum + Newton-Schulz in float64, everything else against
    torch.optim.AdamW, the gradient-norm clip in front of both.  Tolerance of the matrices: an element of the orthogonalised update is off by a few
    1e-6 (split operands) or 1e-3 (single fp16 operands) of its root mean square (tests/test_gpu_muon.py holds the operator itself to its model);
    4 and 40 half steps of fp16 / split fp16 per step times the size of a step, six standard deviations."""
    hp, sd, clips, batch, energy, seed = setup("24k", lr=1e-3, weight_decay=0.01, clip_grad_norm=1.0, matrix_optimizer="muon", muon_lr=2e-3,
                                               muon_precision=precision)
    tr = DiffusionTrainerHip(hp, sd)
    groups, rest = muon_groups(tr.layout, tr.shapes)
    inner = {}
    for off, batch_, stride, rows, cols in groups:
        for i in range(batch_):
            name = next(n for n, o, m in tr.layout if o == off + i * stride)
            inner[name] = (rows, cols)
    others = [n for n, _, _ in tr.layout if n not in inner]
    assert ENERGY in others and "fs2.pitch_embed.weight" in others and "denoise_fn.residual_layers.3.dilated_conv.weight" in inner
    ref = {n: sd[n].double().clone() for n, _, _ in tr.layout}
    mom = {n: torch.zeros_like(ref[n]) for n in inner}
    adam = [torch.nn.Parameter(sd[n].clone()) for n in others]
    opt = torch.optim.AdamW(adam, lr=hp["lr"], betas=(0.9, 0.98), weight_decay=0.01)
    g = torch.Generator().manual_seed(4)
    tol = {None: 40 * 2.0 ** -22, "f16": 4 * 2.0 ** -11}[precision]
    for it in range(2):
        grads = {n: torch.randn(sd[n].shape, generator=g) * 0.02 for n, _, _ in tr.layout}
        for n in grads:
            tr.view(tr.grads, n).copy_(grads[n])
        norm = torch.stack([v.double().square().sum() for v in grads.values()]).sum().sqrt()
        coef = min(1.0, float(1.0 / (norm + 1e-6)))
        assert coef < 1
        tr.optimizer_step()
        for n, (rows, cols) in inner.items():
            gr = grads[n].double().reshape(rows, cols) * coef
            m = mom[n].reshape(rows, cols).mul_(0.95).add_(gr, alpha=0.05)
            step = 2e-3 * muon.rms_scale(rows, cols) * newton_schulz(0.05 * gr + 0.95 * m)
            ref[n] = ((1 - 2e-3 * 0.01) * ref[n].reshape(rows, cols) - step).reshape(ref[n].shape)
            e = tr.view(tr.params, n).cpu().double() - ref[n]
            lim = (it + 1) * (6 * tol * step.square().mean().sqrt() + 4 * 2.0 ** -24 * ref[n].abs().max())
            assert float(e.abs().max()) <= float(lim), (n, it, float(e.abs().max()), float(lim))
        for p, n in zip(adam, others):
            p.grad = grads[n] * coef
        opt.step()
        for p, n in zip(adam, others):
            assert float((tr.view(tr.params, n).cpu() - p.detach()).abs().max()) < 1e-6, n


@pytest.mark.gpu
def test_energy_table_and_muon_together_in_a_training_loop():
    """The whole step as a user runs it, twice from the same state: finite, every trained tensor moves by about its optimizer's step, untouched rows
    of the tables stay, both runs agree (float atomics of the bias gradients aside)."""
    hp, sd, clips, batch, energy, seed = setup("24k", lr=1e-3, weight_decay=0.0, matrix_optimizer="muon")
    hub, m2p, f0, mels, t = cuda(batch)
    runs = []
    for _ in range(2):
        tr = DiffusionTrainerHip(hp, sd)
        for it in range(3):
            loss = tr.train_step(hub, m2p, f0.clone(), mels, t=t, seed=seed + it, energy=energy.cuda())
            assert torch.isfinite(loss).all() and torch.isfinite(tr.params).all()
        runs.append(tr.params.clone())
    assert rel(runs[0], runs[1]) < 1e-3
    used = torch.unique(tr.fs2.energy_tokens(energy)[batch[1] > 0])
    idle = torch.ones(256, dtype=torch.bool)
    idle[used] = False
    idle[0] = True
    new = tr.state_dict()
    assert torch.equal(new[ENERGY][idle], sd[ENERGY][idle]) and bool((new[ENERGY][~idle] != sd[ENERGY][~idle]).any(1).all())
    for off, b, stride, rows, cols in muon_groups(tr.layout, tr.shapes)[0]:
        n = next(n for n, o, _ in tr.layout if o == off)
        moved = float((new[n] - sd[n]).double().square().mean().sqrt())
        # a step of rank k has k singular values of 0.5 ... 1.3 (the rest stay near zero), so its elements have the root mean square
        # 0.2 sqrt(max) * sqrt(k / (rows cols)) * (0.5 ... 1.3) = 0.2 sqrt(k / min) * (0.5 ... 1.3).  The gradient of what the step embedding
        # feeds (mlp, diffusion_projection) is a sum of one outer product per clip: k is 3 there, and 1 at least anywhere
        assert 0.2 * 0.5 * hp["lr"] / min(rows, cols) ** 0.5 < moved < 3 * 0.2 * 1.3 * hp["lr"], (n, moved)


def test_muon_groups_cover_the_flat_layout():
    """CPU: every float of the flat buffer belongs to one group of one optimizer."""
    hp = dict(synth.HPARAMS_44K, use_energy_embed=True)
    sd = dict(synth.acoustic_state(hp, 3))
    sd[ENERGY] = torch.zeros(256, hp["hidden_size"])
    q = ["denoise_fn.input_projection", "denoise_fn.mlp.0", "denoise_fn.mlp.2"]
    for l in range(hp["residual_layers"]):
        q += ["denoise_fn.residual_layers.%d.%s" % (l, n) for n in ("dilated_conv", "diffusion_projection", "conditioner_projection", "output_projection")]
    q += ["denoise_fn.skip_projection", "denoise_fn.output_projection"]
    names = [n + s for n in q for s in (".weight", ".bias")] + ["fs2.pitch_embed.weight", ENERGY]
    layout, off = [], 0
    for n in names:
        layout.append((n, off, sd[n].numel()))
        off += sd[n].numel()
    groups, rest = muon_groups(layout, {n: tuple(sd[n].shape) for n in names})
    seen = torch.zeros(off, dtype=torch.int8)
    for o, b, stride, rows, cols in groups:
        for i in range(b):
            seen[o + i * stride:o + i * stride + rows * cols] += 1
    for o, n, parts, stride in rest:
        for i in range(parts):
            seen[o + i * stride:o + i * stride + n] += 1
    assert bool((seen == 1).all())
    assert len(groups) == 4 + 3 and len(rest) == 4 + 4 and sorted((b, r, c) for _, b, _, r, c in groups)[-1] == (20, 768, 1152)
    assert rest[3][0] + rest[3][1] == off                                 # the last piece runs from the skip projection's bias through both tables
