"""GPU: every way in which csrc/ortho.hip cuts a product -- tiles of 64, 128 (by four or eight waves) and 256, in one piece, in slices along K, or some
of each in one launch, for the symmetric and the full products, on one and two planes -- against the formula in float64 on the device.  Tolerances as in
test_gpu_muon.py.  ``cut`` restates the rule of the source; that every kind of cut it can give is among the cases is checked on the CPU."""
import pytest
import torch

from diffsvc_amd import muon as M
from test_gpu_muon import limit, update

K_STEPS = {(1, 64): 4, (2, 64): 2, (1, 128): 4, (2, 128): 1, (1, "alone"): 8, (2, "alone"): 4, (1, 256): 4}        # 16-wide k steps of a stage
PER_CU = {64: 2, 128: 2, "alone": 1, 256: 1}


def cut(planes, sym, batch, mi, nj, k16):
    t = mi // 128
    tiles = batch * (t * (t + 1) // 2 if sym else t * (nj // 128))
    if planes == 1 and not sym and mi % 256 == 0 and nj % 256 == 0 and tiles >= 1024:
        kind = 256
    else:
        kind = 128 if tiles > 256 else "alone" if tiles >= 192 else 64
    size = 128 if kind == "alone" else kind
    n = mi // size
    total, slots = batch * (n * (n + 1) // 2 if sym else n * (nj // size)), 256 * PER_CU[kind]
    rest = total % slots
    slices = min(slots // rest, k16 // K_STEPS[planes, kind] // 16, 16) if rest else 1
    return kind, "whole" if slices <= 1 else "both" if total > rest else "sliced"


def cuts(planes, shape):
    *b, r, c = shape
    batch, m, n = (b or [1])[0], min(r, c), max(r, c)
    if m <= 64 and (32 if m <= 32 else 64) * n <= 16384:
        return set()                                                       # one workgroup
    m, n = (m + 127) // 128 * 128, (n + 127) // 128 * 128
    return {(planes, "gram", *cut(planes, True, batch, m, m, n // 16)), (planes, "poly", *cut(planes, True, batch, m, m, m // 16)),
            (planes, "full", *cut(planes, False, batch, m, n, m // 16))}


ONE = [(100, 100), (120, 2040), (24570, 127), (20, 128, 1660), (64, 380, 380), (64, 250, 256), (2048, 2048), (3, 1150, 2040), (8, 1400, 2040), (2, 2040, 2170),
       (4, 2047, 2047), (256, 65530), (2045, 8440)]
TWO = [(3, 100, 101), (120, 1020), (24570, 127), (20, 128, 1660), (64, 380, 380), (64, 250, 256), (1024, 1024), (1020, 2176), (5, 890, 1024), (4, 1020, 1024),
       (5, 510, 3328), (64, 510, 510), (20, 768, 1152)]
STEPS = [((2048, 8448), torch.bfloat16, "f16"), ((8, 1400, 2040), torch.bfloat16, "f16"), ((20, 768, 1152), torch.float32, None), ((20, 1152, 768), torch.bfloat16, None),
         ((24571, 127), torch.float16, None), ((5, 510, 3328), torch.bfloat16, None)]


def check(got, x, dtype, planes, **kw):
    for a, b in zip(got.reshape(-1, *got.shape[-2:]), x.reshape(-1, *x.shape[-2:])):
        with torch.device("cuda"):
            want, two, big = limit(b, dtype, planes, **kw)
        e = a.double() - want
        assert torch.isfinite(e).all()
        f, m = float(e.square().sum().sqrt() / two), float((e.abs() / big).max())
        assert f <= 1 and m <= 1, (f, m)


@pytest.mark.gpu
@pytest.mark.parametrize("shape, planes, dtype", [(s, 1, t) for s, t in zip(ONE, (torch.float32, torch.bfloat16) * 7)] + [(s, 2, t) for s, t in zip(TWO, (torch.float32, torch.float16) * 7)])
def test_products_in_every_cut(shape, planes, dtype):
    x = update(shape, 5).to(dtype).cuda()
    run = lambda: M.orthogonalize(x, precision="f16" if planes == 1 else None)
    got = run()
    check(got, x, dtype, planes)
    assert torch.equal(got, run())                                         # slices are added up in their order, whoever comes last


@pytest.mark.gpu
@pytest.mark.parametrize("shape, dtype, precision", STEPS)
def test_steps_in_the_large_cuts(shape, dtype, precision):
    """The weight step in the last product's epilogue: with a weight of zero, the new weight is the orthogonalised momentum."""
    g = update(shape, 6).to(dtype).cuda()
    p, m = torch.zeros_like(g), torch.zeros(shape, device="cuda")
    M.muon_step_(p, g, m, lr=1.0, momentum=0.5, nesterov=False, weight_decay=0.25, precision=precision)
    check(-p, m, dtype, 1 if precision == "f16" else 2)
    # a weight: (1 - lr wd) w - lr O, each rounded once
    w = update(shape, 7, 1.0).to(dtype).cuda()
    q, m = w.clone(), torch.zeros(shape, device="cuda")
    M.muon_step_(q, g, m, lr=0.5, momentum=0.5, nesterov=False, weight_decay=0.25, precision=precision)
    half = torch.finfo(dtype).eps / 2
    want = 0.875 * w.double() + 0.5 * p.double()
    # |p + O| is half a step of p, lr times that remains; q is rounded once; the two float32 operations take 2^-24 of their terms each
    lim = half * want.abs() + 0.5 * half * (1 + 2.0 ** -7) * p.double().abs() + 2.0 ** -23 * (w.double().abs() + p.double().abs()) + torch.finfo(dtype).tiny
    assert bool(((q.double() - want).abs() <= lim).all())


def test_the_cases_hold_every_cut():
    have = set().union(*(cuts(1, s) for s in ONE), *(cuts(2, s) for s in TWO))
    can = set()
    for planes in (1, 2):
        for b in (1, 2, 3, 4, 5, 6, 8, 12, 16, 20, 24, 32, 64):
            for m in range(128, 2561, 128):
                for n in (m, *range(m + 128, 2561, 256), 3328, 4096, 8192, 8448, 16384, 24576, 65536):
                    can |= cuts(planes, (b, m, n))
    assert can <= have, can - have
    assert len(have) == 35
    steps = set().union(*(cuts(1 if q == "f16" else 2, s) for s, _, q in STEPS))
    assert {(1, "full", 256, "both"), (2, "full", 128, "both"), (2, "full", "alone", "whole"), (1, "full", 128, "whole")} <= steps, steps
