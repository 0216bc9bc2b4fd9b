"""The workloads of the token-embedding and update-orthogonalising operators: sizes, inputs, their plain form in elementary torch
operations, what one pass has to move and compute, and the exact result in 64 bits.

A case is one call of one operator:
  embed       y = scale * W[tokens]                                                 (diffsvc_amd.tokens.embed_tokens)
  embed_grad  dW[v] = scale * sum of dy over the places of token v, v != padding   (diffsvc_amd.tokens.embed_tokens_grad)
  ortho       Newton-Schulz iteration of a batch of matrices                        (diffsvc_amd.muon.orthogonalize)
  muon        momentum, Newton-Schulz iteration and weight step, in place           (diffsvc_amd.muon.muon_step_)
"""
import math

import torch

own = False

STEPS, COEF, EPS = 5, (3.4445, -4.7750, 2.0315), 1e-7
MU, LR, WD = 0.95, 0.02, 0.01
PAD = 0
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # the energy table's lookup for one ten-second clip: 861 frames, 256 bins of 256 channels; latency counts
        dict(name="embed clip", op="embed", N=861, V=256, H=256, dtype="f32", ids="i64", spread="runs"),
        # one token of a decoding step
        dict(name="embed one token", op="embed", N=1, V=65536, H=2048, dtype="bf16", ids="i64", spread="zipf"),
        # a training batch of a model over a text-sized vocabulary
        dict(name="embed batch", op="embed", N=65536, V=50000, H=2048, dtype="bf16", ids="i32", spread="zipf"),
        # the energy table's gradient of a training batch of 64 x 128 frames: long runs of few bins
        dict(name="grad frames", op="embed_grad", N=8192, V=256, H=256, dtype="f32", ids="i64", spread="runs"),
        # the same batch as "embed batch", half as long, backwards: most rows of the table get nothing, a few get thousands
        dict(name="grad batch", op="embed_grad", N=32768, V=50000, H=2048, dtype="bf16", ids="i64", spread="zipf"),
        # odd sizes: rows that no vector width divides
        dict(name="grad odd", op="embed_grad", N=5003, V=1009, H=333, dtype="f16", ids="i32", spread="zipf"),
        # one diffusion projection of the denoiser: the smallest matrix that it trains; launches and latency count
        dict(name="ortho one", op="ortho", B=1, rows=384, cols=384, dtype="f32"),
        # the dilated convolutions of the 20 residual layers, each as a matrix of 2C x 3C
        dict(name="ortho layers", op="ortho", B=20, rows=768, cols=1152, dtype="f32"),
        # tall matrices of odd sizes
        dict(name="ortho odd", op="ortho", B=3, rows=1007, cols=301, dtype="f16"),
        # one large square matrix: the matrix cores count
        dict(name="ortho large", op="ortho", B=1, rows=4096, cols=4096, dtype="bf16"),
        # the output projections of the 20 residual layers: the whole optimisation step of one group
        dict(name="muon layers", op="muon", B=20, rows=768, cols=384, dtype="f32"),
        # one wide matrix of a larger model
        dict(name="muon wide", op="muon", B=1, rows=2048, cols=8192, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["embed", "embed_grad", "ortho", "muon"])
    dtype = rng.choice(["f32", "f16", "bf16"] if op != "muon" else ["f32", "bf16"])
    if op in ("embed", "embed_grad"):
        H = _log(rng, 1, 8192)
        N = _log(rng, 1, max(1, min(131072, (1 << 25) // H)))
        V = _log(rng, 2, max(2, min(131072, (1 << 25) // H)))
        return dict(op=op, N=N, V=V, H=H, dtype=dtype, ids=rng.choice(["i32", "i64"]), spread=rng.choice(["zipf", "runs", "even", "one"]))
    rows, cols = _log(rng, 1, 4096), _log(rng, 1, 4096)
    return dict(op=op, B=max(1, min(_log(rng, 1, 24), (1 << 33) // (min(rows, cols) ** 2 * max(rows, cols)))), rows=rows, cols=cols, dtype=dtype)


def _tokens(case, g, dev):
    """zipf: text; runs: a quantised contour that moves slowly, with padding behind each 128 frames; even: any; one: a single token."""
    N, V = case["N"], case["V"]
    if case["spread"] == "zipf":
        u = torch.rand(N, generator=g, device=dev, dtype=torch.float64)
        t = torch.exp(u * math.log(V)).long() - 1
        t = (t * 7919 + 13) % V if V % 7919 else t
    elif case["spread"] == "runs":
        walk = torch.cumsum(torch.randn(N, generator=g, device=dev), 0)
        t = (V * (0.5 + 0.4 * torch.sin(walk * 0.1))).long()
        at = torch.arange(N, device=dev)
        t = torch.where(at % 128 >= 100 + (at // 128 * 5) % 28, torch.zeros_like(t), t)
    elif case["spread"] == "one":
        t = torch.full((N,), min(V - 1, 1 + int(torch.randint(0, V, (1,), generator=g, device=dev))), device=dev)
    else:
        t = torch.randint(0, V, (N,), generator=g, device=dev)
    return t.clamp_(0, V - 1).to(torch.int32 if case["ids"] == "i32" else torch.int64)


def _updates(case, g, dev, size):
    """Gradients of a matrix: a signal of a few directions and noise of about its size."""
    B, r, c = case["B"], case["rows"], case["cols"]
    k = max(1, min(r, c) // 16)
    u = torch.randn(B, r, k, generator=g, device=dev)
    v = torch.randn(B, k, c, generator=g, device=dev)
    return (u @ v / math.sqrt(k) + torch.randn(B, r, c, generator=g, device=dev)) * size


def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    s = dict(case=case)
    if case["op"] in ("embed", "embed_grad"):
        N, V, H = case["N"], case["V"], case["H"]
        s["tokens"] = _tokens(case, g, dev)
        s["scale"] = math.sqrt(H)
        if case["op"] == "embed":
            s["table"] = (torch.randn(V, H, generator=g, device=dev) / math.sqrt(H)).to(dt)
        else:
            s["dy"] = (torch.randn(N, H, generator=g, device=dev) * 1e-3).to(dt)
    elif case["op"] == "ortho":
        s["update"] = _updates(case, g, dev, 1e-4).to(dt)
    else:
        s["grad"] = _updates(case, g, dev, 1e-4).to(dt)
        s["momentum"] = _updates(case, g, dev, 3e-5)
        s["param"] = (torch.randn(case["B"], case["rows"], case["cols"], generator=g, device=dev) / math.sqrt(case["cols"])).to(dt)
    return s


def _rms(case):
    """The size of an update whose elements have the root mean square of an AdamW step's."""
    return 0.2 * math.sqrt(max(case["rows"], case["cols"]))


def _embed(s):
    return (s["table"][s["tokens"].long()].float() * s["scale"]).to(s["table"].dtype)


def _embed_grad(s):
    t = s["tokens"].long()
    d = s["dy"].float() * s["scale"] * (t != PAD)[:, None]
    w = torch.zeros(s["case"]["V"], s["case"]["H"], device=d.device)
    return w.index_add_(0, t, d).to(s["dy"].dtype)


def _ortho(u):
    x = u.float()
    tall = x.shape[1] > x.shape[2]
    if tall:
        x = x.transpose(1, 2).contiguous()
    norm = x.double().square().sum((1, 2), keepdim=True).sqrt()
    x = (x / (norm + EPS)).float()
    a, b, c = COEF
    for _ in range(STEPS):
        gram = torch.bmm(x, x.transpose(1, 2).contiguous())
        x = a * x + torch.bmm(b * gram + c * torch.bmm(gram, gram), x)
    return x.transpose(1, 2).contiguous() if tall else x


def _muon(s):
    p, m, g = s["param"], s["momentum"], s["grad"].float()
    m.mul_(MU).add_(g, alpha=1 - MU)
    u = (1 - MU) * g + MU * m
    p.copy_((1 - LR * WD) * p.float() - LR * _rms(s["case"]) * _ortho(u))
    return {"param": p, "momentum": m}


def run(state):
    s, op = state, state["case"]["op"]
    if own:
        from diffsvc_amd import muon, tokens
        if op == "embed":
            return tokens.embed_tokens(s["tokens"], s["table"], scale=s["scale"], padding_idx=PAD)
        if op == "embed_grad":
            return tokens.embed_tokens_grad(s["tokens"], s["dy"], s["case"]["V"], scale=s["scale"], padding_idx=PAD)
        if op == "ortho":
            return muon.orthogonalize(s["update"], steps=STEPS, coefficients=COEF, eps=EPS)
        muon.muon_step_(s["param"], s["grad"], s["momentum"], lr=LR, momentum=MU, nesterov=True, weight_decay=WD, scale=_rms(s["case"]),
                        steps=STEPS, coefficients=COEF, eps=EPS)
        return {"param": s["param"], "momentum": s["momentum"]}
    if op == "embed":
        return _embed(s)
    if op == "embed_grad":
        return _embed_grad(s)
    if op == "ortho":
        return _ortho(s["update"]).to(s["update"].dtype)
    return _muon(s)


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] in ("embed", "embed_grad"):
        N, V, H = case["N"], case["V"], case["H"]
        ids = N * (4 if case["ids"] == "i32" else 8)
        if case["op"] == "embed":       # the rows that are looked up, once each, and the output
            return {"bytes": ids + (min(N, V) + N) * H * size, "flops": N * H}
        return {"bytes": ids + (N + V) * H * size, "flops": N * H}
    B, m, n = case["B"], min(case["rows"], case["cols"]), max(case["rows"], case["cols"])
    # the two products with a symmetric result count half
    flops = B * STEPS * (m * m * n + m * m * m + 2 * m * m * n)
    if case["op"] == "ortho":
        return {"bytes": B * m * n * 2 * size, "flops": flops}
    return {"bytes": B * m * n * (3 * size + 8), "flops": flops}


def _exact_ortho(u):
    """Every iterate is P X0 with P a polynomial of the first Gram matrix: the recursion runs on matrices of the short side alone."""
    tall = u.shape[1] > u.shape[2]
    x = u.transpose(1, 2).contiguous() if tall else u
    x = x / (torch.linalg.vector_norm(x, dim=(1, 2), keepdim=True) + EPS)
    gram = torch.bmm(x, x.transpose(1, 2).contiguous())
    eye = torch.eye(x.shape[1], dtype=x.dtype, device=x.device).expand_as(gram)
    poly = eye
    for _ in range(STEPS):
        step = COEF[0] * eye + torch.bmm(COEF[1] * eye + COEF[2] * gram, gram)
        poly = torch.bmm(step, poly)
        gram = torch.bmm(torch.bmm(step, gram), step)
    x = torch.bmm(poly, x)
    return x.transpose(1, 2) if tall else x


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "embed":
        return torch.index_select(s["table"].double(), 0, s["tokens"].long()) * s["scale"]
    if case["op"] == "embed_grad":
        # sums of neighbours after sorting, from the differences of a running sum
        t, order = torch.sort(s["tokens"].long())
        run_sum = torch.cumsum(s["dy"].double()[order], 0)
        v = torch.arange(case["V"], device=t.device)
        ends, starts = torch.searchsorted(t, v, right=True), torch.searchsorted(t, v)
        run_sum = torch.cat([torch.zeros_like(run_sum[:1]), run_sum])
        w = (run_sum[ends] - run_sum[starts]) * s["scale"]
        w[PAD] = 0
        return w
    if case["op"] == "ortho":
        return _exact_ortho(s["update"].double())
    g, m, p = s["grad"].double(), s["momentum"].double(), s["param"].double()
    m = MU * m + (1 - MU) * g
    u = (1 - MU) * g + MU * m
    return {"param": (1 - LR * WD) * p - LR * _rms(case) * _exact_ortho(u), "momentum": m}
