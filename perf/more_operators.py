"""Cases that measure the two ends of a recovery pass: the loss at the LM head with
its gradients, and the masked, orthogonalised step of a pruned weight.

`run` computes a case with elementary torch operations in FP32 (own = False) or
through the C ABI (own = True); both take what `prepare` made.

loss         z = h W^T, capped by c tanh(z / c) where a cap is given; lse = log sum exp z and
             loss = lse - z[target] for each token; a target outside the vocabulary leaves the
             token out: zeros, whatever its values
loss's gradients   of sum dloss * loss + dlse * lse: dh and dW
orthogonalise      X = U / (|U| + eps); five times X <- (a I + b A + c A^2) X with A = X X^T, on
             the shorter side
step         m <- mask (beta m + g), U = mask (g + beta m), W <- mask ((1 - lr wd) W - lr s O(U))
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
CODE = {"f32": 0, "bf16": 2}
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS, EPS = 5, 1e-7
BETA, LR, DECAY = 0.95, 0.002, 0.1

#: No case costs more than the largest listed one: n d V of the loss alone and with gradients, the step's k^2 D.
MAX_LOSS, MAX_GRADS, MAX_STEP = 8000 * 4096 * 128000, 4001 * 8192 * 128000, 8192 * 8192 * 28672


def listed():
    return [
        # The next token of one evaluated request: launch latency and one pass over the head.
        dict(name="loss: one token", op="loss", n=1, d=4096, vocab=32000, left=0.0, cap=0.0),
        # A batch of calibration text at the 32000-entry head.
        dict(name="loss: calibration batch", op="loss", n=2048, d=4096, vocab=32000, left=0.0, cap=0.0),
        # Perplexity over a long batch with a large vocabulary, prompts left out, capped logits.
        dict(name="loss: large vocabulary", op="loss", n=8000, d=4096, vocab=128000, left=0.25, cap=30.0),
        # One short sample's loss and gradients.
        dict(name="gradients: short sample", op="grads", n=37, d=4096, vocab=32000, left=0.0, cap=0.0, dlse=False),
        # A batch of recovery training, prompts left out, with a penalty on lse.
        dict(name="gradients: batch", op="grads", n=2048, d=4096, vocab=32000, left=0.25, cap=0.0, dlse=True),
        # The 8192-wide model with a large vocabulary, an odd number of tokens.
        dict(name="gradients: 8192 wide", op="grads", n=4001, d=8192, vocab=128000, left=0.0, cap=30.0, dlse=False),
        # The 128 x 128 mock tensor's gradient.
        dict(name="orthogonalise: mock", op="ortho", r=128, d=128, g="f32"),
        # A k_proj's gradient.
        dict(name="orthogonalise: k_proj", op="ortho", r=1024, d=4096, g="bf16"),
        # A gate_proj's, which is tall.
        dict(name="orthogonalise: gate_proj", op="ortho", r=14336, d=4096, g="bf16"),
        # The step of the 128 x 128 mock tensor under its 2:4 mask.
        dict(name="step: mock", op="step", r=128, d=128, g="f32", w="f32", m=4),
        # A pruned q_proj in FP32, as the pruning pass leaves it.
        dict(name="step: q_proj", op="step", r=4096, d=4096, g="bf16", w="f32", m=4),
        # The 8192-wide model's down_proj in BF16, 4:8.
        dict(name="step: 28672 wide", op="step", r=8192, d=28672, g="bf16", w="bf16", m=8),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["loss", "grads", "ortho", "step"])
    if op in ("loss", "grads"):
        d, vocab = _log(rng, 64, 8192), _log(rng, 128, 128000)
        most = (MAX_LOSS if op == "loss" else MAX_GRADS) / (d * vocab)
        case = dict(op=op, n=_log(rng, 1, max(1, min(8192, int(most)))), d=d, vocab=vocab, left=rng.choice([0.0, 0.0, 0.25, 0.7]),
                    cap=rng.choice([0.0, 0.0, 30.0]))
        return dict(case, dlse=rng.random() < 0.5) if op == "grads" else case
    short = _log(rng, 1, 8192)
    long = _log(rng, short, max(short, min(28672, int(MAX_STEP / (short * short)))))
    r, d = (short, long) if rng.random() < 0.5 else (long, short)
    case = dict(op=op, r=r, d=d, g=rng.choice(["f32", "bf16"]))
    return case if op == "ortho" else dict(case, w=rng.choice(["f32", "bf16"]), m=rng.choice([m for m in (0, 4, 4, 8) if not m or r * d % m == 0]))


# ---- inputs ---------------------------------------------------------------------
def _up(v, m):
    return (v + m - 1) // m * m


def _rows(n, d, dtype):
    """[n][d] in rows of a stride that is a multiple of 16."""
    return torch.zeros(max(1, n), _up(d, 16), device="cuda", dtype=dtype)[:n, :d]


def _gradient(g, r, d):
    """What a batch's gradient looks like: some strong directions, falling off, above noise."""
    k = max(1, min(64, r, d))
    fall = torch.arange(1, k + 1, device="cuda").float() ** -0.5
    G = (torch.randn(r, k, device="cuda", generator=g) * fall) @ torch.randn(k, d, device="cuda", generator=g)
    return G.add_(torch.randn(r, d, device="cuda", generator=g), alpha=0.3).mul_(1e-3)


def _mask(w, m):
    """Half of each m weights in a row of memory kept, the larger ones: (bytes, truth values)."""
    groups = w.reshape(-1, m).abs()
    keep = torch.zeros(groups.shape, device="cuda", dtype=torch.bool)
    keep.scatter_(1, groups.topk(m // 2, dim=1).indices, True)
    bits = (keep * (2 ** torch.arange(m, device="cuda"))).sum(1)
    return bits.to(torch.uint8), keep.view(w.shape)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = dict(case)
    if case["op"] in ("loss", "grads"):
        n, d, vocab = case["n"], case["d"], case["vocab"]
        s["w"] = _rows(vocab, d, torch.bfloat16)
        s["w"].copy_(torch.randn(vocab, d, device="cuda", generator=g).mul_(0.02).add_(torch.randn(d, device="cuda", generator=g), alpha=0.005))
        s["target"] = torch.randint(0, vocab, (n,), device="cuda", generator=g)
        # tokens from certain ones to ones that say nothing about the next
        toward = s["w"][s["target"]].float()
        toward /= toward.norm(dim=1, keepdim=True).clamp_min(1e-6)
        sure = 10 * torch.rand(n, 1, device="cuda", generator=g)
        s["h"] = _rows(n, d, torch.bfloat16)
        s["h"].copy_(torch.randn(n, d, device="cuda", generator=g) + sure * toward)
        out = int(n * case["left"])
        s["target"][torch.randperm(n, device="cuda", generator=g)[:out]] = -100
        if case["op"] == "grads":
            s["dloss"] = torch.full((n,), 1.0 / max(1, n - out), device="cuda")
            s["dlse"] = 1e-3 * s["dloss"] * (1 + torch.rand(n, device="cuda", generator=g)) if case["dlse"] else None
        return s
    r, d = case["r"], case["d"]
    s["grad"] = _rows(r, d, DTYPES[case["g"]])
    s["grad"].copy_(_gradient(g, r, d))
    if case["op"] == "step":
        w = torch.randn(r, d, device="cuda", generator=g).mul_(0.02)
        s["keep"] = s["mask"] = None
        if case["m"]:
            s["mask"], s["keep"] = _mask(w, case["m"])
            w.mul_(s["keep"])
        s["momentum"] = _gradient(g, r, d).mul_(5)
        s["weights"] = w.to(DTYPES[case["w"]])
    return s


# ---- the plain forms --------------------------------------------------------------
def _loss(s, grads):
    kept = (s["target"] >= 0) & (s["target"] < s["vocab"])
    zero = torch.zeros((), device="cuda")
    h, w = torch.where(kept[:, None], s["h"].float(), zero), s["w"].float()
    at = torch.where(kept, s["target"], 0)[:, None]
    z = h @ w.t()
    if s["cap"]:
        z = torch.tanh(z / s["cap"]).mul_(s["cap"])
    top = z.amax(1, keepdim=True)
    lse = torch.log(torch.exp(z - top).sum(1)) + top[:, 0]
    out = dict(loss=torch.where(kept, lse - z.gather(1, at)[:, 0], zero), lse=torch.where(kept, lse, zero))
    if not grads:
        return out
    dloss = torch.where(kept, s["dloss"], zero)
    both = dloss if s["dlse"] is None else torch.where(kept, s["dloss"] + s["dlse"], zero)
    g = torch.exp(z - lse[:, None]) * both[:, None]
    g.scatter_add_(1, at, -dloss[:, None])
    if s["cap"]:
        g *= 1 - (z / s["cap"]) ** 2
    return dict(out, dh=(g @ w).to(torch.bfloat16), dw=(g.t() @ h).to(torch.bfloat16))


def _ortho(u):
    x = u / (torch.sqrt((u.double() ** 2).sum()).float() + EPS)
    tall = x.shape[0] > x.shape[1]
    x = x.t() if tall else x
    a, b, c = COEFFICIENTS
    for _ in range(STEPS):
        A = x @ x.t()
        x = a * x + (b * A + c * (A @ A)) @ x
    return x.t() if tall else x


def _scale(r, d):
    return 0.2 * math.sqrt(max(r, d))


def _plain(s):
    if s["op"] in ("loss", "grads"):
        return _loss(s, s["op"] == "grads")
    if s["op"] == "ortho":
        return _ortho(s["grad"].float()).to(torch.bfloat16)
    keep = (lambda x: x) if s["keep"] is None else (lambda x: torch.where(s["keep"], x, torch.zeros((), device="cuda")))
    g, m, w = s["grad"].float(), s["momentum"], s["weights"]
    m.copy_(keep(BETA * m + g))
    o = _ortho(keep(g + BETA * m))
    w.copy_(keep((1 - LR * DECAY) * w.float() - LR * _scale(s["r"], s["d"]) * o))
    return dict(weights=w, momentum=m)


# ---- the framework's operators ------------------------------------------------------
def _abi():
    import os
    import sys
    pkg = os.path.join(os.getcwd(), "tensorbit-core_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import tbabi
    return tbabi


def _own(s):
    tb = _abi()
    stream = torch.cuda.current_stream().cuda_stream
    if s["op"] in ("loss", "grads"):
        n, d, vocab = s["n"], s["d"], s["vocab"]
        out = dict(loss=torch.empty(n, device="cuda"), lse=torch.empty(n, device="cuda"))
        common = dict(n=n, d=d, vocab=vocab, h=s["h"].data_ptr(), ldh=s["h"].stride(0), w=s["w"].data_ptr(), ldw=s["w"].stride(0),
                      target=s["target"].data_ptr(), softcap=s["cap"], loss=out["loss"].data_ptr(), lse=out["lse"].data_ptr())
        if s["op"] == "loss":
            tb.check(tb.lm_loss(tb.lm_loss_args(**common), stream=stream))
            return out
        dh = torch.empty(n, _up(d, 8), device="cuda", dtype=torch.bfloat16)
        dw = torch.empty(vocab, _up(d, 8), device="cuda", dtype=torch.bfloat16)
        args = tb.lm_loss_args(**common, dloss=s["dloss"].data_ptr(), dlse=None if s["dlse"] is None else s["dlse"].data_ptr(),
                               dh=dh.data_ptr(), lddh=dh.stride(0), dw=dw.data_ptr(), lddw=dw.stride(0))
        tb.check(tb.lm_loss(args, stream=stream))
        tb.check(tb.lm_loss_backward(args, stream=stream))
        return dict(out, dh=dh[:, :d], dw=dw[:, :d])
    r, d, g = s["r"], s["d"], s["grad"]
    if s["op"] == "ortho":
        o = torch.empty(r, d, device="cuda", dtype=torch.bfloat16)
        tb.check(tb.orthogonalize(g.data_ptr(), CODE[s["g"]], g.stride(0), r, d, o.data_ptr(), tb.BF16, d, steps=STEPS, eps=EPS, stream=stream))
        return o
    w, m = s["weights"], s["momentum"]
    args = tb.muon_args(r=r, d=d, grad=g.data_ptr(), g_dtype=CODE[s["g"]], ldg=g.stride(0), momentum=m.data_ptr(), w=w.data_ptr(),
                        w_dtype=CODE[s["w"]], mask=None if s["mask"] is None else s["mask"].data_ptr(), nm_m=s["m"], beta=BETA, lr=LR,
                        weight_decay=DECAY, scale=_scale(r, d), nesterov=True, steps=STEPS, eps=EPS)
    tb.check(tb.muon_step(args, stream=stream))
    return dict(weights=w, momentum=m)


def run(state):
    with torch.no_grad():
        return _own(state) if own else _plain(state)


# ---- the definition in 64 bits ----------------------------------------------------------
def exact(case, seed):
    """From the definitions, tokens in blocks, the iteration by the eigenvalues' polynomial on one side."""
    s = prepare(case, seed)
    if case["op"] in ("loss", "grads"):
        n, d, vocab = case["n"], case["d"], case["vocab"]
        w = s["w"].double()
        loss, lse = torch.zeros(n, device="cuda", dtype=torch.float64), torch.zeros(n, device="cuda", dtype=torch.float64)
        grads = case["op"] == "grads"
        dh = torch.zeros(n, d, device="cuda", dtype=torch.float64) if grads else None
        dw = torch.zeros(vocab, d, device="cuda", dtype=torch.float64) if grads else None
        kept = torch.nonzero((s["target"] >= 0) & (s["target"] < vocab)).flatten()
        for t in kept.split(512):
            h = s["h"][t].double()
            raw = h @ w.t()
            z = case["cap"] * torch.tanh(raw / case["cap"]) if case["cap"] else raw
            y = s["target"][t]
            i = torch.arange(len(t), device="cuda")
            lse[t] = torch.logsumexp(z, 1)
            loss[t] = lse[t] - z[i, y]
            if grads:
                dl = s["dloss"][t].double()
                total = dl + s["dlse"][t].double() if s["dlse"] is not None else dl
                g = torch.softmax(z, 1) * total[:, None]
                g[i, y] -= dl
                if case["cap"]:
                    g *= 1 / torch.cosh(raw / case["cap"]) ** 2
                dh[t] = g @ w
                dw += g.t() @ h
        return dict(loss=loss, lse=lse, dh=dh, dw=dw) if grads else dict(loss=loss, lse=lse)
    r, d = case["r"], case["d"]

    def ortho(u):
        x = u / (u.norm() + EPS)
        a, b, c = COEFFICIENTS
        for _ in range(STEPS):
            if r <= d:
                A = x @ x.t()
                x = a * x + b * (A @ x) + c * (A @ (A @ x))
            else:
                A = x.t() @ x
                x = a * x + b * (x @ A) + c * ((x @ A) @ A)
        return x

    g = s["grad"].double()
    if case["op"] == "ortho":
        return ortho(g)
    keep = torch.ones((), device="cuda", dtype=torch.float64) if s["keep"] is None else s["keep"].double()
    m = keep * (BETA * s["momentum"].double() + g)
    o = ortho(keep * (g + BETA * m))
    w = keep * (s["weights"].double() * (1 - LR * DECAY) - LR * _scale(r, d) * o)
    return dict(weights=w, momentum=m)


# ---- what a pass cannot do without --------------------------------------------------------
def work(case):
    if case["op"] in ("loss", "grads"):
        n, d, vocab = case["n"], case["d"], case["vocab"]
        kept = n - int(n * case["left"])
        ndv = 2 * kept * d * vocab
        if case["op"] == "loss":
            return dict(bytes=2 * kept * d + 2 * vocab * d + 16 * n, flops=ndv)
        return dict(bytes=4 * n * d + 4 * vocab * d + (24 if case["dlse"] else 20) * n, flops=3 * ndv)
    r, d = case["r"], case["d"]
    k, D = min(r, d), max(r, d)
    size = {"f32": 4, "bf16": 2}
    flops = 6 * k * k * D + 14 * k ** 3
    if case["op"] == "ortho":
        return dict(bytes=r * d * (size[case["g"]] + 2), flops=flops)
    return dict(bytes=r * d * (size[case["g"]] + 8 + 2 * size[case["w"]]) + (r * d // case["m"] if case["m"] else 0), flops=flops)
