"""Cases that measure the calibration operators: 8-bit activation checkpoints,
what their backward pass makes of them (weight gradients per sample, the Fisher
EMA, X^T X for exact OBS), and low-rank adapters beside a shared projection.

`run` computes a case with elementary torch operations in FP32 (own = False) or
through the C ABI (own = True); both take what `prepare` made.

A checkpoint holds activations X [n][d] as int8 codes q and one exponent byte
E for each feature and block of 128 consecutive tokens:

    amax  = max |x| over the block's kept tokens
    E     = max(1, ((bits(amax) + 0x10000) >> 23) - 6)    the smallest power of two 2^(E - 127)
    q     = rint(x * 2^(127 - E))                         with |q| <= 127
    xhat  = q * 2^(E - 127)                               exact in BF16
"""
import math

import torch

own = False

BLOCK = 128
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODE = {"f32": 0, "f16": 1, "bf16": 2}

#: No case costs more than the largest listed one.
MAX_FLOPS, MAX_OUT, MAX_ROUND_TRIP = 9.0e11, 3.0e8, 2.3e8


def listed():
    return [
        # A short prompt's activations of a 4096-wide layer, kept and read back: launch latency.
        dict(name="round trip, 7 tokens", op="checkpoint", n=7, d=4096, x="bf16", padded=False),
        # A padded batch of calibration text at the input of a 14336-wide down_proj.
        dict(name="round trip, padded batch", op="checkpoint", n=16000, d=14336, x="bf16", padded=True),
        # One calibration sample's gradient of a k_proj, in FP32 from an FP32 backward pass.
        dict(name="gradient, k_proj f32", op="grad", S=1, n=509, r=1024, d=4096, dy="f32", g="f32"),
        # Sixteen ragged samples' gradients of a q_proj, as the scoring pass reads them.
        dict(name="gradients, 16 of q_proj", op="grad", S=16, n=8000, r=4096, d=4096, dy="bf16", g="bf16"),
        # The 128 x 128 mock tensor with eight short samples.
        dict(name="fisher, mock", op="fisher", S=8, n=200, r=128, d=128, dy="f32", first=True),
        # Sixty-four ragged calibration samples of a q_proj: the Fisher state without the gradients in memory.
        dict(name="fisher, 64 of q_proj", op="fisher", S=64, n=20000, r=4096, d=4096, dy="bf16", first=True),
        # Calibration Hessian at a 4096-wide input, a second batch added to the first.
        dict(name="hessian, 4096", op="hessian", n=2048, d=4096, accumulate=True),
        # The exact-OBS layer: 2048 tokens at the input of a 14336-wide down_proj.
        dict(name="hessian, 14336", op="hessian", n=2048, d=14336, accumulate=False),
        # One token of one request, a square projection.
        dict(name="adapters, one token", op="forward", n=1, d=4096, r=4096, rank=16, adapters=8, mixed=True),
        # Prompts of several requests at a gate_proj, each with its adapter, some without.
        dict(name="adapters, prompts", op="forward", n=7000, d=4096, r=14336, rank=16, adapters=8, mixed=False),
        # A short batch's gradients at a k_proj.
        dict(name="adapters' gradients, short", op="backward", n=96, d=4096, r=1024, rank=8, adapters=3, mixed=False),
        # A training batch of four adapters of a q_proj.
        dict(name="adapters' gradients", op="backward", n=8000, d=4096, r=4096, rank=64, adapters=4, mixed=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["checkpoint", "grad", "fisher", "hessian", "forward", "backward"])
    d = _log(rng, 64, 14336)
    if op == "checkpoint":
        n = _log(rng, 1, max(1, min(32768, int(MAX_ROUND_TRIP / d))))
        return dict(op=op, n=n, d=d, x=rng.choice(["f32", "f16", "bf16", "bf16"]), padded=rng.random() < 0.5)
    if op == "hessian":
        return dict(op=op, n=_log(rng, 1, max(1, min(16384, int(MAX_FLOPS / (2 * d * d))))), d=d, accumulate=rng.random() < 0.5)
    r = _log(rng, 64, 14336)
    parts = {"bf16": 1, "f16": 2, "f32": 3}
    if op in ("grad", "fisher"):
        dy = rng.choice(["bf16", "bf16", "f16", "f32"])
        S = _log(rng, 1, max(1, min(64, int(MAX_OUT / (r * d)))))
        n = _log(rng, S, max(S, min(16384, int(MAX_FLOPS / (2 * r * d * parts[dy])))))
        if op == "grad":
            return dict(op=op, S=S, n=n, r=r, d=d, dy=dy, g=rng.choice(["f32", "bf16"]))
        return dict(op=op, S=S, n=n, r=r, d=d, dy=dy, first=rng.random() < 0.7)
    n = _log(rng, 1, max(1, min(16384, int(MAX_FLOPS / (4 * r * d)))))
    return dict(op=op, n=n, d=d, r=r, rank=rng.choice([1, 4, 8, 16, 16, 24, 32, 64, 128]), adapters=_log(rng, 1, 16),
                mixed=rng.random() < 0.3)


# ---- inputs ---------------------------------------------------------------------
def _up(v, m):
    return (v + m - 1) // m * m


def _rows(g, n, d, dtype, scale=1.0, heavy=0.0):
    """[n][d] normal values in rows of a stride that is a multiple of 16, 1 % of the columns heavy."""
    buf = torch.zeros(max(1, n), _up(d, 16), device="cuda", dtype=dtype)
    x = buf[:n, :d]
    if n:
        cols = torch.ones(d, device="cuda")
        if heavy:
            cols[torch.randperm(d, device="cuda", generator=g)[: max(1, d // 100)]] = heavy
        x.copy_(torch.randn(n, d, device="cuda", generator=g) * cols * scale)
    return x


def _quantise(x, keep=None):
    """(codes [n][d], exponent bytes [blocks][d]) of x in FP32."""
    n, d = x.shape
    blocks = max(1, -(-n // BLOCK))
    x = x.float()
    if keep is not None:
        x = torch.where(keep[:, None], x, torch.zeros((), device=x.device))
    full = torch.zeros(blocks * BLOCK, d, device=x.device)
    full[:n] = x
    amax = full.abs().view(blocks, BLOCK, d).amax(1)
    e = (((amax.view(torch.int32) + 0x10000) >> 23) - 6).clamp_min(1)
    inv = torch.exp2((127 - e).double()).float()
    codes = torch.round(full.view(blocks, BLOCK, d) * inv[:, None]).view(-1, d)[:n]
    return codes.to(torch.int8), e.to(torch.uint8)


def _values(codes, exps):
    """xhat in FP32."""
    n = codes.shape[0]
    s = torch.exp2(exps.double() - 127).float()
    return codes.float() * s.repeat_interleave(BLOCK, 0)[:n]


def _checkpoint(g, n, d):
    """A checkpoint of n tokens: codes and exponents in rows of a stride that is a multiple of 16."""
    q, e = _quantise(_rows(g, n, d, torch.float32, heavy=20.0))
    codes = torch.zeros(max(1, n), _up(d, 16), device="cuda", dtype=torch.int8)
    exps = torch.zeros(e.shape[0], _up(d, 16), device="cuda", dtype=torch.uint8)
    codes[:n, :d] = q
    exps[:, :d] = e
    return codes, exps


def _samples(g, n, S):
    """S ragged samples that cover n tokens, as [S][2] begins and ends."""
    w = torch.rand(S, device="cuda", generator=g) + 0.25
    ends = (torch.cumsum(w, 0) / w.sum() * n).round().long()
    ends[-1] = n
    begins = torch.cat([torch.zeros(1, device="cuda", dtype=torch.int64), ends[:-1]])
    return torch.stack([begins, ends], 1).contiguous()


def _adapter_of_token(g, n, adapters, mixed):
    """Each token's adapter, -1 for none: runs of tokens of one request, or tokens of many requests mixed."""
    if mixed:
        return torch.randint(0, adapters, (n,), device="cuda", generator=g, dtype=torch.int32)
    runs = 2 * adapters
    ends = _samples(g, n, runs)[:, 1].contiguous()
    who = torch.randint(-1, adapters, (runs,), device="cuda", generator=g, dtype=torch.int32)
    run_of = torch.searchsorted(ends, torch.arange(n, device="cuda"), right=True).clamp_max(runs - 1)
    return who[run_of].contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, n, d = case["op"], case["n"], case["d"]
    s = dict(case)
    if op == "checkpoint":
        s["data"] = _rows(g, n, d, DTYPES[case["x"]], heavy=20.0)
        s["keep"] = None
        if case["padded"]:  # sequences padded to one length: 1 for text
            length = max(1, n // 8)
            text = torch.randint(length // 2, length + 1, (n // length + 1,), device="cuda", generator=g)
            t = torch.arange(n, device="cuda")
            s["keep"] = (t % length < text[t // length]).to(torch.uint8)
        return s
    s["codes"], s["exps"] = _checkpoint(g, n, d)
    if op == "hessian":
        s["H"] = torch.zeros(d, d, device="cuda")
        if case["accumulate"]:
            s["H"].copy_(torch.randn(d, d, device="cuda", generator=g).mul_(0.1).add_(torch.eye(d, device="cuda")))
        return s
    r = case["r"]
    if op in ("grad", "fisher"):
        s["dy_data"] = _rows(g, n, r, DTYPES[case["dy"]], scale=1e-2)
        s["samples"] = _samples(g, n, case["S"])
        if op == "fisher":
            s["F"] = torch.zeros(r, d, device="cuda")
            if not case["first"]:
                s["F"].copy_(torch.rand(r, d, device="cuda", generator=g) * 1e-6)
        return s
    na, rank = case["adapters"], case["rank"]
    bf = torch.bfloat16
    s["w"] = _rows(g, r, d, bf, scale=0.02)
    s["a"] = _rows(g, na * rank, d, bf, scale=1.0 / math.sqrt(d))
    s["b"] = _rows(g, na * r, rank, bf, scale=0.05)
    s["scale"] = torch.rand(na, device="cuda", generator=g) + 0.5
    s["who"] = _adapter_of_token(g, n, na, case["mixed"])
    if op == "forward":
        s["data"] = _rows(g, n, d, bf)
    else:
        s["dy_data"] = _rows(g, n, r, bf, scale=1e-2)
    return s


# ---- the plain forms --------------------------------------------------------------
def _by_sample(s, x):
    """x's rows as [S][longest][...], zeros behind each sample's end."""
    begins, ends = s["samples"][:, 0], s["samples"][:, 1]
    longest = max(1, int((ends - begins).max()))
    t = begins[:, None] + torch.arange(longest, device=x.device)
    inside = t < ends[:, None]
    return torch.where(inside[..., None], x[torch.where(inside, t, 0)], torch.zeros((), device=x.device))


def _lower_tiles(d):
    t = torch.arange(d, device="cuda") // 128
    return t[:, None] >= t[None, :]


def _one_hot(s):
    """[n][adapters] in FP32: the scale of each token's adapter, 0 elsewhere."""
    na = s["adapters"]
    return (s["who"][:, None] == torch.arange(na, device="cuda")[None]) * s["scale"]


def _plain(s):
    op, n, d = s["op"], s["n"], s["d"]
    if op == "checkpoint":
        keep = None if s["keep"] is None else s["keep"] != 0
        return _values(*_quantise(s["data"], keep)).to(torch.bfloat16)
    x = _values(s["codes"][:n, :d], s["exps"][:, :d]) if op != "forward" else None
    if op == "hessian":
        H = torch.where(_lower_tiles(d), (x.t() @ x) / max(1, n), torch.zeros((), device="cuda"))
        return torch.where(_lower_tiles(d), s["H"] + H, s["H"]) if s["accumulate"] else H
    r = s["r"]
    if op in ("grad", "fisher"):
        dy = _by_sample(s, s["dy_data"].float())
        grads = dy.transpose(1, 2) @ _by_sample(s, x)
        if op == "grad":
            return grads.to(DTYPES[s["g"]])
        S, alpha, beta = s["S"], 0.01, 0.99
        c = alpha * (1 - beta) * beta ** torch.arange(S - 1, -1, -1, dtype=torch.float64, device="cuda")
        if s["first"]:
            c[0] = alpha * beta ** (S - 1)
        F = (grads.square_() * c.float()[:, None, None]).sum(0)
        return F if s["first"] else F + s["F"] * beta ** S
    na, rank = s["adapters"], s["rank"]
    w, a, b = s["w"].float(), s["a"].float(), s["b"].float()
    hot = _one_hot(s)
    rows = b.view(na, r, rank)
    flat_b = rows.transpose(1, 2).reshape(na * rank, r)
    if op == "forward":
        xf = s["data"].float()
        u = ((xf @ a.t()).view(n, na, rank) * hot[..., None]).view(n, na * rank)
        return (xf @ w.t() + u @ flat_b).to(torch.bfloat16)
    dy = s["dy_data"].float()
    v = ((dy @ flat_b.t()).view(n, na, rank) * hot[..., None]).view(n, na * rank)
    u = ((x @ a.t()).view(n, na, rank) * hot[..., None]).view(n, na * rank)
    dx = dy @ w + v @ a
    da = v.t() @ x
    db = (u.t() @ dy).view(na, rank, r).transpose(1, 2)
    return dict(dx=dx.to(torch.bfloat16), da=da.view(na, rank, d).to(torch.bfloat16), db=db.contiguous().to(torch.bfloat16))


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
    op, n, d = s["op"], s["n"], s["d"]
    stream = torch.cuda.current_stream().cuda_stream
    if op == "checkpoint":
        x, ld = s["data"], _up(d, 16)
        codes = torch.empty(n, ld, device="cuda", dtype=torch.int8)
        exps = torch.empty(-(-n // BLOCK), ld, device="cuda", dtype=torch.uint8)
        out = torch.empty(n, d, device="cuda", dtype=torch.bfloat16)
        ck = tb.act8(n=n, d=d, codes=codes.data_ptr(), ldq=ld, exps=exps.data_ptr(), lde=ld)
        keep = None if s["keep"] is None else s["keep"].data_ptr()
        tb.check(tb.act8_pack(ck, x.data_ptr(), CODE[s["x"]], x.stride(0), keep=keep, stream=stream))
        tb.check(tb.act8_unpack(ck, out.data_ptr(), tb.BF16, d, stream=stream))
        return out
    ck = tb.act8(n=n, d=d, codes=s["codes"].data_ptr(), ldq=s["codes"].stride(0), exps=s["exps"].data_ptr(),
                 lde=s["exps"].stride(0))
    if op == "hessian":
        H = s["H"].clone() if s["accumulate"] else torch.zeros(d, d, device="cuda")
        tb.check(tb.act8_hessian(ck, 1.0 / max(1, n), H.data_ptr(), accumulate=s["accumulate"], stream=stream))
        return H
    r = s["r"]
    if op in ("grad", "fisher"):
        dy = s["dy_data"]
        if op == "grad":
            out = torch.empty(s["S"], r, d, device="cuda", dtype=DTYPES[s["g"]])
            tb.check(tb.act8_weight_grad(ck, dy.data_ptr(), CODE[s["dy"]], dy.stride(0), r, s["samples"].data_ptr(), s["S"],
                                         out.data_ptr(), CODE[s["g"]], stream=stream))
            return out
        F = torch.empty(r, d, device="cuda") if s["first"] else s["F"].clone()
        tb.check(tb.act8_fisher(ck, dy.data_ptr(), CODE[s["dy"]], dy.stride(0), r, s["samples"].data_ptr(), s["S"],
                                F.data_ptr(), alpha=0.01, beta=0.99, first_step=s["first"], stream=stream))
        return F
    na, rank = s["adapters"], s["rank"]
    common = dict(n=n, d=d, r=r, rank=rank, n_adapters=na, w=s["w"].data_ptr(), ldw=s["w"].stride(0), a=s["a"].data_ptr(),
                  lda=s["a"].stride(0), b=s["b"].data_ptr(), ldb=s["b"].stride(0), scale=s["scale"].data_ptr(),
                  token_adapter=s["who"].data_ptr())
    if op == "forward":
        y = torch.empty(n, _up(r, 8), device="cuda", dtype=torch.bfloat16)
        args = tb.adapter_args(**common, x=s["data"].data_ptr(), ldx=s["data"].stride(0), y=y.data_ptr(), ldy=y.stride(0))
        tb.check(tb.adapter_forward(args, stream=stream))
        return y[:, :r]
    dx = torch.empty(n, _up(d, 8), device="cuda", dtype=torch.bfloat16)
    da = torch.empty(na, rank, s["a"].stride(0), device="cuda", dtype=torch.bfloat16)
    db = torch.empty(na, r, s["b"].stride(0), device="cuda", dtype=torch.bfloat16)
    args = tb.adapter_args(**common, dy=s["dy_data"].data_ptr(), lddy=s["dy_data"].stride(0), x8=ck, dx=dx.data_ptr(),
                           lddx=dx.stride(0), da=da.data_ptr(), db=db.data_ptr())
    tb.check(tb.adapter_backward(args, stream=stream))
    return dict(dx=dx[:, :d], da=da[..., :d], db=db[..., :rank])


def run(state):
    with torch.no_grad():
        return _own(state) if own else _plain(state)


# ---- the definition in 64 bits ----------------------------------------------------------
def exact(case, seed):
    """From the definitions, sample by sample and adapter by adapter."""
    s = prepare(case, seed)
    op, n, d = case["op"], case["n"], case["d"]
    if op == "checkpoint":
        x = s["data"].double()
        out = torch.zeros(n, d, device="cuda", dtype=torch.float64)
        for t0 in range(0, n, BLOCK):
            blk = x[t0:t0 + BLOCK]
            if s["keep"] is not None:
                blk = blk * (s["keep"][t0:t0 + BLOCK, None] != 0)
            amax = blk.abs().amax(0)
            step = torch.exp2(torch.floor(torch.log2(amax.clamp_min(2.0 ** -120))) - 6)
            step = torch.where(torch.round(amax / step) > 127, 2 * step, step)
            step = torch.where(torch.round(amax / (step / 2)) <= 127, step / 2, step).clamp_min(2.0 ** -126)
            out[t0:t0 + BLOCK] = torch.round(blk / step) * step
        return out
    if op != "forward":
        x = s["codes"][:n, :d].double()
        for t0 in range(0, n, BLOCK):
            x[t0:t0 + BLOCK] *= torch.pow(2.0, s["exps"][t0 // BLOCK, :d].double() - 127.0)
    if op == "hessian":
        H = s["H"].double()
        for i in range(0, d, 128):
            part = x[:, i:i + 128].t() @ x[:, :i + 128] / max(1, n)
            H[i:i + 128, :i + 128] = part + (H[i:i + 128, :i + 128] if case["accumulate"] else 0.0)
        return H
    r = case["r"]
    if op in ("grad", "fisher"):
        dy = s["dy_data"].double()
        F = None if op == "grad" or case["first"] else s["F"].double()
        grads = []
        for i, (lo, hi) in enumerate(s["samples"].tolist()):
            G = dy[lo:hi].t() @ x[lo:hi]
            if op == "grad":
                grads.append(G)
            elif F is None:
                F = 0.01 * G * G
            else:
                F = 0.99 * F + 0.01 * (1 - 0.99) * G * G
        return torch.stack(grads) if op == "grad" else F
    na, rank = case["adapters"], case["rank"]
    w, a, b = s["w"].double(), s["a"].double().view(na, rank, d), s["b"].double().view(na, r, rank)
    scale = s["scale"].double()
    if op == "forward":
        xd = s["data"].double()
        y = xd @ w.t()
        for k in range(na):
            t = torch.nonzero(s["who"] == k).flatten()
            y[t] += scale[k] * ((xd[t] @ a[k].t()) @ b[k].t())
        return y
    dy = s["dy_data"].double()
    dx, da, db = dy @ w, torch.zeros_like(a), torch.zeros_like(b)
    for k in range(na):
        t = torch.nonzero(s["who"] == k).flatten()
        v = scale[k] * (dy[t] @ b[k])
        dx[t] += v @ a[k]
        da[k] = v.t() @ x[t]
        db[k] = scale[k] * (dy[t].t() @ (x[t] @ a[k].t()))
    return dict(dx=dx, da=da, db=db)


# ---- what a pass cannot do without --------------------------------------------------------
def work(case):
    op, n, d = case["op"], case["n"], case["d"]
    size = {"f32": 4, "f16": 2, "bf16": 2}
    blocks = -(-n // BLOCK)
    if op == "checkpoint":  # the values in, codes and exponents out; those in, values out
        return dict(bytes=n * d * (size[case["x"]] + 1 + 1 + 2) + 2 * blocks * d, flops=4 * n * d)
    if op == "hessian":  # the lower triangle alone
        return dict(bytes=n * d + blocks * d + (4 if case["accumulate"] else 2) * d * (d + 128), flops=n * d * (d + 1))
    r = case["r"]
    if op == "grad":
        return dict(bytes=n * d + blocks * d + n * r * size[case["dy"]] + case["S"] * r * d * size[case["g"]], flops=2 * n * r * d)
    if op == "fisher":
        return dict(bytes=n * d + blocks * d + n * r * size[case["dy"]] + r * d * (4 if case["first"] else 8),
                    flops=2 * n * r * d + 3 * case["S"] * r * d)
    na, rank = case["adapters"], case["rank"]
    used = min(na, n)
    shared = 2 * r * d + used * rank * (r + d) * 2
    if op == "forward":
        return dict(bytes=shared + 2 * n * (r + d), flops=2 * n * r * d + 2 * n * rank * (r + d))
    return dict(bytes=shared + n * d + blocks * d + 2 * n * r + 2 * n * d + na * rank * (r + d) * 2,
                flops=2 * n * r * d + 6 * n * rank * (r + d))
