"""The loss at the LM head and its gradients in 64 bits, with bounds on what the
kernels' arithmetic may add, from the unit roundoffs alone.

A logit is a sum of exact products: groups of 1024 terms in the tensor core (in the
backward one of all), whose steps of 16 terms each cut off less than 2^-23 of what the
terms' magnitudes have added up to (and within a step as much again, counted as two
steps more), then FP32 additions of the groups.  A rounding to BF16, whose values have 8 bits, is off by at
most half a step, 2^-8 of the value.  exp, log and the capping's tanh add a few units of 2^-24 and
their arguments' roundings."""
import torch


def inside(target, vocab):
    return (target >= 0) & (target < vocab)


def reference(h, w, target, cap=0.0, dloss=None, dlse=None):
    """dict of float64 results and `*_bound` elementwise; h, w any float type, on their device."""
    n, d = h.shape
    vocab = w.shape[0]
    kept = inside(target, vocab)
    t = torch.nonzero(kept).flatten()
    hd, wd, y = h[t].double(), w.double(), target[t]
    i = torch.arange(len(t), device=h.device)
    raw = hd @ wd.t()
    size = hd.abs() @ wd.abs().t()
    off = size * ((min(d, 1024) / 16 + 2) * 2.0 ** -23 + (d / 1024 + 1) * 2.0 ** -24)
    off_backward = size * (d / 16 + 2) * 2.0 ** -23
    z = raw
    if cap:
        z = cap * torch.tanh(raw / cap)
        off = off + raw.abs() * 2.0 ** -22 + z.abs() * 2.0 ** -21
        off_backward = off_backward + raw.abs() * 2.0 ** -22 + z.abs() * 2.0 ** -21
    lse = torch.logsumexp(z, 1)
    worst = off.amax(1)
    lse_off = worst + 2.0 ** -21 * (4 + z.abs().amax(1) + lse.abs())
    out = {}

    def spread(v, shape, like=0.0):
        x = torch.full(shape, like, dtype=torch.float64, device=h.device)
        x[t] = v
        return x

    out["lse"], out["lse_bound"] = spread(lse, (n,)), spread(lse_off, (n,))
    out["loss"] = spread(lse - z[i, y], (n,))
    out["loss_bound"] = spread(lse_off + off[i, y] + 2.0 ** -23 * (lse.abs() + z[i, y].abs()), (n,))
    if dloss is None:
        return out
    dl = dloss[t].double()
    both = dl + (dlse[t].double() if dlse is not None else 0.0)
    slope = 1 - (z / cap) ** 2 if cap else torch.ones_like(z)
    p = torch.exp(z - lse[:, None])
    hot = torch.zeros_like(z)
    hot[i, y] = 1.0
    g = slope * (both[:, None] * p - dl[:, None] * hot)
    g_size = both.abs()[:, None] * p + dl.abs()[:, None] * hot
    # p's relative error, then the rounding to BF16 and those of FP32; the slope's own error
    p_off = off_backward + lse_off[:, None] + 2.0 ** -21 * (4 + z.abs() + lse.abs()[:, None])
    g_off = slope * (both.abs()[:, None] * p * p_off + g_size * 2.0 ** -22) + g.abs() * 2.0 ** -8 + g_size * 2.0 ** -22 + 2.0 ** -133
    if cap:
        g_off = g_off + g_size * 2 * (off_backward + 2.0 ** -21 * z.abs()) / cap

    def product(a, a_off, b):
        v = a @ b
        k = a.shape[1]
        terms = a.abs() @ b.abs()
        bound = a_off @ b.abs() * 1.01 + terms * (k / 16 + 8) * 2.0 ** -23 + v.abs() * 2.0 ** -8 * 1.01 + 2.0 ** -133
        return v, bound

    dh, dh_off = product(g, g_off, wd)
    out["dh"], out["dh_bound"] = spread(dh, (n, d)), spread(dh_off, (n, d))
    out["dw"], out["dw_bound"] = product(g.t(), g_off.t(), hd)
    return out


def assert_within(got, ref, name):
    """Every value finite where the reference is, and within its bound."""
    err = (got.double() - ref[name]).abs()
    bad = ~(err <= ref[name + "_bound"])
    if bad.any():
        at = torch.nonzero(bad)[0].tolist()
        worst = (err / ref[name + "_bound"].clamp_min(1e-300)).nan_to_num(1e30).max().item()
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} values off, worst {worst:.3g} of its bound, first at {at}: "
                             f"{got[tuple(at)].item()} for {ref[name][tuple(at)].item()}")
