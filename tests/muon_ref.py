"""Orthogonalised updates in 64 bits, and how far the kernels' may be off.

The result is rounded to BF16 once: half a step, 2^-8 of the value.  Before that, sums
of 256 terms in the tensor core: 48 steps (three products of each 16 terms), each
cutting off less than 2^-23 of the terms' sum, so 5.7e-6 of A at most.  A is carried
through two more steps at most, each of which stretches what is added in a direction
of a small singular value by a^2 = 11.9 at most: 8e-4 of P = a + b A + ... there
(|b| / a = 1.4 times 141 times 4e-6 on average over the signs), so that 1e-3 of the
result, as 2-norms, bounds it."""
import torch

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
OFF = 1e-3


def ortho(u, steps=5, eps=1e-7):
    x = u.double()
    x = x / (x.norm() + eps) if bool((x != 0).any()) else torch.zeros_like(x)
    tall = x.shape[0] > x.shape[1]
    x = x.t() if tall else x
    a, b, c = COEFFICIENTS
    for _ in range(steps):
        A = x @ x.t()
        x = a * x + (b * A + c * A @ A) @ x
    return x.t() if tall else x


def unpack_mask(mask, r, d, m):
    """Truth values [r][d] of the .tb mask bytes."""
    bits = (mask.long()[:, None] >> torch.arange(m, device=mask.device)) & 1
    return bits.reshape(-1)[: r * d].view(r, d).bool()


def step(w, grad, momentum, keep, *, beta, lr, weight_decay, scale, nesterov=True, steps=5, eps=1e-7):
    """(W, m, O) after one step, in float64."""
    zero = torch.zeros((), dtype=torch.float64, device=w.device)
    g = torch.where(keep, grad.double(), zero)
    if momentum is None:
        m, u = None, g
    else:
        m = torch.where(keep, beta * momentum.double() + g, zero)
        u = g + beta * m if nesterov else m
    o = ortho(u, steps, eps)
    return torch.where(keep, (1 - lr * weight_decay) * w.double() - lr * scale * o, zero), m, o


def assert_near(got, want, rounding, off, what):
    """|got - want| beyond `rounding` of each value (and of the sum's terms) is below `off` in the 2-norm."""
    err = (got.double() - want).abs()
    assert torch.isfinite(err).all(), f"{what}: {int((~torch.isfinite(err)).sum())} values are not finite"
    rest = (err - rounding).clamp_min(0).norm().item()
    assert rest <= off, f"{what}: {rest:.3g} beyond the rounding, {off:.3g} allowed (norm {want.norm().item():.3g})"
