"""Plain restatements, in float64, of the 8-bit checkpoints and of what the
calibration operators compute from them.  All on whatever device the inputs are."""
import math

BLOCK = 128


def up(v, m):
    return (v + m - 1) // m * m


def pack(torch, x, keep=None):
    """(codes, exponents) of x [n][d]: per feature and block of 128 tokens the
    smallest power of two for which every code rounds into [-127, 127], by search."""
    n, d = x.shape
    x = x.double()
    if keep is not None:
        x = torch.where(keep[:, None] != 0, x, torch.zeros((), dtype=torch.float64, device=x.device))
    blocks = -(-n // BLOCK)
    codes = torch.zeros(n, d, dtype=torch.int8, device=x.device)
    exps = torch.zeros(blocks, d, dtype=torch.uint8, device=x.device)
    for i in range(blocks):
        b = x[i * BLOCK:(i + 1) * BLOCK]
        amax = b.abs().amax(0)
        bad = ~torch.isfinite(b).all(0)
        e = torch.ones(d, dtype=torch.int64, device=x.device)
        for _ in range(260):  # raise the exponent while the largest value does not fit
            over = torch.round(amax * torch.exp2((127 - e).double())) > 127
            over &= ~bad
            if not bool(over.any()):
                break
            e += over.long()
        q = torch.round(b * torch.exp2((127 - e).double()))
        q = torch.where(bad[None], torch.zeros_like(q), q)
        codes[i * BLOCK:(i + 1) * BLOCK] = q.to(torch.int8)
        exps[i] = torch.where(bad, torch.full_like(e, 255), e).to(torch.uint8)
    return codes, exps


def values(torch, codes, exps):
    """xhat in float64."""
    s = torch.exp2(exps.double() - 127)
    s = torch.where(exps == 255, torch.full_like(s, math.nan), s)
    return codes.double() * s.repeat_interleave(BLOCK, 0)[: codes.shape[0]]


def gradients(torch, dy, xh, samples):
    """[(G, A)] per sample: the gradient and the sum of its terms' magnitudes."""
    out = []
    n = xh.shape[0]
    for lo, hi in samples:
        lo, hi = max(0, lo), min(n, hi)
        hi = max(lo, hi)
        a, b = dy[lo:hi].double(), xh[lo:hi]
        out.append((a.t() @ b, a.abs().t() @ b.abs()))
    return out


def fisher(torch, grads, alpha, beta, F=None):
    for G in grads:
        F = alpha * G * G if F is None else beta * F + alpha * (1 - beta) * G * G
    return F


class Adapters:
    """Forward and backward of W + scale[a] B_a A_a in float64, with magnitude sums beside each result."""

    def __init__(self, torch, w, a, b, scale, who):
        self.torch, self.w, self.a, self.b, self.scale, self.who = torch, w.double(), a.double(), b.double(), scale.double(), who

    def tokens(self, k):
        return self.torch.nonzero(self.who == k).flatten()

    def forward(self, x, mag=False):
        f = (lambda v: v.abs()) if mag else (lambda v: v)
        x = f(x.double())
        y = x @ f(self.w).t()
        for k in range(self.a.shape[0]):
            t = self.tokens(k)
            y[t] += f(self.scale[k]) * ((x[t] @ f(self.a[k]).t()) @ f(self.b[k]).t())
        return y

    def backward(self, dy, xh, mag=False):
        f = (lambda v: v.abs()) if mag else (lambda v: v)
        dy, xh = f(dy.double()), f(xh)
        dx = dy @ f(self.w)
        da, db = self.torch.zeros_like(self.a), self.torch.zeros_like(self.b)
        for k in range(self.a.shape[0]):
            t = self.tokens(k)
            s, A, B = f(self.scale[k]), f(self.a[k]), f(self.b[k])
            v = s * (dy[t] @ B)
            dx[t] += v @ A
            da[k] = v.t() @ xh[t]
            db[k] = s * (dy[t].t() @ (xh[t] @ A.t()))
        return dx, da, db
