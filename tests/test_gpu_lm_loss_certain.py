"""GPU: the loss at the LM head where a token's target has nearly all of the probability,
with logits far from zero."""
import pytest
import torch

import tbabi as tb
from lm_loss_ref import assert_within, reference

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def call(h, w, target, cap=0.0, dloss=None, dh=None, dw=None, dlse=None):
    n, d = h.shape
    loss, lse = torch.full((n,), 7.0, device="cuda"), torch.full((n,), 7.0, device="cuda")
    args = tb.lm_loss_args(n=n, d=d, vocab=w.shape[0], h=h.data_ptr(), ldh=h.stride(0), w=w.data_ptr(), ldw=w.stride(0), target=target.data_ptr(),
                           softcap=cap, loss=loss.data_ptr(), lse=lse.data_ptr())
    stream = torch.cuda.current_stream().cuda_stream
    tb.check(tb.lm_loss(args, stream=stream))
    if dloss is not None:
        args.dlse = None if dlse is None else dlse.data_ptr()
        args.dloss, args.dh, args.lddh, args.dw, args.lddw = dloss.data_ptr(), dh.data_ptr(), dh.stride(0), dw.data_ptr(), dw.stride(0)
        tb.check(tb.lm_loss_backward(args, stream=stream))
    tb.check(tb.call("tb_gemm_status", stream))
    return loss, lse


def between(n, lo, hi, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (lo + (hi - lo) * torch.rand(n, device="cuda", generator=g)).to(BF)


@pytest.mark.parametrize("n", [1, 100, 129, 700])  # in one pass over w, and by tiles
@pytest.mark.parametrize("lo,hi", [(30, 45), (200, 300), (1000, 1500)])
def test_certain_tokens_have_a_loss_of_zero(cuda, n, lo, hi):
    """z is one exact product, and zeros: the loss is log(1 + 999 exp(-z)), below 1e-10."""
    d, vocab = 64, 1000
    for at in (0, 130, 999):
        h, w = torch.zeros(n, d, device="cuda", dtype=BF), torch.zeros(vocab, d, device="cuda", dtype=BF)
        h[:, 3] = between(n, lo, hi, at)
        w[at, 3] = 1.0
        loss, lse = call(h, w, torch.full((n,), at, device="cuda"))
        # the sum of exponentials is 1 and terms below half of its last place, and the maximum's is 1 exactly
        assert (loss >= 0).all() and (loss <= 1e-10).all()
        assert torch.equal(lse, h[:, 3].float())


@pytest.mark.parametrize("n", [100, 700])
@pytest.mark.parametrize("lo,hi", [(30, 45), (200, 300), (1000, 1500)])
def test_nearly_certain_tokens(cuda, n, lo, hi):
    """One other entry of weight: the loss is log(1 + exp(-gap)) of exact logits, however large they are."""
    d, vocab = 64, 1000
    h, w = torch.zeros(n, d, device="cuda", dtype=BF), torch.zeros(vocab, d, device="cuda", dtype=BF)
    h[:, 3], h[:, 5] = between(n, lo, hi, 1), -between(n, 0.25, 12, 2)
    w[20, 3] = w[700, 3] = w[700, 5] = 1.0
    z = torch.stack([h[:, 3].float(), h[:, 3].float() + h[:, 5].float()], 1)  # (rounded once, as the kernel's FP32 sum is)
    loss, _ = call(h, w, torch.full((n,), 20, device="cuda"))
    want = torch.log1p(torch.exp((z[:, 1] - z[:, 0]).double()))
    # logits and gap are exact (sums of 20 bits at most); two exponentials of two units of 2^-23 each, products with log2(e) and a few sums
    off = 2.0 ** -21 * (1 + want)
    assert (loss >= 0).all() and ((loss.double() - want).abs() <= off).all()


@pytest.mark.parametrize("n", [100, 700])
@pytest.mark.parametrize("cap", [0.0, 4000.0])
@pytest.mark.parametrize("size", [60, 1000])
def test_gradients_of_nearly_certain_tokens(cuda, n, cap, size):
    """8192 terms of one sign, which the tensor core's additions cut off: p - 1 of a target with p near 1 is a small difference."""
    d, vocab, at, other = 8192, 300, 20, 290
    g = torch.Generator(device="cuda").manual_seed(0)
    h = (0.5 + torch.rand(n, d, device="cuda", generator=g)).to(BF)
    w = torch.zeros(vocab, d, device="cuda", dtype=BF)
    w[at] = ((0.5 + torch.rand(d, device="cuda", generator=g)) * size / d).to(BF)
    w[other] = (w[at].float() * (1 - 9.2 / size)).to(BF)
    target = torch.full((n,), at, device="cuda")
    dh, dw = torch.empty(n, d, device="cuda", dtype=BF), torch.empty(vocab, d, device="cuda", dtype=BF)
    call(h, w, target, cap, torch.ones(n, device="cuda"), dh, dw)
    hd, wd = h.double(), w.double()
    raw = hd @ wd.t()
    z = cap * torch.tanh(raw / cap) if cap else raw
    lse = torch.logsumexp(z, 1, keepdim=True)
    p = torch.exp(z - lse)
    slope = 1 - (z / cap) ** 2 if cap else torch.ones_like(z)
    one = p.clone()
    one[:, at] -= 1.0
    assert (one[:, at] > -1e-3).all() and (one[:, at] < -1e-5).all()
    # Forward and backward cut the same sums off (of 1024 terms at most, up to 66 steps of 2^-23, and nine additions), and two logits'
    # difference moves p by p (1 - p) of it; tanh and the cap round z twice more, by a few 2^-24.  lse is held to half of its last place;
    # the argument's product with log2(e) and the exponential are off by a few 2^-23.
    moved = 2 * raw.amax(1, keepdim=True) * (66 * 2.0 ** -23 + 9 * 2.0 ** -24) + (4 * 2.0 ** -22 * z.abs().amax(1, keepdim=True) if cap else 0.0)
    p_off = p * ((1 - p) * moved + lse.abs() * 2.0 ** -24 + 2.0 ** -20)
    if cap:  # (the forward's and the backward's z are the same values here too: only the difference to the definition's)
        p_off = p_off + p * (1 - p) * moved
    off = slope * p_off + one.abs() * slope * (2.0 ** -8 + 2.0 ** -20) + one.abs() * 2.0 ** -21
    grad = one * slope
    dh_want, dw_want = grad @ wd, grad.t() @ hd
    dh_off = off @ wd.abs() * 1.01 + grad.abs() @ wd.abs() * (vocab / 16 + 8) * 2.0 ** -23 + dh_want.abs() * 2.0 ** -8 * 1.01
    dw_off = off.t() @ hd.abs() * 1.01 + grad.abs().t() @ hd.abs() * (n / 16 + 8) * 2.0 ** -23 + dw_want.abs() * 2.0 ** -8 * 1.01
    for got, want, bound, name in ((dh, dh_want, dh_off, "dh"), (dw, dw_want, dw_off, "dw")):
        err = (got.double() - want).abs()
        assert (err <= bound + 2.0 ** -133).all(), f"{name}: worst {float((err / (bound + 2.0 ** -133)).max()):.3g} of its bound"


@pytest.mark.parametrize("n", [5, 300])
@pytest.mark.parametrize("cap", [1e-40, 2.0 ** -126, 3e38])
def test_smallest_and_largest_caps(cuda, n, cap):
    """Tokens of zeros: every logit is zero, its slope one.  (1 / 1e-40 is beyond FP32.)"""
    d, vocab = 64, 500
    g = torch.Generator(device="cuda").manual_seed(0)
    w = torch.randn(vocab, d, device="cuda", generator=g).to(BF)
    h = torch.randn(n, d, device="cuda", generator=g).to(BF)
    h[::2] = 0
    target = torch.randint(0, vocab, (n,), device="cuda", generator=g)
    dh, dw = torch.empty(n, d, device="cuda", dtype=BF), torch.empty(vocab, d, device="cuda", dtype=BF)
    loss, lse = call(h, w, target, cap, torch.ones(n, device="cuda"), dh, dw)
    want = torch.log(torch.tensor(float(vocab), device="cuda", dtype=torch.float64))
    for x in (loss[::2], lse[::2]) if cap > 1 else (loss, lse):  # (capped so low all logits are zeros beside one)
        assert ((x.double() - want).abs() <= want * 2.0 ** -22).all()
    one = torch.full((len(target[::2]), vocab), 1.0 / vocab, device="cuda", dtype=torch.float64)
    one[torch.arange(len(one)), target[::2]] -= 1.0
    rows, size = one @ w.double(), one.abs() @ w.double().abs()
    # G's rounding, the result's, and 32 steps of the tensor core's sum
    assert ((dh[::2].double() - rows).abs() <= size * (2.0 ** -8 + 40 * 2.0 ** -23) + rows.abs() * 2.0 ** -8 * 1.01).all()
    assert torch.isfinite(dw).all() and torch.isfinite(dh).all()


@pytest.mark.parametrize("n", [40, 300])
@pytest.mark.parametrize("cap", [0.0, 30.0])
def test_left_out_rows_change_no_bit(cuda, n, cap):
    """Tokens left out hold zeros, then values whose logits are far beyond the cap, then NaN."""
    d, vocab = 256, 700
    g = torch.Generator(device="cuda").manual_seed(0)
    w = (torch.randn(vocab, d, device="cuda", generator=g) * 0.1).to(BF)
    h = torch.randn(n, d, device="cuda", generator=g).to(BF)
    target = torch.randint(0, vocab, (n,), device="cuda", generator=g)
    target[::3] = -100
    got = []
    for size in (0.0, 300.0, float("nan")):
        h[::3] = (torch.randn(len(h[::3]), d, device="cuda", generator=g) * size).to(BF)
        dh, dw = torch.empty(n, d, device="cuda", dtype=BF), torch.empty(vocab, d, device="cuda", dtype=BF)
        got.append((*call(h, w, target, cap, torch.ones(n, device="cuda"), dh, dw), dh, dw))
    for other in got[1:]:
        for x, y in zip(got[0], other):
            assert torch.equal(x, y)


@pytest.mark.parametrize("n", [40, 300])
def test_factors_that_nearly_cancel(cuda, n):
    """dloss + dlse is a small difference: for all entries but the target it alone counts."""
    d, vocab = 64, 500
    g = torch.Generator(device="cuda").manual_seed(0)
    w = torch.randn(vocab, d, device="cuda", generator=g).to(BF)
    h = (torch.randn(n, d, device="cuda", generator=g) * 0.2).to(BF)
    target = torch.randint(0, vocab // 2, (n,), device="cuda", generator=g)  # (the other half of dw is of the differences alone)
    dloss = torch.rand(n, device="cuda", generator=g) + 0.1
    dlse = -dloss * (1 + 2.0 ** -16 * torch.rand(n, device="cuda", generator=g))
    dh, dw = torch.empty(n, d, device="cuda", dtype=BF), torch.empty(vocab, d, device="cuda", dtype=BF)
    call(h, w, target, 0.0, dloss, dh, dw, dlse)
    ref = reference(h, w, target, 0.0, dloss, dlse)
    assert_within(dh, ref, "dh")
    assert_within(dw, ref, "dw")
