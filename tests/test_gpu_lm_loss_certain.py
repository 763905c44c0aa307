"""GPU: the loss at the LM head where a token's target has nearly all of the probability,
with logits far from zero."""
import pytest
import torch

import tbabi as tb

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def call(h, w, target, cap=0.0):
    n, d = h.shape
    loss, lse = torch.full((n,), 7.0, device="cuda"), torch.full((n,), 7.0, device="cuda")
    args = tb.lm_loss_args(n=n, d=d, vocab=w.shape[0], h=h.data_ptr(), ldh=h.stride(0), w=w.data_ptr(), ldw=w.stride(0), target=target.data_ptr(),
                           softcap=cap, loss=loss.data_ptr(), lse=lse.data_ptr())
    stream = torch.cuda.current_stream().cuda_stream
    tb.check(tb.lm_loss(args, stream=stream))
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
