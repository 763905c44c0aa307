"""GPU: the loss at the LM head and its gradients against their definition in 64 bits."""
import pytest
import torch

import tbabi as tb
from lm_loss_ref import assert_within, reference

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def up(v, m):
    return (v + m - 1) // m * m


def rows(n, d, pad=8, fill=float("nan")):
    """[n][d] in rows of a stride that is a multiple of 8, NaN behind each row's end and two rows behind the last."""
    return torch.full((n + 2, up(d, 8) + pad), fill, device="cuda", dtype=BF)


def make(n, d, vocab, left=0.0, seed=0, pad=8, sure=6.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    hb, wb = rows(n, d, pad), rows(vocab, d, pad)
    h, w = hb[:n, :d], wb[:vocab, :d]
    w.copy_(torch.randn(vocab, d, device="cuda", generator=g) * 0.5 / d ** 0.5)
    target = torch.randint(0, vocab, (n,), device="cuda", generator=g)
    toward = w[target].float()
    toward /= toward.norm(dim=1, keepdim=True).clamp_min(1e-6)
    h.copy_(torch.randn(n, d, device="cuda", generator=g) * 2 + toward * sure * torch.rand(n, 1, device="cuda", generator=g))
    out = torch.rand(n, device="cuda", generator=g) < left
    target[out] = torch.where(torch.rand(n, device="cuda", generator=g) < 0.5, -100, vocab)[out]
    dloss = torch.rand(n, device="cuda", generator=g) / n
    dlse = torch.randn(n, device="cuda", generator=g) * 0.1 / n
    return h, w, target, dloss, dlse


def call(h, w, target, cap=0.0, dloss=None, dlse=None, dh=None, dw=None, backward=False, lse=None, stream=None):
    n, d = h.shape
    loss = torch.full((n,), 7.0, device="cuda")
    lse = torch.full((n,), 7.0, device="cuda") if lse is None else lse
    args = tb.lm_loss_args(n=n, d=d, vocab=w.shape[0], h=h.data_ptr(), ldh=h.stride(0), w=w.data_ptr(), ldw=w.stride(0), target=target.data_ptr(),
                           softcap=cap, loss=loss.data_ptr(), lse=lse.data_ptr(), dloss=None if dloss is None else dloss.data_ptr(),
                           dlse=None if dlse is None else dlse.data_ptr(), dh=None if dh is None else dh.data_ptr(),
                           lddh=0 if dh is None else dh.stride(0), dw=None if dw is None else dw.data_ptr(), lddw=0 if dw is None else dw.stride(0))
    s = torch.cuda.current_stream().cuda_stream if stream is None else stream
    tb.check(tb.lm_loss(args, stream=s))
    if backward:
        tb.check(tb.lm_loss_backward(args, stream=s))
    return loss, lse


def status():
    tb.check(tb.call("tb_gemm_status", torch.cuda.current_stream().cuda_stream))


FORWARD = [
    # n, d, vocab, left, cap
    (1, 8, 1, 0.0, 0.0), (1, 1, 2, 0.0, 0.0), (1, 64, 127, 0.0, 0.0), (3, 65, 128, 0.0, 30.0), (7, 100, 129, 0.3, 0.0), (64, 512, 257, 0.0, 0.0),
    (255, 513, 1000, 0.5, 2.0), (256, 576, 255, 0.0, 0.0), (257, 1024, 3001, 0.3, 0.0), (1, 4096, 32000, 0.0, 0.0), (600, 200, 5000, 0.9, 30.0),
    (9000, 72, 300, 0.4, 0.0),
]


@pytest.mark.parametrize("n,d,vocab,left,cap", FORWARD)
def test_forward(cuda, n, d, vocab, left, cap):
    h, w, target, _, _ = make(n, d, vocab, left)
    loss, lse = call(h, w, target, cap)
    ref = reference(h, w, target, cap)
    assert_within(lse, ref, "lse")
    assert_within(loss, ref, "loss")
    status()


BACKWARD = [
    # n, d, vocab, left, cap, with dlse
    (1, 8, 1, 0.0, 0.0, False), (1, 1, 2, 0.0, 0.0, True), (2, 64, 127, 0.0, 0.0, False), (3, 65, 129, 0.0, 30.0, True), (37, 100, 700, 0.3, 0.0, False),
    (64, 512, 257, 0.0, 2.0, False), (255, 513, 1000, 0.5, 0.0, True), (300, 264, 3001, 0.3, 0.0, False), (1, 4096, 32000, 0.0, 0.0, False),
    (600, 200, 5000, 0.9, 30.0, True), (9000, 72, 300, 0.4, 0.0, False), (8200, 40, 9000, 0.1, 0.0, False),
]


@pytest.mark.parametrize("n,d,vocab,left,cap,with_dlse", BACKWARD)
def test_gradients(cuda, n, d, vocab, left, cap, with_dlse):
    h, w, target, dloss, dlse = make(n, d, vocab, left, seed=1)
    dlse = dlse if with_dlse else None
    dhb, dwb = rows(n, d, fill=3.0), rows(vocab, d, fill=3.0)
    dh, dw = dhb[:n, :d], dwb[:vocab, :d]
    loss, lse = call(h, w, target, cap, dloss, dlse, dh, dw, backward=True)
    ref = reference(h, w, target, cap, dloss, dlse)
    for name, got in (("lse", lse), ("loss", loss), ("dh", dh), ("dw", dw)):
        assert_within(got, ref, name)
    for buf, r in ((dhb, n), (dwb, vocab)):  # what lies behind rows and their ends stays
        assert (buf[r:] == 3.0).all() and (buf[:, d:] == 3.0).all()
    status()
