"""GPU: the operators of a recovery pass as they are used together: the mask of a
pruned projection, the loss behind it, its gradient through the projection's 8-bit
checkpoint, and the masked step; each stage against its definition in 64 bits."""
import pytest
import torch

import tbabi as tb
from lm_loss_ref import assert_within, reference
from muon_ref import OFF, assert_near, step, unpack_mask

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.mark.parametrize("n,d,r,vocab", [(200, 192, 256, 900), (50, 128, 64, 333)])
@pytest.mark.parametrize("captured", [False, True])
def test_recovery_pass(cuda, n, d, r, vocab, captured):
    gen = torch.Generator(device="cuda").manual_seed(0)
    randn = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    x, W = randn(n, d).to(BF), randn(r, d) * 0.1
    head = (randn(vocab, r) * 0.1).to(BF)
    target = torch.randint(0, vocab, (n,), device="cuda", generator=gen)
    target[::5] = -100
    dloss = torch.full((n,), 1.0 / n, device="cuda")
    mask = torch.empty(r * d // 4, device="cuda", dtype=torch.uint8)
    scores, w16, h = torch.empty(r, d, device="cuda"), torch.empty(r, d, device="cuda", dtype=BF), torch.empty(n, r, device="cuda", dtype=BF)
    mom = torch.zeros(r, d, device="cuda")
    codes, exps = torch.empty(n, d, device="cuda", dtype=torch.int8), torch.empty((n + 127) // 128, d, device="cuda", dtype=torch.uint8)
    loss, lse = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    dh, dw, grad = torch.empty(n, r, device="cuda", dtype=BF), torch.empty(vocab, r, device="cuda", dtype=BF), torch.empty(r, d, device="cuda")
    how = dict(beta=0.9, lr=0.01, weight_decay=0.1, scale=1.0)
    tb.check(tb.call("tb_prepare_nm", 2, 4))
    first = torch.cuda.current_stream().cuda_stream
    tb.check(tb.call("tb_importance", W.data_ptr(), tb.F32, None, scores.data_ptr(), r * d, 0.01, 0, first))
    tb.check(tb.call("tb_nm_mask", scores.data_ptr(), mask.data_ptr(), r * d, 2, 4, 0, 3, 0, first))
    keep = unpack_mask(mask, r, d, 4)
    assert (keep.view(-1, 4).sum(1) == 2).all()
    W *= keep

    def one_pass():
        s = torch.cuda.current_stream().cuda_stream
        w16.copy_(W)
        tb.check(tb.adapter_forward(tb.adapter_args(n=n, d=d, r=r, rank=0, n_adapters=0, w=w16.data_ptr(), ldw=d, x=x.data_ptr(), ldx=d, y=h.data_ptr(), ldy=r), s))
        ck = tb.act8(n=n, d=d, codes=codes.data_ptr(), ldq=d, exps=exps.data_ptr(), lde=d)
        tb.check(tb.act8_pack(ck, x.data_ptr(), tb.BF16, d, stream=s))
        args = tb.lm_loss_args(n=n, d=r, vocab=vocab, h=h.data_ptr(), ldh=r, w=head.data_ptr(), ldw=r, target=target.data_ptr(), loss=loss.data_ptr(), lse=lse.data_ptr(),
                               dloss=dloss.data_ptr(), dh=dh.data_ptr(), lddh=r, dw=dw.data_ptr(), lddw=r)
        tb.check(tb.lm_loss(args, s))
        tb.check(tb.lm_loss_backward(args, s))
        tb.check(tb.act8_weight_grad(ck, dh.data_ptr(), tb.BF16, r, r, None, 1, grad.data_ptr(), tb.F32, stream=s))
        tb.check(tb.muon_step(tb.muon_args(r=r, d=d, grad=grad.data_ptr(), g_dtype=tb.F32, momentum=mom.data_ptr(), w=W.data_ptr(), w_dtype=tb.F32, mask=mask.data_ptr(),
                                           nm_m=4, **how), s))

    graph = None
    if captured:
        side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.stream(side):
            graph.capture_begin()
            one_pass()
            graph.capture_end()
        torch.cuda.synchronize()
    for _ in range(3):
        before, momentum = W.clone(), mom.clone()
        graph.replay() if captured else one_pass()
        torch.cuda.synchronize()
        ref = reference(h, head, target, 0.0, dloss)
        for name, got in (("lse", lse), ("loss", loss), ("dh", dh), ("dw", dw)):
            assert_within(got, ref, name)
        # codes hold 7 bits of each feature's largest value of a block: x to half a step of them, 2^-7 of that value
        want = dh.double().t() @ x.double()
        off = dh.double().abs().t() @ (x.double().abs().amax(0) * 2.0 ** -7).expand(n, d)
        assert ((grad.double() - want).abs() <= off + 1e-9).all()
        want_w, want_m, o = step(before, grad, momentum, keep, **how)
        assert_near(W, want_w, (before.double().abs() + 0.01 * o.abs()) * 2.0 ** -22, 0.01 * OFF * o.norm().item(), "weights")
        assert_near(mom, want_m, (momentum.double().abs() + grad.double().abs()) * 2.0 ** -22, 0.0, "momentum")
        assert (W[~keep] == 0).all()
    tb.check(tb.call("tb_gemm_status", torch.cuda.current_stream().cuda_stream))


FIRST_CALL_CAPTURED = """
import sys
import torch
import tbabi as tb
BF, what = torch.bfloat16, sys.argv[1]
n = 20 if what == "few tokens" else 300
r, d = {"short": (40, 100), "clusters": (300, 200), "pairs": (3000, 2600)}.get(what, (0, 0))
h, w = torch.randn(n, 64, device="cuda").to(BF), torch.randn(500, 64, device="cuda").to(BF)
y, one = torch.randint(0, 500, (n,), device="cuda"), torch.ones(n, device="cuda")
loss, lse = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
dh, dw = torch.zeros(n, 64, device="cuda", dtype=BF), torch.zeros(500, 64, device="cuda", dtype=BF)
x = torch.randn(max(1, r), max(1, d), device="cuda")
o = torch.zeros(max(1, r), max(1, d), device="cuda", dtype=BF)
a = tb.lm_loss_args(n=n, d=64, vocab=500, h=h.data_ptr(), ldh=64, w=w.data_ptr(), ldw=64, target=y.data_ptr(), loss=loss.data_ptr(), lse=lse.data_ptr(),
                    dloss=one.data_ptr(), dh=dh.data_ptr(), lddh=64, dw=dw.data_ptr(), lddw=64)


def call():
    s = torch.cuda.current_stream().cuda_stream
    if r:
        tb.check(tb.orthogonalize(x.data_ptr(), tb.F32, d, r, d, o.data_ptr(), tb.BF16, d, stream=s))
    else:
        tb.check(tb.lm_loss(a, s))
        tb.check(tb.lm_loss_backward(a, s))


torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    call()
g.replay()
torch.cuda.synchronize()
got = [t.clone() for t in (loss, lse, dh, dw, o)]
call()
torch.cuda.synchronize()
assert all(torch.equal(p, q) for p, q in zip(got, (loss, lse, dh, dw, o)))
assert (o if r else dw).float().abs().sum() > 0
"""


@pytest.mark.parametrize("what", ["few tokens", "tokens", "short", "clusters", "pairs"])
def test_a_process_first_call_may_be_captured(cuda, tblib, what):
    import os
    import subprocess
    import sys
    env = dict(os.environ, PYTHONPATH=os.path.dirname(tblib.__file__))
    p = subprocess.run([sys.executable, "-c", FIRST_CALL_CAPTURED, what], env=env, capture_output=True, text=True, timeout=300)
    assert p.returncode == 0, p.stderr[-2000:]


def test_host_threads_at_once(cuda):
    """Four host threads, each with a stream and operands of its own."""
    import threading
    from lm_loss_ref import reference
    from muon_ref import ortho
    jobs, failures = [], []
    for i, (n, r, d) in enumerate(((30, 90, 200), (400, 300, 500), (130, 700, 600), (600, 128, 900))):
        gen = torch.Generator(device="cuda").manual_seed(i)
        jobs.append(dict(h=torch.randn(n, 64, device="cuda", generator=gen).to(BF), w=(torch.randn(900, 64, device="cuda", generator=gen) * 0.2).to(BF),
                         y=torch.randint(0, 900, (n,), device="cuda", generator=gen), dloss=torch.rand(n, device="cuda", generator=gen),
                         x=torch.randn(r, d, device="cuda", generator=gen), s=torch.cuda.Stream()))
    torch.cuda.synchronize()

    def run(j):
        try:
            n, (r, d) = len(j["y"]), j["x"].shape
            with torch.cuda.stream(j["s"]):
                for key, shape, t in (("loss", (n,), torch.float32), ("lse", (n,), torch.float32), ("dh", (n, 64), BF), ("dw", (900, 64), BF), ("o", (r, d), BF)):
                    j[key] = torch.empty(shape, device="cuda", dtype=t)
            s = j["s"].cuda_stream
            a = tb.lm_loss_args(n=n, d=64, vocab=900, h=j["h"].data_ptr(), ldh=64, w=j["w"].data_ptr(), ldw=64, target=j["y"].data_ptr(), loss=j["loss"].data_ptr(),
                                lse=j["lse"].data_ptr(), dloss=j["dloss"].data_ptr(), dh=j["dh"].data_ptr(), lddh=64, dw=j["dw"].data_ptr(), lddw=64)
            for _ in range(20):
                tb.check(tb.lm_loss(a, s))
                tb.check(tb.lm_loss_backward(a, s))
                tb.check(tb.orthogonalize(j["x"].data_ptr(), tb.F32, d, r, d, j["o"].data_ptr(), tb.BF16, d, stream=s))
        except Exception as e:  # (a thread's own does not reach the test)
            failures.append(e)

    threads = [threading.Thread(target=run, args=(j,)) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not failures, failures
    for j in jobs:
        ref = reference(j["h"], j["w"], j["y"], 0.0, j["dloss"])
        for name in ("lse", "loss", "dh", "dw"):
            assert_within(j[name], ref, name)
        want = ortho(j["x"])
        assert_near(j["o"], want, want.abs() * 2.0 ** -8, OFF * want.norm().item(), "o")
