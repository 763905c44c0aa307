"""GPU: gradients of the loss at the LM head whose vocabulary is gone through in several
pieces although the tokens are few, and the scratch that they take."""
import os
import subprocess
import sys

import pytest
import torch

import tbabi as tb
from lm_loss_ref import assert_within, reference

pytestmark = pytest.mark.gpu
BF = torch.bfloat16

#: 128 MB of BF16 for up to 128 (16) tokens
PIECE = {100: 524288, 16: 4194304}


def inputs(n, d, vocab):
    g = torch.Generator(device="cuda").manual_seed(n)
    w = torch.empty(vocab, d, device="cuda", dtype=BF).normal_(generator=g).mul_(0.5)
    h = torch.randn(n, d, device="cuda", generator=g).to(BF)
    target = torch.randint(0, vocab, (n,), device="cuda", generator=g)
    target[:6] = torch.tensor([0, PIECE[n] - 1, PIECE[n], PIECE[n] + 1, vocab - 1, -100], device="cuda")
    dloss = torch.rand(n, device="cuda", generator=g)
    dlse = torch.randn(n, device="cuda", generator=g) * 0.1
    return h, w, target, dloss, dlse


def gradients(h, w, target, dloss, dlse):
    (n, d), vocab = h.shape, w.shape[0]
    loss, lse = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    dh, dw = torch.full((n, d), 3.0, device="cuda", dtype=BF), torch.full((vocab, d), 3.0, device="cuda", dtype=BF)
    args = tb.lm_loss_args(n=n, d=d, vocab=vocab, h=h.data_ptr(), ldh=d, w=w.data_ptr(), ldw=d, target=target.data_ptr(), loss=loss.data_ptr(),
                           lse=lse.data_ptr(), dloss=dloss.data_ptr(), dlse=dlse.data_ptr(), dh=dh.data_ptr(), lddh=d, dw=dw.data_ptr(), lddw=d)
    stream = torch.cuda.current_stream().cuda_stream
    tb.check(tb.lm_loss(args, stream=stream))
    tb.check(tb.lm_loss_backward(args, stream=stream))
    tb.check(tb.call("tb_gemm_status", stream))
    return loss, lse, dh, dw


@pytest.mark.parametrize("n,vocab", [(100, PIECE[100]), (100, PIECE[100] + 3), (100, 2 * PIECE[100] + 70001), (16, PIECE[16] + 9)])
def test_few_tokens_of_a_large_vocabulary(cuda, n, vocab):
    h, w, target, dloss, dlse = inputs(n, 8, vocab)
    ref = reference(h, w, target, 0.0, dloss, dlse)
    for name, got in zip(("loss", "lse", "dh", "dw"), gradients(h, w, target, dloss, dlse)):
        assert_within(got, ref, name)


def test_scratch_of_few_tokens(cuda):
    """Three million entries and 100 tokens: 770 MB if G were held whole."""
    code = """
import torch, tbabi as tb
from test_gpu_lm_loss_pieces import gradients, inputs
x = inputs(100, 8, 3000000)
dummy = torch.empty(600 << 20, device="cuda", dtype=torch.uint8)
del dummy  # room for the results, held by torch
small = inputs(100, 8, 600000)
gradients(*small)
torch.cuda.synchronize()
before = torch.cuda.mem_get_info()[0]
gradients(*x)
torch.cuda.synchronize()
print("taken", before - torch.cuda.mem_get_info()[0])
"""
    here = os.path.dirname(os.path.abspath(__file__))
    env = dict(os.environ, PYTHONPATH=os.pathsep.join([here, os.path.join(os.path.dirname(here), "tensorbit-core_b200")]))
    r = subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
    taken = int(r.stdout.split("taken")[1])
    assert taken < 300 << 20, f"{taken >> 20} MB"
