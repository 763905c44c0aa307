"""CPU: argument checks of the loss and update entries that return before any
device work, and the layout of their structures."""
import ctypes as C

import pytest

import tbabi as tb

P = 1 << 20  # a 16-byte aligned address that is never read


def test_struct_layouts():
    assert C.sizeof(tb.LmLossArgs) == 136  # 24 of sizes, 40 of h, w and targets, 24 of cap, loss, lse, 48 backward
    assert C.sizeof(tb.MuonArgs) == 112    # 16 of sizes, 48 of gradient, momentum and weights, 16 of types and mask, 32 of factors


def loss(**kw):
    a = dict(n=5, d=64, vocab=100, h=P, ldh=64, w=P, ldw=64, target=P, loss=P, lse=P, dloss=P, dh=P, lddh=64, dw=P, lddw=64)
    a.update(kw)
    return tb.lm_loss_args(**a)


@pytest.mark.parametrize("kw,code", [
    (dict(d=0), tb.TB_ERR_ZERO_SIZE), (dict(vocab=0), tb.TB_ERR_ZERO_SIZE), (dict(n=-1), tb.TB_ERR_SHAPE), (dict(n=1 << 31), tb.TB_ERR_SHAPE),
    (dict(d=(1 << 31) - 200, ldh=1 << 31, ldw=1 << 31), tb.TB_ERR_SHAPE), (dict(vocab=(1 << 31) - 200), tb.TB_ERR_SHAPE),
    (dict(dtype=tb.F32), tb.TB_ERR_UNSUPPORTED), (dict(dtype=tb.F16), tb.TB_ERR_UNSUPPORTED), (dict(softcap=-1.0), tb.TB_ERR_CONFIG),
    (dict(softcap=float("nan")), tb.TB_ERR_CONFIG), (dict(softcap=float("inf")), tb.TB_ERR_CONFIG), (dict(h=None), tb.TB_ERR_ARG), (dict(w=None), tb.TB_ERR_ARG),
    (dict(h=P + 2), tb.TB_ERR_ARG), (dict(w=P + 8), tb.TB_ERR_ARG), (dict(ldh=63), tb.TB_ERR_ARG), (dict(ldh=68), tb.TB_ERR_ARG), (dict(ldw=56), tb.TB_ERR_ARG),
    (dict(target=None), tb.TB_ERR_ARG), (dict(target=P + 4), tb.TB_ERR_ARG), (dict(lse=None), tb.TB_ERR_ARG), (dict(lse=P + 1), tb.TB_ERR_ARG)])
def test_loss_refusals(tblib, kw, code):
    a = loss(**kw)
    assert tb.lm_loss(a) == code
    assert tb.lm_loss_backward(a) == code


def test_loss_call_refusals(tblib):
    assert tb.lm_loss(loss(loss=None)) == tb.TB_ERR_ARG
    assert tb.lm_loss_backward(loss(dloss=None)) == tb.TB_ERR_ARG
    assert tb.lm_loss_backward(loss(dlse=P + 2)) == tb.TB_ERR_ARG
    assert tb.lm_loss_backward(loss(lddh=63)) == tb.TB_ERR_ARG
    assert tb.lm_loss_backward(loss(lddw=60)) == tb.TB_ERR_ARG
    assert tb.lm_loss_backward(loss(dh=P + 1)) == tb.TB_ERR_ARG
    assert tb.lm_loss_backward(loss(dw=P + 1)) == tb.TB_ERR_ARG
    a = loss()
    a.struct_size = 8
    assert tb.lm_loss(a) == tb.TB_ERR_ARG and tb.lm_loss_backward(a) == tb.TB_ERR_ARG
    assert b"struct_size" in tb.lib().tb_last_error()
    # nothing to do: no device is asked for
    assert tb.lm_loss(loss(n=0, h=None, target=None, loss=None, lse=None)) == tb.TB_OK
    assert tb.lm_loss_backward(loss(dh=None, dw=None)) == tb.TB_OK
    assert tb.lm_loss_backward(loss(n=0, dw=None)) == tb.TB_OK


def ortho(x=P, x_dtype=tb.F32, ldx=64, r=32, d=64, out=P, out_dtype=tb.BF16, ldo=64, steps=5, eps=1e-7):
    return tb.orthogonalize(x, x_dtype, ldx, r, d, out, out_dtype, ldo, steps=steps, eps=eps)


@pytest.mark.parametrize("kw,code", [
    (dict(r=0), tb.TB_ERR_ZERO_SIZE), (dict(d=0), tb.TB_ERR_ZERO_SIZE), (dict(r=(1 << 31) - 100), tb.TB_ERR_SHAPE),
    (dict(r=32769, d=32769, ldx=32769, ldo=32769), tb.TB_ERR_CAPACITY), (dict(x_dtype=tb.F16), tb.TB_ERR_UNSUPPORTED), (dict(x_dtype=9), tb.TB_ERR_ARG),
    (dict(out_dtype=tb.F32), tb.TB_ERR_UNSUPPORTED), (dict(out_dtype=-1), tb.TB_ERR_ARG), (dict(steps=0), tb.TB_ERR_CONFIG), (dict(steps=33), tb.TB_ERR_CONFIG),
    (dict(eps=-1.0), tb.TB_ERR_CONFIG), (dict(eps=float("nan")), tb.TB_ERR_CONFIG), (dict(x=None), tb.TB_ERR_ARG), (dict(out=None), tb.TB_ERR_ARG),
    (dict(x=P + 2), tb.TB_ERR_ARG), (dict(out=P + 1), tb.TB_ERR_ARG), (dict(ldx=63), tb.TB_ERR_ARG), (dict(ldo=63), tb.TB_ERR_ARG)])
def test_orthogonalize_refusals(tblib, kw, code):
    assert ortho(**kw) == code


def muon(**kw):
    a = dict(r=32, d=64, grad=P, g_dtype=tb.BF16, momentum=P, w=P, w_dtype=tb.F32, mask=P, nm_m=4, lr=0.1)
    a.update(kw)
    return tb.muon_args(**a)


@pytest.mark.parametrize("kw,code", [
    (dict(r=0), tb.TB_ERR_ZERO_SIZE), (dict(g_dtype=tb.F16), tb.TB_ERR_UNSUPPORTED), (dict(w_dtype=tb.F16), tb.TB_ERR_UNSUPPORTED), (dict(g_dtype=5), tb.TB_ERR_ARG),
    (dict(w_dtype=5), tb.TB_ERR_ARG), (dict(grad=None), tb.TB_ERR_ARG), (dict(w=None), tb.TB_ERR_ARG), (dict(w=P + 2), tb.TB_ERR_ARG), (dict(momentum=P + 2), tb.TB_ERR_ARG),
    (dict(ldg=63), tb.TB_ERR_ARG), (dict(ldm=63), tb.TB_ERR_ARG), (dict(ldw=63), tb.TB_ERR_ARG), (dict(ldw=-1), tb.TB_ERR_ARG), (dict(nm_m=0), tb.TB_ERR_CONFIG),
    (dict(nm_m=9), tb.TB_ERR_UNSUPPORTED), (dict(nm_m=5), tb.TB_ERR_SHAPE), (dict(lr=float("nan")), tb.TB_ERR_CONFIG), (dict(beta=float("inf")), tb.TB_ERR_CONFIG),
    (dict(scale=float("-inf")), tb.TB_ERR_CONFIG), (dict(steps=0), tb.TB_ERR_CONFIG), (dict(eps=float("inf")), tb.TB_ERR_CONFIG)])
def test_muon_refusals(tblib, kw, code):
    assert tb.muon_step(muon(**kw)) == code
    a = muon()
    a.struct_size = 16
    assert tb.muon_step(a) == tb.TB_ERR_ARG
