"""GPU: steps of pruned weights of the sizes whose last product is made by pairs of CTAs,
and steps without a momentum."""
import pytest
import torch

import tbabi as tb
from muon_ref import assert_near, step, unpack_mask
from test_gpu_muon import DT, gradient, status, stream
from test_gpu_muon_ranges import PROMISED

pytestmark = pytest.mark.gpu


def check_step(r, d, g, w, m, nesterov, pad, momentum):
    gen = torch.Generator(device="cuda").manual_seed(r + d)
    grad = torch.full((r, d + pad), float("nan"), device="cuda", dtype=DT[g][0])[:, :d]
    grad.copy_(gradient(r, d, "falling"))
    W = torch.full((r + 1, d + pad), 5.0, device="cuda", dtype=DT[w][0])
    W[:r, :d] = torch.randn(r, d, device="cuda", generator=gen) * 0.02
    mom = torch.full((r + 1, d + pad), 5.0, device="cuda") if momentum else None
    if momentum:
        mom[:r, :d] = gradient(r, d, "noise", 4) * 0.1
    assert not m or r * d % m == 0
    mask = torch.randint(0, 256, (r * d // m,), device="cuda", generator=gen, dtype=torch.uint8) if m else None
    keep = unpack_mask(mask, r, d, m) if m else torch.ones(r, d, device="cuda", dtype=torch.bool)
    # what pruned positions hold reaches nothing
    grad[~keep] = float("nan")
    W[:r, :d][~keep] = float("inf")
    if momentum:
        mom[:r, :d][~keep] = float("nan")
    how = dict(beta=0.9, lr=0.01, weight_decay=0.1, scale=2.0, nesterov=nesterov)
    clean = [None if x is None else torch.where(keep, x, torch.zeros((), dtype=x.dtype, device="cuda")) for x in (W[:r, :d], grad, mom[:r, :d] if momentum else None)]
    want_w, want_m, o = step(*clean, keep, **how)
    args = tb.muon_args(r=r, d=d, grad=grad.data_ptr(), g_dtype=DT[g][1], ldg=grad.stride(0), momentum=mom.data_ptr() if momentum else None,
                        ldm=mom.stride(0) if momentum else 0, w=W.data_ptr(), w_dtype=DT[w][1], ldw=W.stride(0), mask=None if mask is None else mask.data_ptr(),
                        nm_m=m, **how)
    tb.check(tb.muon_step(args, stream=stream()))
    status()
    half = 2.0 ** -8 if w == "bf16" else 2.0 ** -24
    terms = clean[0].double().abs() + 0.02 * o.abs()
    assert_near(W[:r, :d], want_w, want_w.abs() * half + terms * 2.0 ** -22, 0.02 * PROMISED * o.norm().item(), "weights")
    assert (W[r:] == 5.0).all() and (W[:, d:] == 5.0).all() and (W[:r, :d][~keep] == 0).all()
    if momentum:
        assert_near(mom[:r, :d], want_m, (clean[2].double().abs() + clean[1].double().abs()) * 2.0 ** -23, 0.0, "momentum")
        assert (mom[r:] == 5.0).all() and (mom[:, d:] == 5.0).all() and (mom[:r, :d][~keep] == 0).all()


@pytest.mark.parametrize("r,d,g,w,m,nesterov,pad,momentum", [
    (1536, 2304, "bf16", "f32", 4, True, 0, True), (2304, 1536, "f32", "bf16", 8, True, 0, True),      # whole pieces, both ways round
    (1600, 2056, "bf16", "bf16", 8, False, 8, True), (1601, 2060, "f32", "f32", 2, True, 4, True),     # ragged edges, rows on whole units
    (2100, 1501, "bf16", "f32", 3, True, 3, True), (2101, 1505, "f32", "bf16", 7, True, 2, True),      # rows on none
    (1500, 2100, "f32", "bf16", 0, True, 1, True), (1505, 2101, "bf16", "f32", 7, False, 0, True),
    (1500, 2100, "bf16", "f32", 4, True, 0, False), (2102, 1502, "f32", "bf16", 1, False, 0, False)])
def test_large_step(cuda, r, d, g, w, m, nesterov, pad, momentum):
    check_step(r, d, g, w, m, nesterov, pad, momentum)


@pytest.mark.parametrize("r,d", [(1, 4), (96, 252), (64, 2048), (2050, 60), (500, 600)])  # in one launch, with one launch for Q, by clusters
@pytest.mark.parametrize("w,m,nesterov", [("f32", 4, True), ("bf16", 2, False), ("f32", 0, True)])
def test_step_without_momentum(cuda, r, d, w, m, nesterov):
    check_step(r, d, "f32" if w == "bf16" else "bf16", w, m, nesterov, 1, False)
