"""GPU: orthogonalised updates far below eps, of few directions and of other numbers of steps,
within what the header promises."""
import pytest
import torch

import tbabi as tb
from muon_ref import assert_near, ortho
from test_gpu_muon import gradient, run_ortho, status, stream

pytestmark = pytest.mark.gpu

#: as stated beside the entry: 2-norm, before the rounding to BF16
PROMISED = 5e-4


def f32(x):
    return torch.tensor(x, dtype=torch.float32).item()


# in one launch, with one launch for Q, by clusters, and by pairs of CTAs
@pytest.mark.parametrize("r,d", [(40, 90), (90, 40), (64, 2049), (2049, 64), (300, 200), (2100, 1501), (3100, 3000)])
@pytest.mark.parametrize("far", [1.0, 1e2, 1e5, 1e8, 1e15])
def test_far_below_eps(cuda, r, d, far):
    x = gradient(r, d, "falling")
    eps = f32(x.double().norm().item() * far)
    want = ortho(x, eps=eps)
    assert_near(run_ortho(x, eps=eps), want, want.abs() * 2.0 ** -8, PROMISED * want.norm().item(), f"{far:g}")


@pytest.mark.parametrize("steps", [1, 3, 4, 7, 10])
@pytest.mark.parametrize("far", [3.0, 1e4, 1e12])
@pytest.mark.parametrize("r,d", [(100, 300), (300, 200)])
def test_far_below_eps_in_other_steps(cuda, r, d, far, steps):
    """The power of two that X has goes down with each forming of X anew."""
    x = gradient(r, d, "falling")
    eps = f32(x.double().norm().item() * far)
    want = ortho(x, steps, eps)
    assert_near(run_ortho(x, steps, eps), want, want.abs() * 2.0 ** -8, PROMISED * want.norm().item(), f"{far:g}, {steps} steps")


@pytest.mark.parametrize("r,d", [(128, 128), (64, 2049), (500, 600), (3100, 3000)])
@pytest.mark.parametrize("far", [1e3, 1e9])
def test_step_far_below_eps(cuda, r, d, far):
    x = gradient(r, d, "falling")
    eps = f32(x.double().norm().item() * far)
    want = -ortho(x, eps=eps)
    scale = f32(1.0 / want.abs().max().item())
    want *= scale
    W = torch.zeros(r, d, device="cuda")
    args = tb.muon_args(r=r, d=d, grad=x.data_ptr(), g_dtype=tb.F32, w=W.data_ptr(), w_dtype=tb.F32, lr=1.0, scale=scale, eps=eps)
    tb.check(tb.muon_step(args, stream=stream()))
    status()
    assert_near(W, want, want.abs() * 2.0 ** -22, PROMISED * want.norm().item(), f"{far:g}")


def few_directions(r, d, k, seed=7):
    """k directions and exact zeros beside them but for FP32's rounding (k = 1: all values of one sign)."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    make = (lambda *s: 0.5 + torch.rand(*s, device="cuda", generator=g)) if k == 1 else (lambda *s: torch.randn(*s, device="cuda", generator=g))
    return make(r, k) @ make(k, d) * 1e-3


def allowed(steps):
    """The polynomial's slope is at most a = 3.4445, so much a further step can make of an error; what it adds itself is far smaller."""
    return PROMISED * 3.4445 ** max(0, steps - 5)


@pytest.mark.parametrize("r,d", [(100, 100), (128, 1000), (64, 2049), (130, 260), (1024, 1024), (300, 4000), (3100, 3000)])
@pytest.mark.parametrize("k", [1, 2, 8, 48])
def test_few_directions(cuda, r, d, k):
    x = few_directions(r, d, k)
    for steps in (1, 2, 3, 4, 5, 6, 7, 8):
        want = ortho(x, steps)
        assert_near(run_ortho(x, steps), want, want.abs() * 2.0 ** -8, allowed(steps) * want.norm().item(), f"{steps} steps")


@pytest.mark.parametrize("r,d", [(100, 100), (64, 2049), (130, 260), (300, 200), (1500, 2100), (3300, 3300)])
@pytest.mark.parametrize("kind", ["noise", "falling", "low"])
def test_as_promised(cuda, r, d, kind):
    x = gradient(r, d, kind)
    want = ortho(x)
    assert_near(run_ortho(x), want, want.abs() * 2.0 ** -8, PROMISED * want.norm().item(), kind)
