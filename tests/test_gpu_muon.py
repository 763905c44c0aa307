"""GPU: orthogonalised updates and the masked step against their definition in 64 bits."""
import pytest
import torch

import tbabi as tb
from muon_ref import OFF, assert_near, ortho, step, unpack_mask

pytestmark = pytest.mark.gpu
DT = {"f32": (torch.float32, tb.F32), "bf16": (torch.bfloat16, tb.BF16)}


def status():
    tb.check(tb.call("tb_gemm_status", torch.cuda.current_stream().cuda_stream))


def stream():
    return torch.cuda.current_stream().cuda_stream


def gradient(r, d, kind, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    if kind == "noise":
        return randn(r, d) * 1e-3
    k = min(r, d, 48)
    fall = torch.arange(1, k + 1, device="cuda").float() ** (-1.0 if kind == "falling" else 0.0)
    x = (randn(r, k) * fall) @ randn(k, d)
    return (x + {"falling": 1e-2, "low": 0.0}[kind] * randn(r, d)) * 1e-4


def run_ortho(x, steps=5, eps=1e-7, pad=0):
    r, d = x.shape
    buf = torch.full((r + 1, d + pad), 3.0, device="cuda", dtype=torch.bfloat16)
    code = {torch.float32: tb.F32, torch.bfloat16: tb.BF16}[x.dtype]
    tb.check(tb.orthogonalize(x.data_ptr(), code, x.stride(0), r, d, buf.data_ptr(), tb.BF16, d + pad, steps=steps, eps=eps, stream=stream()))
    assert (buf[r:] == 3.0).all() and (buf[:, d:] == 3.0).all()
    status()
    return buf[:r, :d]


SHAPES = [(1, 1), (1, 7), (5, 1), (2, 3), (16, 130), (127, 128), (128, 128), (129, 64), (255, 257), (256, 512), (300, 1000), (1111, 333), (513, 700), (777, 776)]


@pytest.mark.parametrize("r,d", SHAPES)
@pytest.mark.parametrize("kind", ["noise", "falling", "low"])
def test_orthogonalize(cuda, r, d, kind):
    x = gradient(r, d, kind)
    want = ortho(x)
    assert_near(run_ortho(x), want, want.abs() * 2.0 ** -8, OFF * want.norm().item(), kind)


@pytest.mark.parametrize("steps", [1, 2, 3, 4, 6, 7, 10])
def test_steps(cuda, steps):
    x = gradient(130, 260, "falling").bfloat16()
    want = ortho(x, steps)
    assert_near(run_ortho(x, steps, pad=3), want, want.abs() * 2.0 ** -8, OFF * want.norm().item(), f"{steps} steps")


@pytest.mark.parametrize("r,d,g,w,m,nesterov,pad", [
    (1, 4, "f32", "f32", 4, True, 0), (128, 128, "f32", "f32", 4, True, 0), (128, 128, "bf16", "bf16", 0, False, 0), (96, 250, "bf16", "f32", 8, True, 3),
    (301, 130, "f32", "bf16", 2, True, 1), (257, 129, "bf16", "f32", 3, False, 0), (500, 600, "bf16", "bf16", 8, True, 8), (64, 2049, "f32", "f32", 7, True, 5)])
def test_step(cuda, r, d, g, w, m, nesterov, pad):
    gen = torch.Generator(device="cuda").manual_seed(3)
    if m and r * d % m:
        r = r * m
    grad = torch.full((r, d + pad), float("nan"), device="cuda", dtype=DT[g][0])[:, :d]
    grad.copy_(gradient(r, d, "falling"))
    W = torch.full((r + 1, d + pad), 5.0, device="cuda", dtype=DT[w][0])
    W[:r, :d] = torch.randn(r, d, device="cuda", generator=gen) * 0.02
    mom = torch.full((r + 1, d + pad), 5.0, device="cuda")
    mom[:r, :d] = gradient(r, d, "noise", 4) * 0.1
    mask = torch.randint(0, 256, (max(1, r * d // max(1, m)),), device="cuda", generator=gen, dtype=torch.uint8) if m else None
    keep = unpack_mask(mask, r, d, m) if m else torch.ones(r, d, device="cuda", dtype=torch.bool)
    # what pruned positions hold reaches nothing
    grad[~keep] = float("nan")
    W[:r, :d][~keep] = float("inf")
    mom[:r, :d][~keep] = float("nan")
    how = dict(beta=0.9, lr=0.01, weight_decay=0.1, scale=2.0, nesterov=nesterov)
    clean = [torch.where(keep, x, torch.zeros((), dtype=x.dtype, device="cuda")) for x in (W[:r, :d], grad, mom[:r, :d])]
    want_w, want_m, o = step(*clean, keep, **how)
    args = tb.muon_args(r=r, d=d, grad=grad.data_ptr(), g_dtype=DT[g][1], ldg=grad.stride(0), momentum=mom.data_ptr(), ldm=mom.stride(0), w=W.data_ptr(),
                        w_dtype=DT[w][1], ldw=W.stride(0), mask=None if mask is None else mask.data_ptr(), nm_m=m, **how)
    tb.check(tb.muon_step(args, stream=stream()))
    status()
    half = 2.0 ** -8 if w == "bf16" else 2.0 ** -24
    terms = clean[0].double().abs() + 0.02 * o.abs()
    assert_near(W[:r, :d], want_w, want_w.abs() * half + terms * 2.0 ** -22, 0.02 * OFF * o.norm().item(), "weights")
    assert_near(mom[:r, :d], want_m, (clean[2].double().abs() + clean[1].double().abs()) * 2.0 ** -23, 0.0, "momentum")
    assert (W[r:] == 5.0).all() and (W[:, d:] == 5.0).all() and (mom[r:] == 5.0).all() and (mom[:, d:] == 5.0).all()
    assert (W[:r, :d][~keep] == 0).all() and (mom[:r, :d][~keep] == 0).all()


@pytest.mark.parametrize("r,d", [(1500, 2100), (2100, 1501), (4097, 1700), (3100, 3000), (3300, 3300)])  # by clusters, and by pairs of CTAs
def test_larger(cuda, r, d):
    x = gradient(r, d, "falling")
    want = ortho(x)
    assert_near(run_ortho(x, pad=1), want, want.abs() * 2.0 ** -8, OFF * want.norm().item(), "larger")


@pytest.mark.parametrize("r,d", [(40, 90), (300, 200)])
def test_zeros_and_ranges(cuda, r, d):
    z = torch.zeros(r, d, device="cuda")
    assert (run_ortho(z) == 0).all()
    assert (run_ortho(z, eps=0.0) == 0).all()
    x = gradient(r, d, "noise")
    want = ortho(x, eps=0.0)
    for scale in (2.0 ** -100, 2.0 ** 100):  # (the squares leave FP32's range)
        assert_near(run_ortho(x * scale, eps=0.0), want, want.abs() * 2.0 ** -8, OFF * want.norm().item(), f"times {scale:g}")
    tiny = run_ortho(x * 2.0 ** -100)  # far below eps
    assert (tiny.float().abs() <= 1e-20).all()
    for bad in (float("nan"), float("inf")):
        y = x.clone()
        y[r // 2, d // 3] = bad
        assert torch.isnan(run_ortho(y)).all()


@pytest.mark.parametrize("r,d", [(100, 300), (700, 900)])
def test_same_bits_again(cuda, r, d):
    x = gradient(r, d, "falling")
    first = run_ortho(x).clone()
    for _ in range(3):
        assert torch.equal(run_ortho(x), first)


@pytest.mark.parametrize("r,d", [(64, 200), (600, 520)])
def test_step_captured_and_replayed(cuda, r, d):
    """Steps of a graph follow steps of the formula, new gradients each."""
    m = 4
    gen = torch.Generator(device="cuda").manual_seed(1)
    W = torch.randn(r, d, device="cuda", generator=gen) * 0.02
    mom = torch.zeros(r, d, device="cuda")
    mask = torch.randint(0, 16, (r * d // m,), device="cuda", generator=gen, dtype=torch.uint8)
    keep = unpack_mask(mask, r, d, m)
    grad = torch.zeros(r, d, device="cuda")
    how = dict(beta=0.9, lr=0.01, weight_decay=0.1, scale=1.0)
    args = tb.muon_args(r=r, d=d, grad=grad.data_ptr(), g_dtype=tb.F32, momentum=mom.data_ptr(), w=W.data_ptr(), w_dtype=tb.F32, mask=mask.data_ptr(), nm_m=m, **how)
    side = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        g.capture_begin()
        tb.check(tb.muon_step(args, stream=torch.cuda.current_stream().cuda_stream))
        g.capture_end()
    torch.cuda.synchronize()
    for i in range(3):
        grad.copy_(gradient(r, d, "falling", seed=20 + i))
        want_w, want_m, o = step(W, grad, mom, keep, **how)
        before = W.double().abs()
        g.replay()
        torch.cuda.synchronize()
        assert_near(W, want_w, (before + 0.01 * o.abs()) * 2.0 ** -22, 0.01 * OFF * o.norm().item(), f"step {i}")
        assert_near(mom, want_m, want_m.abs() * 2.0 ** -22 + grad.double().abs() * 2.0 ** -22, 0.0, f"momentum {i}")


def test_two_streams_at_once(cuda):
    xs = [gradient(*s, "falling") for s in ((100, 400), (900, 500))]
    wants = [ortho(x) for x in xs]
    outs = [torch.empty(x.shape, device="cuda", dtype=torch.bfloat16) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    for _ in range(4):
        for x, o, s in zip(xs, outs, streams):
            r, d = x.shape
            tb.check(tb.orthogonalize(x.data_ptr(), tb.F32, d, r, d, o.data_ptr(), tb.BF16, d, stream=s.cuda_stream))
    torch.cuda.synchronize()
    for o, want in zip(outs, wants):
        assert_near(o, want, want.abs() * 2.0 ** -8, OFF * want.norm().item(), "beside another")
    status()


@pytest.mark.parametrize("tall", [False, True])
def test_more_than_31_bits_of_values(cuda, tall):
    """2.2e9 values: by way of the short side's 64 x 64 matrices, at the long side's ends."""
    k, D = 64, (1 << 25) + 11
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.empty((D, k) if tall else (k, D), device="cuda", dtype=torch.bfloat16).normal_(generator=g)
    (x[:, :9] if tall else x[:9]).mul_(30)
    got = run_ortho(x)
    long = x if tall else x.t()
    A = torch.zeros(k, k, device="cuda", dtype=torch.float64)
    for i in range(0, D, 1 << 20):
        part = long[i:i + (1 << 20)].double()
        A += part.t() @ part
    norm = A.trace().sqrt() + 1e-7
    A, Q, eye = A / norm ** 2, torch.eye(k, device="cuda", dtype=torch.float64), torch.eye(k, device="cuda", dtype=torch.float64)
    for _ in range(5):
        P = 3.4445 * eye - 4.7750 * A + 2.0315 * A @ A
        Q, A = P @ Q, P @ A @ P
    for rows in (slice(0, 2000), slice((1 << 25) - 500, D)):
        want = (long[rows].double() / norm) @ Q
        part = (got[rows] if tall else got[:, rows].t())
        assert_near(part, want, want.abs() * 2.0 ** -8, OFF * want.norm().item(), str(rows))
