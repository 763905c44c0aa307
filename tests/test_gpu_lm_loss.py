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


@pytest.mark.parametrize("n,d,vocab", [(40, 72, 500), (300, 72, 500)])  # in one pass over w, and by tiles
def test_left_out_tokens_reach_nothing(cuda, n, d, vocab):
    """Whatever a token that is left out holds: as if its row were zeros."""
    h, w, target, dloss, dlse = make(n, d, vocab, left=0.4, seed=2)
    out = (target < 0) | (target >= vocab)
    assert out.any() and not out.all()
    ref = reference(h, w, target, 0.0, dloss, dlse)
    h[out] = float("nan")
    h[torch.nonzero(out)[0]] = float("inf")
    dloss[out] = float("inf")
    dlse[out] = float("nan")
    dh, dw = torch.full((n, d), 3.0, device="cuda", dtype=BF), torch.full((vocab, d), 3.0, device="cuda", dtype=BF)
    loss, lse = call(h, w, target, 0.0, dloss, dlse, dh, dw, backward=True)
    for name, got in (("lse", lse), ("loss", loss), ("dh", dh), ("dw", dw)):
        assert_within(got, ref, name)
    assert (loss[out] == 0).all() and (lse[out] == 0).all() and (dh[out] == 0).all()


@pytest.mark.parametrize("n", [30, 400])
def test_all_tokens_left_out(cuda, n):
    h, w, target, dloss, _ = make(n, 64, 200)
    target[:] = -1
    target[::2] = 1 << 40
    dh, dw = torch.full((n, 64), 3.0, device="cuda", dtype=BF), torch.full((200, 64), 3.0, device="cuda", dtype=BF)
    loss, lse = call(h, w, target, 0.0, dloss, None, dh, dw, backward=True)
    for x in (loss, lse, dh, dw):
        assert (x == 0).all()
    status()


def test_no_tokens(cuda):
    w = torch.randn(50, 64, device="cuda").to(BF)
    buf = torch.full((51, 80), 3.0, device="cuda", dtype=BF)
    args = tb.lm_loss_args(n=0, d=64, vocab=50, h=None, ldh=64, w=w.data_ptr(), ldw=64, target=None, lse=None, dw=buf.data_ptr(), lddw=80)
    tb.check(tb.lm_loss_backward(args, stream=torch.cuda.current_stream().cuda_stream))
    assert (buf[:50, :64] == 0).all() and (buf[50:] == 3.0).all() and (buf[:, 64:] == 3.0).all()


@pytest.mark.parametrize("n", [20, 300])
def test_infinities_stay_with_their_token(cuda, n):
    d, vocab = 64, 300
    h, w, target, dloss, _ = make(n, d, vocab)
    ref = reference(h, w, target, 0.0, dloss)
    h[3, 5] = float("inf")
    h[7, 1] = float("nan")
    dloss[9] = float("inf")
    dh = torch.empty(n, d, device="cuda", dtype=BF)
    loss, lse = call(h, w, target, 0.0, dloss, None, dh, None, backward=True)
    fine = torch.ones(n, device="cuda", dtype=torch.bool)
    fine[[3, 7]] = False
    for name, got in (("lse", lse), ("loss", loss)):
        assert_within(got[fine], {k: v[fine] for k, v in ref.items() if k.startswith(name)}, name)
        assert not torch.isfinite(got[~fine]).any()
    fine[9] = False
    # (the unit that the tokens' factors share is the largest finite one, with or without token 9)
    assert_within(dh[fine], {k: v[fine] for k, v in ref.items() if k.startswith("dh")}, "dh")
    assert not torch.isfinite(dh[9]).all()


@pytest.mark.parametrize("n,d,vocab", [(33, 100, 257), (300, 264, 500)])
@pytest.mark.parametrize("which", ["dh", "dw"])
def test_one_gradient_in_rows_of_any_stride(cuda, n, d, vocab, which):
    h, w, target, dloss, _ = make(n, d, vocab, left=0.2)
    r = n if which == "dh" else vocab
    buf = torch.full((r * (d + 3) + 2,), 3.0, device="cuda", dtype=BF)
    out = torch.as_strided(buf, (r, d), (d + 3, 1), 1)  # rows that start on two bytes
    call(h, w, target, 0.0, dloss, None, backward=True, **{which: out})
    assert_within(out, reference(h, w, target, 0.0, dloss), which)
    out.fill_(3.0)
    assert (buf == 3.0).all()


@pytest.mark.parametrize("n", [60, 700])
@pytest.mark.parametrize("cap", [0.0, 5.0])
def test_gradients_against_differences(cuda, n, cap):
    """dh and dw along random directions against central differences of the loss in 64 bits."""
    d, vocab, eps = 96, 400, 1e-5
    h, w, target, dloss, dlse = make(n, d, vocab, left=0.2, seed=5)
    dh, dw = torch.empty(n, d, device="cuda", dtype=BF), torch.empty(vocab, d, device="cuda", dtype=BF)
    call(h, w, target, cap, dloss, dlse, dh, dw, backward=True)
    ref = reference(h, w, target, cap, dloss, dlse)
    kept = (target >= 0) & (target < vocab)

    def total(hh, ww):
        z = hh[kept] @ ww.t()
        z = cap * torch.tanh(z / cap) if cap else z
        lse = torch.logsumexp(z, 1)
        loss = lse - z.gather(1, target[kept][:, None])[:, 0]
        return (loss * dloss[kept].double() + lse * dlse[kept].double()).sum()

    for got, name, x in ((dh, "dh", h), (dw, "dw", w)):
        u = torch.randn(x.shape, device="cuda", dtype=torch.float64)
        moved = [(h.double() + s * eps * u, w.double()) if name == "dh" else (h.double(), w.double() + s * eps * u) for s in (1, -1)]
        slope = (total(*moved[0]) - total(*moved[1])) / (2 * eps)
        along = (got.double() * u).sum()
        # the values' bounds, and what differences leave: eps^2 of a third derivative of order one, 2^-50 / eps
        assert abs(along - slope) <= (ref[name + "_bound"] * u.abs()).sum() + 1e-8


@pytest.mark.parametrize("n", [48, 900])
def test_same_bits_again(cuda, n):
    h, w, target, dloss, dlse = make(n, 200, 3000, left=0.2)
    got = []
    for _ in range(3):
        dh, dw = torch.empty(n, 200, device="cuda", dtype=BF), torch.empty(3000, 200, device="cuda", dtype=BF)
        got.append((*call(h, w, target, 0.0, dloss, dlse, dh, dw, backward=True), dh, dw))
    for other in got[1:]:
        for x, y in zip(got[0], other):
            assert torch.equal(x, y)


@pytest.mark.parametrize("n", [5, 500])
def test_captured_and_replayed(cuda, n):
    """Two graphs of one call, replayed in turn with other tokens and targets."""
    d, vocab = 128, 700
    h, w, target, dloss, _ = make(n, d, vocab, left=0.3)
    graphs = []
    side = torch.cuda.Stream()
    for _ in range(2):
        dh, dw = torch.empty(n, d, device="cuda", dtype=BF), torch.empty(vocab, d, device="cuda", dtype=BF)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.stream(side):
            g.capture_begin()
            loss, lse = call(h, w, target, 0.0, dloss, None, dh, dw, backward=True)
            g.capture_end()
        graphs.append((g, loss, lse, dh, dw))
    torch.cuda.synchronize()
    for seed in range(4):
        h2, _, target2, dloss2, _ = make(n, d, vocab, left=0.1 * seed, seed=seed + 10)
        h.copy_(h2)
        target.copy_(target2)
        dloss.copy_(dloss2)
        ref = reference(h, w, target, 0.0, dloss)
        for g, loss, lse, dh, dw in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, loss, lse, dh, dw in graphs:
            for name, got in (("lse", lse), ("loss", loss), ("dh", dh), ("dw", dw)):
                assert_within(got, ref, name)


def test_two_streams_at_once(cuda):
    cases = [make(n, 256, 2000, left=0.2, seed=n) for n in (90, 600)]
    refs = [reference(c[0], c[1], c[2], 0.0, c[3]) for c in cases]
    outs = [(torch.empty(c[0].shape, device="cuda", dtype=BF), torch.empty(c[1].shape, device="cuda", dtype=BF)) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    results = []
    for _ in range(3):
        results = []
        for c, (dh, dw), s in zip(cases, outs, streams):
            with torch.cuda.stream(s):
                results.append(call(c[0], c[1], c[2], 0.0, c[3], None, dh, dw, backward=True))
    torch.cuda.synchronize()
    for ref, (dh, dw), (loss, lse) in zip(refs, outs, results):
        for name, got in (("lse", lse), ("loss", loss), ("dh", dh), ("dw", dw)):
            assert_within(got, ref, name)


def test_offsets_beyond_32_bits(cuda):
    """h's rows lie 2^31 bytes and more apart."""
    n, d, vocab = 4, 64, 300
    ld = 1 << 30
    buf = torch.empty(3 * ld + 128, device="cuda", dtype=BF)
    h, w, target, dloss, _ = make(n, d, vocab)
    far = torch.as_strided(buf, (n, d), (ld, 1))
    far.copy_(h)
    dh, dw = torch.empty(n, d, device="cuda", dtype=BF), torch.empty(vocab, d, device="cuda", dtype=BF)
    loss, lse = call(far, w, target, 0.0, dloss, None, dh, dw, backward=True)
    ref = reference(h, w, target, 0.0, dloss)
    for name, got in (("lse", lse), ("loss", loss), ("dh", dh), ("dw", dw)):
        assert_within(got, ref, name)


@pytest.mark.parametrize("n", [21, 333])
def test_gradient_in_the_tokens_place(cuda, n):
    h, w, target, dloss, dlse = make(n, 104, 600, left=0.3)
    ref = reference(h, w, target, 0.0, dloss, dlse)
    call(h, w, target, 0.0, dloss, dlse, h, None, backward=True)
    assert_within(h, ref, "dh")


@pytest.mark.parametrize("n", [21, 333])
@pytest.mark.parametrize("size,penalty", [(1e-20, 1e20), (0.0, 1.0), (1e30, 1.0), (1e-38, 0.0)])
def test_factors_of_any_size(cuda, n, size, penalty):
    """dloss and dlse far apart, or far from one."""
    h, w, target, dloss, dlse = make(n, 96, 500, left=0.2)
    dloss, dlse = dloss * size, dlse * penalty
    dh, dw = torch.empty(n, 96, device="cuda", dtype=BF), torch.empty(500, 96, device="cuda", dtype=BF)
    call(h, w, target, 0.0, dloss, dlse, dh, dw, backward=True)
    ref = reference(h, w, target, 0.0, dloss, dlse)
    for name, got in (("dh", dh), ("dw", dw)):
        # (a dloss 2^-133 below the unit, and results below FP32's smallest normal value, may be zero)
        ref[name + "_bound"] = ref[name + "_bound"] + 2.0 ** -126 + 2.0 ** -120 * max(float(dloss.abs().max()), float(dlse.abs().max()))
        assert_within(got, ref, name)


def test_more_than_31_bits_of_weights(cuda):
    """w and dw of 2.2e9 values: the last entries of the vocabulary, and all of them together in lse and dh."""
    n, d, vocab = 3, 4096, 530000
    g = torch.Generator(device="cuda").manual_seed(0)
    w = torch.empty(vocab, d, device="cuda", dtype=BF).normal_(generator=g).mul_(0.02)
    h = torch.randn(n, d, device="cuda", generator=g).to(BF)
    target = torch.tensor([0, vocab - 1, 524288], device="cuda")
    dloss = torch.ones(n, device="cuda")
    dh, dw = torch.empty(n, d, device="cuda", dtype=BF), torch.empty(vocab, d, device="cuda", dtype=BF)
    loss, lse = call(h, w, target, 0.0, dloss, None, dh, dw, backward=True)
    status()
    z = torch.cat([h.double() @ part.double().t() for part in w.split(20000)], 1)
    want = torch.logsumexp(z, 1)
    top = z.gather(1, target[:, None])[:, 0]
    # (bounds as in lm_loss_ref, with |h| . |w| at most 100 here)
    off = 100 * (6 * 2.0 ** -23 + 65 * 2.0 ** -24) + 2.0 ** -21 * 40
    assert ((lse.double() - want).abs() <= off).all() and ((loss.double() - want + top).abs() <= 2 * off).all()
    p = torch.exp(z - want[:, None])
    p.scatter_add_(1, target[:, None], torch.full((n, 1), -1.0, device="cuda", dtype=torch.float64))
    size = torch.exp(z - want[:, None])
    size.scatter_add_(1, target[:, None], torch.ones(n, 1, device="cuda", dtype=torch.float64))
    for rows in (slice(0, 300), slice(524288, 524600), slice(vocab - 300, vocab)):
        dw_want, terms = p[:, rows].t() @ h.double(), size[:, rows].t() @ h.double().abs()
        assert ((dw[rows].double() - dw_want).abs() <= dw_want.abs() * 2.0 ** -8 * 1.01 + terms * (2.0 ** -8 + 4 * off) + 2.0 ** -133).all()
    dh_want = sum(p[:, i:i + 20000] @ w[i:i + 20000].double() for i in range(0, vocab, 20000))
    terms = sum(size[:, i:i + 20000] @ w[i:i + 20000].double().abs() for i in range(0, vocab, 20000))
    assert ((dh.double() - dh_want).abs() <= dh_want.abs() * 2.0 ** -8 * 1.01 + terms * (2.0 ** -8 + 4 * off + vocab / 16 / 32 * 2.0 ** -23)).all()


def test_gradients_of_many_tokens_of_one_sign(cuda):
    """Sums over 200000 tokens whose terms all have one sign, which the tensor core's additions cut off."""
    n, d, vocab = 200000, 32, 64
    h = torch.full((n, d), 1.0, device="cuda", dtype=BF)
    h[:, ::2] = 0.75
    w = torch.zeros(vocab, d, device="cuda", dtype=BF)
    w[0] = 0.25
    target = torch.zeros(n, device="cuda", dtype=torch.int64)
    dloss = torch.full((n,), 1.0, device="cuda")
    dh, dw = torch.empty(n, d, device="cuda", dtype=BF), torch.empty(vocab, d, device="cuda", dtype=BF)
    call(h, w, target, 0.0, dloss, None, dh, dw, backward=True)
    z = h[:1].double() @ w.double().t()
    p = torch.softmax(z, 1)[0]
    p[0] -= 1.0
    want = n * p[:, None] * h[0].double()
    # G's rounding and dW's own, and 300 steps cut off at 2^-24 on average
    assert ((dw.double() - want).abs() <= want.abs() * (2.0 ** -8 + 2.0 ** -8 + 300 * 2.0 ** -23)).all()
