"""GPU: low-rank adapters beside a shared projection, against float64.

Bars.  A BF16 result is off by half a step, 2^-8 of its value, and by its sum:
every product of two BF16 values is exact and each of the K additions loses at
most 2^-23 of the sum of magnitudes; u and v, FP32 sums themselves, enter their
second product as two BF16 parts, 2^-16 of their magnitude (2^-9 of 2^-9, with
room for the parts' sum).  So |error| <= 2^-8 |y| + (K 2^-23 + 2^-16) * mag."""
import math

import pytest

import act8_ref as ref
from test_gpu_act8 import packed, rows

pytestmark = pytest.mark.gpu


def bf(torch, n, d, seed, scale=1.0):
    return rows(torch, n, d, torch.bfloat16, seed, ref.up(d, 8), scale, 0)


class Case:
    def __init__(self, torch, n, d, r, rank, na, who, seed=0):
        self.torch, self.n, self.d, self.r, self.rank, self.na = torch, n, d, r, rank, na
        self.w = bf(torch, r, d, seed + 1, 0.05)
        self.a = bf(torch, max(1, na) * rank, d, seed + 2, 1 / math.sqrt(d))
        self.b = bf(torch, max(1, na) * r, rank, seed + 3, 0.3)
        self.x, self.dy = bf(torch, n, d, seed + 4), bf(torch, n, r, seed + 5, 0.1)
        self.scale = torch.rand(max(1, na), device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)) + 0.5
        self.who = who.to(torch.int32).cuda().contiguous()
        self.y = torch.full((n + 1, r + 5), 3.0, device="cuda", dtype=torch.bfloat16)
        self.dx = torch.full((n + 1, d + 3), 3.0, device="cuda", dtype=torch.bfloat16)
        self.da = torch.full((max(1, na) * rank, self.a.stride(0)), 3.0, device="cuda", dtype=torch.bfloat16)
        self.db = torch.full((max(1, na) * r, self.b.stride(0)), 3.0, device="cuda", dtype=torch.bfloat16)
        self.ref = ref.Adapters(torch, self.w, self.a.reshape(-1, rank, d)[:na], self.b.reshape(-1, r, rank)[:na],
                                self.scale, self.who)

    def args(self, tb, **kw):
        a = dict(n=self.n, d=self.d, r=self.r, rank=self.rank, n_adapters=self.na, w=self.w.data_ptr(), ldw=self.w.stride(0),
                 a=self.a.data_ptr(), lda=self.a.stride(0), b=self.b.data_ptr(), ldb=self.b.stride(0),
                 scale=self.scale.data_ptr(), token_adapter=self.who.data_ptr(), x=self.x.data_ptr(), ldx=self.x.stride(0),
                 y=self.y.data_ptr(), ldy=self.y.stride(0), dy=self.dy.data_ptr(), lddy=self.dy.stride(0),
                 dx=self.dx.data_ptr(), lddx=self.dx.stride(0), da=self.da.data_ptr(), db=self.db.data_ptr())
        a.update(kw)
        return tb.adapter_args(**a)


def check(torch, got, want, mag, K):
    err = (got.double() - want).abs() - (2.0 ** -8 * want.abs() + (K * 2.0 ** -23 + 2.0 ** -16) * 1.01 * mag + 1e-40)
    assert float(err.max()) <= 0, float(err.max())


def who_of(torch, n, na, kind, seed=0):
    g = torch.Generator().manual_seed(seed)
    if kind == "mixed":
        return torch.randint(-1, max(1, na), (n,), generator=g)
    if kind == "none":
        return torch.full((n,), -1)
    if kind == "one":
        return torch.zeros(n, dtype=torch.int64)
    if kind == "wild":  # indexes that name no adapter
        return torch.tensor([-7, na, na + 5, 0, 2 ** 31 - 1, -2 ** 31])[torch.arange(n) % 6]
    return torch.div(torch.arange(n) * max(1, na), max(1, n), rounding_mode="floor")


SHAPES = [
    (1, 1, 1, 1, 1, "one"), (40, 1, 1, 1, 1, "one"), (1100, 3, 2, 1, 2, "mixed"), (1, 64, 64, 8, 1, "one"), (1, 4096, 1024, 16, 4, "mixed"), (3, 40, 24, 1, 2, "runs"), (8, 520, 136, 16, 8, "runs"),
    (17, 256, 264, 5, 3, "mixed"), (33, 136, 1000, 64, 2, "runs"), (64, 512, 256, 128, 3, "mixed"),
    (130, 384, 520, 33, 4, "runs"), (300, 264, 136, 16, 40, "mixed"), (257, 128, 256, 24, 2, "wild"),
    (520, 1024, 384, 32, 5, "runs"), (100, 77, 51, 8, 2, "none"), (90, 200, 72, 12, 0, "none"),
    (1100, 256, 640, 100, 3, "runs"), (1024, 96, 80, 16, 3, "mixed"), (1025, 96, 80, 16, 3, "mixed"),
    (2500, 264, 392, 64, 2, "mixed"), (3000, 128, 136, 8, 1, "one"), (1500, 72, 40, 128, 20, "mixed"),
    (2500, 2100, 2000, 16, 4, "mixed"), (5, 136, 200, 16, 0, "none"), (32, 264, 136, 16, 0, "none"),
    (2100, 136, 72, 24, 300, "mixed"),
    (1300, 64, 72, 16, 4, "none"), (2048, 72, 64, 40, 2, "wild")]


@pytest.mark.parametrize("n,d,r,rank,na,kind", SHAPES)
def test_forward(cuda, tblib, n, d, r, rank, na, kind):
    torch, tb = cuda, tblib
    c = Case(torch, n, d, r, rank, na, who_of(torch, n, na, kind))
    tb.check(tb.adapter_forward(c.args(tb)))
    torch.cuda.synchronize()
    tb.check(tb.lib().tb_gemm_status(None))
    check(torch, c.y[:n, :r], c.ref.forward(c.x), c.ref.forward(c.x, True), d + rank)
    assert bool((c.y[n:] == 3).all()) and bool((c.y[:, r:] == 3).all())


@pytest.mark.parametrize("n,d,r,rank,na,kind", [
    (16, 8200, 4104, 16, 3, "mixed"), (17, 8200, 4104, 16, 3, "mixed"), (32, 8192, 4096, 24, 3, "runs"), (32, 8192, 4104, 24, 3, "runs"), (32, 8192, 4104, 24, 8, "mixed"),
    (1, 8192, 136, 16, 0, "none"), (1, 8200, 136, 16, 0, "none"), (1, 8200, 136, 16, 1, "one"), (16, 9000, 4000, 8, 0, "none")])
def test_forward_of_few_tokens_on_both_sides_of_its_rule(cuda, tblib, n, d, r, rank, na, kind):
    """Few tokens of large projections, by the kernel of few tokens and by tiles."""
    torch, tb = cuda, tblib
    c = Case(torch, n, d, r, rank, na, who_of(torch, n, na, kind), 3)
    tb.check(tb.adapter_forward(c.args(tb)))
    torch.cuda.synchronize()
    tb.check(tb.lib().tb_gemm_status(None))
    check(torch, c.y[:n, :r], c.ref.forward(c.x), c.ref.forward(c.x, True), d + rank)
    assert bool((c.y[n:] == 3).all()) and bool((c.y[:, r:] == 3).all())


@pytest.mark.parametrize("n,d,r,rank,na,kind", SHAPES)
def test_backward(cuda, tblib, n, d, r, rank, na, kind):
    torch, tb = cuda, tblib
    c = Case(torch, n, d, r, rank, na, who_of(torch, n, na, kind), 10)
    ck = packed(torch, tb, c.x)
    tb.check(tb.adapter_backward(c.args(tb, x8=ck.s)))
    torch.cuda.synchronize()
    tb.check(tb.lib().tb_gemm_status(None))
    xh = ck.values(torch)
    dx, da, db = c.ref.backward(c.dy, xh)
    mx, ma, mb = c.ref.backward(c.dy, xh, True)
    check(torch, c.dx[:n, :d], dx, mx, r + rank)
    assert bool((c.dx[n:] == 3).all()) and bool((c.dx[:, d:] == 3).all())
    if na:
        check(torch, c.da[:, :d].reshape(na, rank, d), da, ma, n + r)
        check(torch, c.db[:, :rank].reshape(na, r, rank), db, mb, n + d)
        assert bool((c.da[:, d:] == 3).all()) and bool((c.db[:, rank:] == 3).all())


@pytest.mark.parametrize("n,d,r,rank,na,kind", [
    (512, 264, 392, 16, 15, "mixed"), (513, 264, 392, 16, 15, "mixed"), (128, 264, 392, 40, 16, "mixed"), (129, 264, 392, 40, 16, "mixed"),
    (512, 136, 72, 8, 1, "one"), (513, 136, 72, 8, 1, "one"), (1024, 72, 40, 3, 2049, "runs"), (1025, 72, 40, 3, 2049, "runs"),
    (600, 72, 40, 8, 2048, "mixed"), (129, 2000, 1000, 128, 20, "wild")])
def test_batches_on_both_sides_of_the_ordering_rule(cuda, tblib, n, d, r, rank, na, kind):
    """Tokens taken as they lie, and ordered by adapter first."""
    torch, tb = cuda, tblib
    c = Case(torch, n, d, r, rank, na, who_of(torch, n, na, kind, 1), 120)
    ck = packed(torch, tb, c.x)
    tb.check(tb.adapter_forward(c.args(tb)))
    tb.check(tb.adapter_backward(c.args(tb, x8=ck.s)))
    torch.cuda.synchronize()
    tb.check(tb.lib().tb_gemm_status(None))
    check(torch, c.y[:n, :r], c.ref.forward(c.x), c.ref.forward(c.x, True), d + rank)
    xh = ck.values(torch)
    want, mag = c.ref.backward(c.dy, xh), c.ref.backward(c.dy, xh, True)
    check(torch, c.dx[:n, :d], want[0], mag[0], r + rank)
    check(torch, c.da[:, :d].reshape(na, rank, d), want[1], mag[1], n + r)
    check(torch, c.db[:, :rank].reshape(na, r, rank), want[2], mag[2], n + d)
    assert bool((c.y[n:] == 3).all()) and bool((c.y[:, r:] == 3).all()) and bool((c.dx[n:] == 3).all()) and bool((c.dx[:, d:] == 3).all())


def test_gradients_against_differences(cuda, tblib):
    """The loss sum(dy * y(xhat)) in float64, differenced along random directions of x, A and B, against the kernels'
    gradients: y is linear in each of them alone, so a central difference is exact to float64 rounding, and the
    gradients' own errors are their entries' half steps, which add to at most 2^-8 sum |g||direction|, and their sums'."""
    torch, tb = cuda, tblib
    c = Case(torch, 70, 96, 80, 8, 3, who_of(torch, 70, 3, "mixed"), 20)
    ck = packed(torch, tb, c.x)
    tb.check(tb.adapter_backward(c.args(tb, x8=ck.s)))
    torch.cuda.synchronize()
    xh = ck.values(torch)
    g = torch.Generator(device="cuda").manual_seed(0)
    R = c.ref
    mags = R.backward(c.dy, xh, True)
    for name, grad, mag in (("x", c.dx[:70, :96], mags[0]), ("a", c.da[:, :96].reshape(3, 8, 96), mags[1]),
                            ("b", c.db[:, :8].reshape(3, 80, 8), mags[2])):
        v = torch.randn(grad.shape, device="cuda", generator=g, dtype=torch.float64)
        loss = []
        for h in (0.5, -0.5):
            m = ref.Adapters(torch, R.w, R.a + (h * v if name == "a" else 0), R.b + (h * v if name == "b" else 0), R.scale, R.who)
            loss.append(float((c.dy.double() * m.forward(xh + (h * v if name == "x" else 0))).sum()))
        want, got = loss[0] - loss[1], float((grad.double() * v).sum())
        bar = float((v.abs() * (2.0 ** -8 * grad.double().abs() + 2.0 ** -15 * mag)).sum())
        assert abs(want - got) <= bar


def test_values_of_other_tokens_stay_out(cuda, tblib):
    """NaN and infinities in one adapter, one token or an adapter's unused rows reach only what uses them."""
    torch, tb = cuda, tblib
    n, d, r, rank, na = 150, 200, 136, 16, 4
    who = who_of(torch, n, 3, "runs")  # adapter 3 is used by nobody
    c = Case(torch, n, d, r, rank, na, who, 30)
    c.a[3 * rank:] = math.nan
    c.b[3 * r:] = math.inf
    c.a[rank] = math.nan  # one row of adapter 1
    c.x[140] = math.inf   # a token of adapter 2
    tb.check(tb.adapter_forward(c.args(tb)))
    y = c.y[:n, :r]
    bad = (c.who == 1) | (torch.arange(n, device="cuda") == 140)
    assert bool(torch.isfinite(y[~bad]).all()) and not bool(torch.isfinite(y[bad]).any())
    c = Case(torch, n, d, r, rank, na, who, 30)
    ck = packed(torch, tb, c.x)
    c.dy[5] = math.nan    # a token of adapter 0
    c.b[3 * r:] = math.nan
    tb.check(tb.adapter_backward(c.args(tb, x8=ck.s)))
    dx, da, db = c.dx[:n, :d], c.da[:, :d].reshape(na, rank, d), c.db[:, :rank].reshape(na, r, rank)
    assert bool(torch.isnan(dx[5]).all()) and int(torch.isnan(dx).sum()) == d
    assert bool(torch.isnan(da[0]).all()) and bool(torch.isfinite(da[1:]).all())
    assert bool(torch.isnan(db[0]).all()) and bool(torch.isfinite(db[1:]).all())
    assert not bool(da[3].any()) and not bool(db[3].any())


@pytest.mark.parametrize("n", [20, 60, 150, 700, 1500])
def test_infinities_of_an_adapter_keep_their_sign(cuda, tblib, n):
    """An infinity in a row of b or a column of a gives its own tokens' results the infinity that the formula gives,
    and leaves every other result within its bar.  (A result with two is of their signs or NaN; b and a get one each.)"""
    torch, tb = cuda, tblib
    d, r, rank, na = 200, 392, 24, 3
    c = Case(torch, n, d, r, rank, na, who_of(torch, n, na, "mixed"), 80)
    want, mag = c.ref.forward(c.x), c.ref.forward(c.x, True)
    c.b[1 * r + 300, 7] = math.inf
    c.b[2 * r + 17, 20] = -math.inf
    tb.check(tb.adapter_forward(c.args(tb)))
    y = c.y[:n, :r]
    u = [c.scale[k].double() * (c.x.double() @ c.a[k * rank:(k + 1) * rank].double().t()) for k in range(na)]
    hit = torch.zeros(n, r, dtype=torch.bool, device="cuda")
    for k, o, j, sign in ((1, 300, 7, 1), (2, 17, 20, -1)):
        t = c.ref.tokens(k)
        hit[t, o] = True
        assert torch.equal(y[t, o].double(), sign * torch.sign(u[k][t, j]) * math.inf)
    check(torch, y[~hit], want[~hit], mag[~hit], d + rank)
    dx, mx = (c.ref.backward(c.dy, c.x.double(), m)[0] for m in (False, True))
    c = Case(torch, n, d, r, rank, na, who_of(torch, n, na, "mixed"), 80)
    c.a[1 * rank + 9, 130] = -math.inf
    tb.check(tb.adapter_backward(c.args(tb, da=None, db=None)))
    t = c.ref.tokens(1)
    v = c.dy.double()[t] @ c.b[r:2 * r, 9].double()
    got = c.dx[:n, :d]
    assert torch.equal(got[t, 130].double(), -torch.sign(v) * math.inf)
    hit = torch.zeros(n, d, dtype=torch.bool, device="cuda")
    hit[t, 130] = True
    check(torch, got[~hit], dx[~hit], mx[~hit], r + rank)


@pytest.mark.parametrize("n", [20, 150, 1500, 4000])
def test_infinities_of_dy_keep_their_sign_in_db(cuda, tblib, n):
    """An infinity in dy gives its feature's row of its adapter's db the infinities that the formula gives (a NaN where two
    of them cancel), and leaves every other entry within its bar."""
    torch, tb = cuda, tblib
    d, r, rank, na = 200, 136, 24, 2
    c = Case(torch, n, d, r, rank, na, torch.arange(n) % 2, 90)
    ck = packed(torch, tb, c.x)
    _, _, want = c.ref.backward(c.dy, ck.values(torch))
    _, _, mag = c.ref.backward(c.dy, ck.values(torch), True)
    u = [c.scale[k].double() * (ck.values(torch) @ c.a[k * rank:(k + 1) * rank].double().t()) for k in range(na)]
    hit = torch.zeros(na, r, dtype=torch.bool, device="cuda")
    for t, o, sign in ((0, 7, 1), (n - 1, 9, -1), (n - 2, 130, 1), (2, 130, 1)):
        c.dy[t, o] = sign * math.inf
        hit[t % 2, o] = True
    tb.check(tb.adapter_backward(c.args(tb, x8=ck.s)))
    db = c.db[:, :rank].reshape(na, r, rank)
    assert torch.equal(db[0, 7].double(), torch.sign(u[0][0]) * math.inf)
    assert torch.equal(db[1, 9].double(), -torch.sign(u[1][n - 1]) * math.inf)
    two, first = torch.sign(u[0][n - 2]), torch.sign(u[0][2])
    assert torch.equal(db[0, 130][two == first].double(), (two * math.inf)[two == first])
    assert bool(torch.isnan(db[0, 130][two != first]).all())
    check(torch, db[~hit], want[~hit], mag[~hit], n + d)


@pytest.mark.parametrize("n", [20, 60, 1500])
def test_infinities_of_token_and_adapter_at_once(cuda, tblib, n):
    """All values positive but for the infinities' signs: a token with one times a factor with one is an infinity, in y and dx."""
    torch, tb = cuda, tblib
    d, r, rank, na, t = 200, 392, 24, 3, 7
    c = Case(torch, n, d, r, rank, na, torch.arange(n) % na, 130)
    for m in (c.w, c.a, c.b, c.x, c.dy):
        m.abs_()
    c.w.clamp_(min=1e-3)
    c.x[t, 9], c.b[(t % na) * r + 300, 7] = math.inf, math.inf
    tb.check(tb.adapter_forward(c.args(tb)))
    y = c.y[:n, :r]
    own = c.who == t % na
    assert bool((y[t] == math.inf).all()) and bool((y[own, 300] == math.inf).all())
    assert int(torch.isinf(y).sum()) == r + int(own.sum()) - 1 and not bool(torch.isnan(y).any())
    c.b[(t % na) * r + 300, 7] = 0.5
    c.dy[t, 9], c.a[(t % na) * rank + 5, 130] = math.inf, -math.inf
    c.w[:, 130] = 0.0
    tb.check(tb.adapter_backward(c.args(tb, da=None, db=None)))
    dx = c.dx[:n, :d]
    assert bool((dx[own, 130][c.who[own] >= 0] == -math.inf).sum() == int(own.sum()) - 1) and bool(torch.isnan(dx[t, 130]))
    rest = torch.ones(d, dtype=torch.bool, device="cuda")
    rest[130] = False
    assert bool((dx[t, rest] == math.inf).all()) and int(torch.isinf(dx).sum()) == d - 1 + int(own.sum()) - 1


def test_products_of_an_adapter_without_numbers_cost_no_more(cuda, tblib):
    """One infinity in each factor, then an adapter of NaN: forward and input gradients take about the time that they take
    without, but for the adapter's own tokens (the bar is 4 times)."""
    torch, tb = cuda, tblib
    n, d, r, rank, na = 4000, 2048, 2048, 32, 8
    c = Case(torch, n, d, r, rank, na, who_of(torch, n, na, "runs"), 96)

    def time(f):
        times = []
        for _ in range(8):
            ev = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
            ev[0].record()
            tb.check(f())
            ev[1].record()
            torch.cuda.synchronize()
            times.append(ev[0].elapsed_time(ev[1]))
        return min(times)

    calls = (lambda: tb.adapter_forward(c.args(tb)), lambda: tb.adapter_backward(c.args(tb, da=None, db=None)))
    plain = [time(f) for f in calls]
    c.b[r + 9, 5] = c.a[rank + 5, 9] = math.inf
    assert all(time(f) <= 4 * p for f, p in zip(calls, plain))
    c.b[r:2 * r] = math.nan
    c.a[rank:2 * rank] = math.nan
    assert all(time(f) <= 4 * p for f, p in zip(calls, plain))


def test_gradients_of_rows_without_numbers_cost_no_more(cuda, tblib):
    """One infinity, one token of NaN: the factors' gradients take about the time that they take without (the bar is 4 times)."""
    torch, tb = cuda, tblib
    n, d, r = 4000, 2048, 2048
    c = Case(torch, n, d, r, 32, 2, who_of(torch, n, 2, "runs"), 95)
    ck = packed(torch, tb, c.x)

    def time():
        times = []
        for _ in range(8):
            ev = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
            ev[0].record()
            tb.check(tb.adapter_backward(c.args(tb, x8=ck.s, dx=None)))
            ev[1].record()
            torch.cuda.synchronize()
            times.append(ev[0].elapsed_time(ev[1]))
        return min(times)

    plain = time()
    c.dy[n - 5, 9] = math.inf
    assert time() <= 4 * plain and bool(torch.isinf(c.db[r + 9, :32]).all())
    c.dy[n - 700] = math.nan
    assert time() <= 4 * plain and bool(torch.isnan(c.db[r:, :32]).all())


def test_large_values_and_tokens_without_numbers(cuda, tblib):
    """u and v that round to an infinity in BF16 but are none count as what they are; tokens that are all NaN, and an
    adapter that is, cost no more time than others: the products' bounded waits do not run out."""
    torch, tb = cuda, tblib
    c = Case(torch, 200, 64, 72, 8, 2, who_of(torch, 200, 2, "one"), 85)
    c.w.zero_()
    c.a.zero_()
    c.b.zero_()
    c.scale.fill_(1.0)
    c.a[0, :2] = torch.tensor([1.0, 2.0 ** -8], device="cuda", dtype=torch.bfloat16)
    c.x.zero_()
    c.x[:, :2] = torch.finfo(torch.bfloat16).max  # u = max (1 + 2^-8), still an FP32 value
    c.b[:72, 0] = 2.0 ** -10
    tb.check(tb.adapter_forward(c.args(tb)))
    u = torch.finfo(torch.bfloat16).max * (1 + 2.0 ** -8)
    assert u < torch.finfo(torch.float32).max
    assert float((c.y[:200, :72].double() / (u * 2.0 ** -10) - 1).abs().max()) <= 2.0 ** -8 + 2.0 ** -16
    n, d, r = 4000, 2048, 2048
    c = Case(torch, n, d, r, 16, 3, who_of(torch, n, 3, "mixed"), 86)
    want, mag = c.ref.forward(c.x), c.ref.forward(c.x, True)
    c.b[r:2 * r] = math.nan
    tb.check(tb.adapter_forward(c.args(tb)))
    tb.check(tb.lib().tb_gemm_status(None))
    own = c.who == 1
    y = c.y[:n, :r]
    assert bool(torch.isnan(y[own]).all())
    check(torch, y[~own], want[~own], mag[~own], d + 16)
    c.x.fill_(math.nan)
    ev = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
    ev[0].record()
    tb.check(tb.adapter_forward(c.args(tb)))
    ev[1].record()
    tb.check(tb.lib().tb_gemm_status(None))
    assert bool(torch.isnan(y).all()) and ev[0].elapsed_time(ev[1]) < 1000.0


def test_outputs_may_be_left_out(cuda, tblib):
    torch, tb = cuda, tblib
    c = Case(torch, 40, 64, 72, 8, 2, who_of(torch, 40, 2, "runs"), 40)
    ck = packed(torch, tb, c.x)
    tb.check(tb.adapter_backward(c.args(tb, x8=ck.s)))
    whole = [t.clone() for t in (c.dx, c.da, c.db)]
    for t in (c.dx, c.da, c.db):
        t.fill_(3.0)
    tb.check(tb.adapter_backward(c.args(tb, da=None, db=None)))
    assert torch.equal(c.dx, whole[0]) and bool((c.da == 3).all())
    c.dx.fill_(3.0)
    tb.check(tb.adapter_backward(c.args(tb, x8=ck.s, dx=None, w=None)))
    assert torch.equal(c.da, whole[1]) and torch.equal(c.db, whole[2]) and bool((c.dx == 3).all())
    # no tokens: the gradients are zero
    empty = packed(torch, tb, c.x)
    empty.s.n = 0
    tb.check(tb.adapter_backward(c.args(tb, n=0, x8=empty.s, dy=None)))
    assert not bool(c.da[:, :64].any()) and not bool(c.db[:, :8].any())


def test_calls_repeat_bit_for_bit_and_under_graphs(cuda, tblib):
    torch, tb = cuda, tblib
    sets = []
    for i in range(2):
        c = Case(torch, 600, 264, 392, 24, 5, who_of(torch, 600, 5, "mixed", i), 50 + i)
        sets.append((c, packed(torch, tb, c.x)))

    def go(k, stream=None):
        c, ck = sets[k]
        tb.check(tb.adapter_forward(c.args(tb), stream=stream))
        tb.check(tb.adapter_backward(c.args(tb, x8=ck.s), stream=stream))

    def outs(k):
        c = sets[k][0]
        return [c.y, c.dx, c.da, c.db]

    want = []
    for k in (0, 1):
        go(k)
        torch.cuda.synchronize()
        want.append([t.clone() for t in outs(k)])
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for t in outs(0) + outs(1):
            t.fill_(3.0)
        torch.cuda.synchronize()
        for k in (0, 1):
            go(k, streams[k].cuda_stream)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for k in (0, 1) for a, b in zip(outs(k), want[k]))
    graphs = []
    for k in (0, 1):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            go(k, torch.cuda.current_stream().cuda_stream)
        graphs.append(g)
    for t in outs(0) + outs(1):
        t.fill_(3.0)
    for k in (0, 1, 1, 0):
        graphs[k].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for k in (0, 1) for a, b in zip(outs(k), want[k]))


def test_larger_batches_under_graphs_with_new_tokens(cuda, tblib):
    """Batches whose tokens are ordered by adapter, with shares of the gradients: two captured graphs, replayed on two
    streams at once with new rows and new adapters of the tokens, against single calls and the formula."""
    torch, tb = cuda, tblib
    n, d, r, rank, na = 2600, 264, 392, 40, 3
    cases, cks, graphs = [], [], []
    for i in range(2):
        c = Case(torch, n, d, r, rank, na, who_of(torch, n, na, "mixed", i), 100 + i)
        cases.append(c)
        cks.append(packed(torch, tb, c.x))

    def go(k, stream=None):
        c, ck = cases[k], cks[k]
        tb.check(tb.adapter_forward(c.args(tb), stream=stream))
        tb.check(tb.adapter_backward(c.args(tb, x8=ck.s), stream=stream))

    for k in (0, 1):
        go(k)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            go(k, torch.cuda.current_stream().cuda_stream)
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for t, kind in enumerate(("runs", "mixed", "none", "one")):
        for k, c in enumerate(cases):
            c.x.copy_(bf(torch, n, d, 110 + 2 * t + k))
            c.who.copy_(who_of(torch, n, na, kind, 9 + t + k).to(torch.int32))
            ck = packed(torch, tb, c.x)
            cks[k].codes.copy_(ck.codes)
            cks[k].exps.copy_(ck.exps)
            for o in (c.y, c.dx, c.da, c.db):
                o.fill_(3.0)
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for k, c in enumerate(cases):
            got = [o.clone() for o in (c.y, c.dx, c.da, c.db)]
            go(k)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, (c.y, c.dx, c.da, c.db)))
            check(torch, c.y[:n, :r], c.ref.forward(c.x), c.ref.forward(c.x, True), d + rank)
            want, mag = (c.ref.backward(c.dy, cks[k].values(torch), m) for m in (False, True))
            check(torch, c.da[:, :d].reshape(na, rank, d), want[1], mag[1], n + r)
            check(torch, c.db[:, :rank].reshape(na, r, rank), want[2], mag[2], n + d)


@pytest.mark.parametrize("n,na", [(1, 3), (5, 0), (20, 3), (32, 3)])
def test_few_tokens_under_graphs_and_on_two_streams(cuda, tblib, n, na):
    """The forward that starts while its down projection runs: captured, replayed with new tokens, two at once."""
    torch, tb = cuda, tblib
    cases = [Case(torch, n, 520, 392, 24, na, who_of(torch, n, na, "mixed", i), 70 + i) for i in range(2)]
    graphs = []
    for c in cases:
        tb.check(tb.adapter_forward(c.args(tb)))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c.x.mul_(1.0)
            tb.check(tb.adapter_forward(c.args(tb), stream=torch.cuda.current_stream().cuda_stream))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for i in range(4):
        for k, c in enumerate(cases):
            c.x.copy_(bf(torch, n, 520, 90 + 2 * i + k))
            c.y.fill_(3.0)
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for c in cases:
            check(torch, c.y[:n, :392], c.ref.forward(c.x), c.ref.forward(c.x, True), 520 + 24)
            assert bool((c.y[n:] == 3).all())


def test_calibration_step_with_adapters(cuda, tblib):
    """Forward with adapters, the checkpoint, the backward, and the shared projection's Fisher from the same tensors."""
    torch, tb = cuda, tblib
    n, d, r = 256, 256, 128
    c = Case(torch, n, d, r, 16, 2, who_of(torch, n, 2, "runs"), 60)
    ck = packed(torch, tb, c.x)
    tb.check(tb.adapter_forward(c.args(tb)))
    tb.check(tb.adapter_backward(c.args(tb, x8=ck.s)))
    F = torch.empty(r, d, device="cuda")
    sp = torch.tensor([[0, 128], [128, 256]], device="cuda")
    tb.check(tb.act8_fisher(ck.s, c.dy.data_ptr(), tb.BF16, c.dy.stride(0), r, sp.data_ptr(), 2, F.data_ptr()))
    w, m = torch.empty(r, d, device="cuda"), torch.empty(r * d // 4, device="cuda", dtype=torch.uint8)
    a = tb.prune_args(weights=c.w.contiguous().data_ptr(), w_dtype=tb.BF16, grads=None, g_dtype=tb.F32, S=0, N=r * d,
                      fisher_in=F.data_ptr(), fisher_steps_in=2, w_out=w.data_ptr(), mask_out=m.data_ptr())
    tb.check(tb.score_mask_pack(a))
    torch.cuda.synchronize()
    assert float((w == 0).float().mean()) >= 0.5 and bool(torch.isfinite(c.y[:n, :r]).all())


def test_offsets_beyond_32_bits(cuda, tblib):
    """270000 tokens of 8192 features, all but the first 50 and the last 300 zero: x, its codes and dx pass 2^31 values."""
    torch, tb = cuda, tblib
    n, d, r, rank, last = 270000, 8192, 64, 16, 300
    x = torch.zeros(n, d, device="cuda", dtype=torch.bfloat16)
    dy = torch.zeros(n, r, device="cuda", dtype=torch.bfloat16)
    for rows_of, cols, seed, scale in ((x, d, 1, 1.0), (dy, r, 3, 0.1)):
        rows_of[:50] = bf(torch, 50, cols, seed, scale)
        rows_of[n - last:] = bf(torch, last, cols, seed + 1, scale)
    who = torch.full((n,), -1)
    who[:50], who[n - last:] = 0, 1
    who = who.to(torch.int32).cuda()
    w, a, b = bf(torch, r, d, 5, 0.05), bf(torch, 2 * rank, d, 6, 0.01), bf(torch, 2 * r, rank, 7, 0.3)
    scale = torch.tensor([1.0, 0.5], device="cuda")
    ck = packed(torch, tb, x)
    b0 = (n - last) // 128 * 128
    q, e = ref.pack(torch, x[b0:])
    assert torch.equal(ck.codes[b0:], q) and torch.equal(ck.exps[b0 // 128:], e)
    dx = torch.full((n, d), 3.0, device="cuda", dtype=torch.bfloat16)
    tb.check(tb.act8_unpack(ck.s, dx.data_ptr(), tb.BF16, d))
    assert torch.equal(dx[b0:].double(), ref.values(torch, q, e)) and not bool(dx[1000:b0:997].any())
    y = torch.full((n, r), 3.0, device="cuda", dtype=torch.bfloat16)
    da, db = torch.empty_like(a), torch.empty_like(b)
    args = tb.adapter_args(n=n, d=d, r=r, rank=rank, n_adapters=2, w=w.data_ptr(), ldw=d, a=a.data_ptr(), lda=d, b=b.data_ptr(),
                           ldb=rank, scale=scale.data_ptr(), token_adapter=who.data_ptr(), x=x.data_ptr(), ldx=d, y=y.data_ptr(),
                           ldy=r, dy=dy.data_ptr(), lddy=r, x8=ck.s, dx=dx.data_ptr(), lddx=d, da=da.data_ptr(), db=db.data_ptr())
    tb.check(tb.adapter_forward(args))
    tb.check(tb.adapter_backward(args))
    G = torch.empty(r, d, device="cuda")
    sp = torch.tensor([[n - last, n]], device="cuda")
    tb.check(tb.act8_weight_grad(ck.s, dy.data_ptr(), tb.BF16, r, r, sp.data_ptr(), 1, G.data_ptr(), tb.F32))
    torch.cuda.synchronize()
    tb.check(tb.lib().tb_gemm_status(None))
    at = torch.cat([torch.arange(50), torch.arange(n - last, n)]).cuda()
    R = ref.Adapters(torch, w, a.reshape(2, rank, d), b.reshape(2, r, rank), scale, who[at])
    check(torch, y[at], R.forward(x[at]), R.forward(x[at], True), d + rank)
    assert not bool(y[50:n - last].any()) and not bool(dx[50:n - last:997].any())
    q0, e0 = ref.pack(torch, x[:128])
    xh = torch.cat([ref.values(torch, q0, e0)[:50], ref.values(torch, q, e)[n - last - b0:]])
    want, mag = R.backward(dy[at], xh), R.backward(dy[at], xh, True)
    check(torch, dx[at], want[0], mag[0], r + rank)
    check(torch, da.reshape(2, rank, d), want[1], mag[1], n + r)
    check(torch, db.reshape(2, r, rank), want[2], mag[2], n + d)
    g = dy[n - last:].double().t() @ xh[50:]
    assert float((G.double() - g).norm() / g.norm()) <= 2e-6
