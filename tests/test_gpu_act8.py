"""GPU: 8-bit activation checkpoints and what is computed from them, against the
float64 restatement in act8_ref.py.

Bars.  Codes, exponents and values read back are exact.  A sum of n products is
held to n * 2^-23 of the sum of its terms' magnitudes: every product is exact,
an FP32 addition (or the alignment of a product in a tensor-core step, which
truncates) loses at most 2^-23 of the largest partial sum, and no partial sum
exceeds that sum of magnitudes; FP32 and F16 dy have three and two parts, hence
three and two times the additions.  A BF16 result adds half a step, 2^-8 of the
value.  Beside that bound, which grows with n, the 2-norm error of FP32 results
stays below 2e-6: rounding errors of n terms add like sqrt(n), and both sides
of the ratio do, so it is a few times 2^-24 times the depth of one partial sum
(32 tensor-core steps) whatever n."""
import math

import pytest

import act8_ref as ref

pytestmark = pytest.mark.gpu


def rows(torch, n, d, dtype, seed, ld=None, scale=1.0, heavy=20.0):
    """[n][d] normal values with 1 % heavy columns, as a view of rows of stride ld."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(n, d, device="cuda", generator=g) * scale
    if heavy:
        x[:, torch.randperm(d, device="cuda", generator=g)[: max(1, d // 100)]] *= heavy
    buf = torch.full((max(1, n), ld or d), 7.0, device="cuda", dtype=dtype)
    buf[:n, :d] = x.to(dtype)
    return buf[:n, :d]


def code(tb, torch, dtype):
    return {torch.float32: tb.F32, torch.float16: tb.F16, torch.bfloat16: tb.BF16}[dtype]


class Checkpoint:
    def __init__(self, torch, tb, n, d, ldq=None, lde=None):
        self.n, self.d = n, d
        self.codes = torch.full((max(1, n), ldq or ref.up(d, 16)), 85, device="cuda", dtype=torch.int8)
        self.exps = torch.full((max(1, -(-n // 128)), lde or ref.up(d, 16)), 85, device="cuda", dtype=torch.uint8)
        self.s = tb.act8(n=n, d=d, codes=self.codes.data_ptr(), ldq=self.codes.stride(0), exps=self.exps.data_ptr(),
                         lde=self.exps.stride(0))

    def values(self, torch):
        return ref.values(torch, self.codes[: self.n, : self.d], self.exps[:, : self.d])


def packed(torch, tb, x, keep=None, **kw):
    n, d = x.shape
    c = Checkpoint(torch, tb, n, d, **kw)
    tb.check(tb.act8_pack(c.s, x.data_ptr(), code(tb, torch, x.dtype), x.stride(0),
                          keep=None if keep is None else keep.data_ptr()))
    return c


@pytest.mark.parametrize("n,d,dtype,ld", [
    (1, 1, "float32", None), (1, 4096, "bfloat16", None), (127, 129, "float16", 131), (128, 128, "float32", None),
    (129, 200, "bfloat16", 208), (300, 77, "bfloat16", 77), (1000, 515, "float32", 516), (257, 1024, "float16", 1024)])
def test_pack_and_unpack_are_exact(cuda, tblib, n, d, dtype, ld):
    torch, tb = cuda, tblib
    x = rows(torch, n, d, getattr(torch, dtype), n + d, ld)
    if n > 2:
        x[1].zero_()
        x[:, 0] = 0.0
        x[0, d // 2] = 1e-4 if dtype == "float16" else 1e-42  # subnormal in FP32
    c = packed(torch, tb, x, ldq=ref.up(d, 16) + 16, lde=ref.up(d, 16) + 32)
    q, e = ref.pack(torch, x)
    assert torch.equal(c.codes[:n, :d], q) and torch.equal(c.exps[:, :d], e)
    assert bool((c.codes[:, d:] == 85).all()) and bool((c.exps[:, d:] == 85).all())
    want = ref.values(torch, q, e)
    for out_t in (torch.float32, torch.bfloat16, torch.float16):
        out = torch.full((n + 1, d + 3), 9.0, device="cuda", dtype=out_t)
        tb.check(tb.act8_unpack(c.s, out.data_ptr(), code(tb, torch, out_t), d + 3))
        assert torch.equal(out[:n, :d], want.to(out_t))
        assert bool((out[n:] == 9).all()) and bool((out[:, d:] == 9).all())
    # half a step of a block's scale, and scales no larger than needed
    amax = x.double().abs().amax(0)
    assert bool(((want - x.double()).abs() <= amax / 126.9).all())


def test_pack_borders(cuda, tblib):
    """Largest values around the border where the exponent steps (127.5 codes), powers of two, the ends of FP32."""
    torch, tb = cuda, tblib
    vals = [127.0, 127.49, 127.5, 127.50001, 128.0, 1.0, 0.99609375, 0.9960937, 1.9921875, 1.9921874, 3.4028235e38,
            1.1754944e-38, 1e-45, 0.0, 2.0 ** -120, 2.0 ** -119]
    x = torch.zeros(3, len(vals), device="cuda")
    x[1] = torch.tensor(vals, device="cuda")
    x[2] = -x[1] / 3
    c = packed(torch, tb, x)
    q, e = ref.pack(torch, x)
    assert torch.equal(c.codes[:3, : len(vals)], q) and torch.equal(c.exps[:, : len(vals)], e)


def test_values_that_round_beyond_the_range_read_back_as_infinities(cuda, tblib):
    """A block that reaches 255 * 2^120 has steps of 2^122: from 254 * 2^120 on its values round to 2^128.  One below keeps
    all its values finite."""
    torch, tb = cuda, tblib
    x = torch.zeros(4, 3, device="cuda")
    x[:, 0] = torch.tensor([255 * 2.0 ** 120, -254 * 2.0 ** 120, 253.9 * 2.0 ** 120, 2.0 ** 121], device="cuda")
    x[:, 1] = torch.tensor([-254.9 * 2.0 ** 120, 254 * 2.0 ** 120, 2.0 ** 119, 0.0], device="cuda")
    x[:, 2] = torch.finfo(torch.bfloat16).min
    c = packed(torch, tb, x)
    assert c.exps[0, :3].tolist() == [249, 248, 249]
    for dt in (torch.float32, torch.bfloat16):
        out = torch.empty(4, 3, device="cuda", dtype=dt)
        tb.check(tb.act8_unpack(c.s, out.data_ptr(), code(tb, torch, dt), 3))
        assert out[:, 0].tolist() == [math.inf, -math.inf, 63 * 2.0 ** 122, 0.0]  # 2^121: half a step, to even
        assert out[:, 1].tolist() == [-127 * 2.0 ** 121, 127 * 2.0 ** 121, 0.0, 0.0]
        assert bool((out[:, 2] == -math.inf).all())


def test_padding_and_values_that_are_no_numbers(cuda, tblib):
    torch, tb = cuda, tblib
    n, d = 300, 40
    x = rows(torch, n, d, torch.float32, 5)
    keep = (torch.arange(n, device="cuda") % 100 < 70).to(torch.uint8)
    x[keep == 0] = math.nan
    x[99] = math.inf
    x[130, 3], x[140, 4], x[150, 5] = math.nan, math.inf, -math.inf
    keep[[130, 140, 150]] = 1
    c = packed(torch, tb, x, keep)
    q, e = ref.pack(torch, x, keep)
    assert torch.equal(c.codes[:n, :d], q) and torch.equal(c.exps[:, :d], e)
    out = torch.empty(n, d, device="cuda")
    tb.check(tb.act8_unpack(c.s, out.data_ptr(), tb.F32, d))
    assert bool((out[:128][keep[:128] == 0] == 0).all()) and bool(torch.isfinite(out[:128]).all())
    assert bool(torch.isnan(out[128:256, 3:6]).all()) and int(torch.isnan(out).sum()) == 3 * 128
    # every token padding: all codes zero
    c = packed(torch, tb, x, torch.zeros(n, device="cuda", dtype=torch.uint8))
    assert not bool(c.codes[:n, :d].any()) and bool((c.exps[:, :d] == 1).all())


PARTS = {"bfloat16": 1, "float16": 2, "float32": 3}


def pairs(torch, samples):
    return torch.tensor(samples, device="cuda", dtype=torch.int64).reshape(-1, 2)


def check_sums(torch, got, want, mag, terms, bf16=False):
    bar = terms * 2.0 ** -23 * mag + 1e-300
    if bf16:
        bar = bar * 1.01 + 2.0 ** -8 * want.abs() + 1e-40
    over = ((got.double() - want).abs() - bar).max().item()
    assert over <= 0, over
    if not bf16 and float(want.norm()) > 0:
        assert float((got.double() - want).norm() / want.norm()) <= 2e-6


@pytest.mark.parametrize("n,r,d,dy_t,g_t,samples", [
    (1, 1, 1, "float32", "float32", None), (5, 3, 7, "bfloat16", "float32", [(0, 5)]),
    (64, 128, 256, "bfloat16", "bfloat16", None), (130, 64, 130, "bfloat16", "float32", [(0, 64), (64, 130)]),
    (333, 257, 511, "bfloat16", "bfloat16", [(0, 1), (1, 64), (64, 64), (64, 333)]),
    (700, 129, 384, "float32", "float32", [(0, 127), (127, 500), (500, 700)]),
    (515, 200, 272, "float16", "float32", [(3, 130), (400, 512)]),
    (2000, 384, 640, "bfloat16", "bfloat16", [(0, 700), (650, 1400), (1400, 2000), (0, 2000), (0, 700)]),
    (4100, 256, 256, "bfloat16", "float32", None),
    (3000, 100, 203, "float32", "bfloat16", [(0, 1500), (1500, 3000)]), (6000, 264, 130, "float16", "float32", [(7, 5900), (0, 10), (3, 3)]),
    (256, 40, 1030, "float32", "bfloat16", [(-5, 100), (200, 999), (90, 20)]),
    (700, 1100, 264, "bfloat16", "float32", [(0, 1), (1, 64), (64, 64), (64, 333), (333, 700)]),
    (515, 600, 272, "float16", "bfloat16", [(3, 130), (400, 512)]), (333, 520, 100, "float32", "float32", [(5, 70), (70, 200), (0, 333)]),
    (5, 1000, 9, "bfloat16", "bfloat16", [(0, 3), (3, 5)]), (256, 1030, 72, "float32", "float32", [(-5, 128), (200, 999), (90, 20)]),
    # large enough that the values are written out first
    (1000, 1300, 2000, "float32", "float32", [(3, 130), (130, 131), (131, 400), (400, 400), (400, 999), (0, 1000)]),
    (3000, 1100, 2610, "bfloat16", "bfloat16", [(301 * i, 300 * i + 290 - 7 * i) for i in range(10)])])
def test_weight_grad(cuda, tblib, n, r, d, dy_t, g_t, samples):
    torch, tb = cuda, tblib
    c = packed(torch, tb, rows(torch, n, d, torch.float32, n))
    # a BF16 dy of odd stride goes through scratch, one of aligned rows does not
    dy = rows(torch, n, r, getattr(torch, dy_t), n + 1, ref.up(r, 8) + (1 if n in (5, 130) else 8), 1e-2, 0)
    S = len(samples) if samples else 1
    stride = r * d + 5
    out = torch.full((S, stride), 3.0, device="cuda", dtype=getattr(torch, g_t))
    sp = pairs(torch, samples) if samples else None
    tb.check(tb.act8_weight_grad(c.s, dy.data_ptr(), code(tb, torch, dy.dtype), dy.stride(0), r,
                                 sp.data_ptr() if samples else None, S, out.data_ptr(), code(tb, torch, out.dtype),
                                 g_stride=stride))
    torch.cuda.synchronize()
    tb.check(tb.lib().tb_gemm_status(None))
    assert bool((out[:, r * d:] == 3).all())
    for s, (G, A) in enumerate(ref.gradients(torch, dy, c.values(torch), samples or [(0, n)])):
        check_sums(torch, out[s, : r * d].view(r, d), G, A, n * PARTS[dy_t], g_t == "bfloat16")


@pytest.mark.parametrize("n,r,d,S", [(300, 130, 72, 3), (520, 300, 328, 2), (90, 33, 8, 4), (1000, 513, 264, 1), (64, 256, 1000, 2)])
@pytest.mark.parametrize("g_t", ["float32", "bfloat16"])
def test_weight_grad_densely_packed(cuda, tblib, n, r, d, S, g_t):
    """Samples one behind the other without gaps, rows that start on 16 bytes: the results that leave by TMA."""
    torch, tb = cuda, tblib
    c = packed(torch, tb, rows(torch, n, d, torch.float32, n))
    dy = rows(torch, n, r, torch.bfloat16, n + 1, ref.up(r, 8), 1e-2, 0)
    samples = [(i * n // S, (i + 1) * n // S) for i in range(S)]
    out = torch.full((S * r * d + 64,), 3.0, device="cuda", dtype=getattr(torch, g_t))
    tb.check(tb.act8_weight_grad(c.s, dy.data_ptr(), tb.BF16, dy.stride(0), r, pairs(torch, samples).data_ptr(), S,
                                 out.data_ptr(), code(tb, torch, out.dtype)))
    torch.cuda.synchronize()
    assert bool((out[S * r * d:] == 3).all())
    for s, (G, A) in enumerate(ref.gradients(torch, dy, c.values(torch), samples)):
        check_sums(torch, out[s * r * d:(s + 1) * r * d].view(r, d), G, A, n, g_t == "bfloat16")


@pytest.mark.parametrize("dy_t", ["float32", "bfloat16"])
def test_many_short_samples_on_many_tiles(cuda, tblib, dy_t):
    """Many units of a few slices for each pair of blocks, the stages' ring wrapping at every phase: right, and the same
    bits every time (gradients and Fisher)."""
    torch, tb = cuda, tblib
    n, r, d, S = 434, 1300, 1677, 10
    c = packed(torch, tb, rows(torch, n, d, torch.float32, 7))
    dy = rows(torch, n, r, getattr(torch, dy_t), 8, ref.up(r, 16), 1e-2, 0)
    samples = [(i * n // S, (i + 1) * n // S) for i in range(S)]
    sp = pairs(torch, samples)
    outs = []
    for _ in range(4):
        G, F = torch.empty(S, r, d, device="cuda"), torch.empty(r, d, device="cuda")
        tb.check(tb.act8_weight_grad(c.s, dy.data_ptr(), code(tb, torch, dy.dtype), dy.stride(0), r, sp.data_ptr(), S,
                                     G.data_ptr(), tb.F32))
        tb.check(tb.act8_fisher(c.s, dy.data_ptr(), code(tb, torch, dy.dtype), dy.stride(0), r, sp.data_ptr(), S, F.data_ptr()))
        outs.append((G, F))
    torch.cuda.synchronize()
    tb.check(tb.lib().tb_gemm_status(None))
    assert all(torch.equal(a, b) for o in outs[1:] for a, b in zip(o, outs[0]))
    ga = ref.gradients(torch, dy, c.values(torch), samples)
    for s, (G, A) in enumerate(ga):
        check_sums(torch, outs[0][0][s], G, A, 50 * PARTS[dy_t])
    want = ref.fisher(torch, [G for G, _ in ga], 0.01, 0.99)
    assert float((outs[0][1].double() - want).norm() / want.norm()) <= 4e-6


def test_weight_grad_leaves_other_tokens_out(cuda, tblib):
    """NaN and infinities in tokens of no sample reach no gradient; those of one sample stay in it."""
    torch, tb = cuda, tblib
    n, r, d = 400, 136, 200
    x = rows(torch, n, d, torch.float32, 1)
    x[384:] = math.nan
    c = packed(torch, tb, x)
    for dt in (torch.bfloat16, torch.float32):
        dy = rows(torch, n, r, dt, 2, 136, 1e-2, 0)
        dy[100:110] = math.inf
        dy[200, 5] = math.nan
        dy[300:310] = -math.inf
        samples = [(10, 100), (110, 201), (201, 300), (310, 384), (310, 390)]
        out = torch.empty(5, r, d, device="cuda")
        tb.check(tb.act8_weight_grad(c.s, dy.data_ptr(), code(tb, torch, dt), dy.stride(0), r,
                                     pairs(torch, samples).data_ptr(), 5, out.data_ptr(), tb.F32))
        fine = torch.isfinite(out)
        assert bool(fine[[0, 2, 3]].all()) and not bool(fine[4].any())
        assert not bool(fine[1, 5].any()) and bool(fine[1, :5].all()) and bool(fine[1, 6:].all())


@pytest.mark.parametrize("n,r,d,dy_t,S,first", [
    (60, 128, 128, "float32", 8, True), (600, 130, 70, "bfloat16", 3, False), (1, 5, 9, "bfloat16", 1, True),
    (900, 256, 640, "bfloat16", 7, True), (513, 384, 257, "float16", 4, False), (3000, 136, 264, "bfloat16", 2, True),
    (5000, 300, 515, "bfloat16", 3, False), (2600, 264, 136, "float32", 4, True), (1025, 72, 520, "bfloat16", 1, False),
    (1024, 72, 520, "bfloat16", 1, True), (4000, 520, 300, "float16", 2, False)])
def test_fisher(cuda, tblib, n, r, d, dy_t, S, first):
    """The EMA of the float64 gradients: each g is within its sum's bar, a square doubles that, and each step rounds four times."""
    torch, tb = cuda, tblib
    c = packed(torch, tb, rows(torch, n, d, torch.float32, n, heavy=0))
    dy = rows(torch, n, r, getattr(torch, dy_t), n + 1, ref.up(r, 8), 1e-2, 0)
    cuts = sorted(torch.randint(0, n + 1, (S - 1,), generator=torch.Generator().manual_seed(n)).tolist())
    samples = list(zip([0] + cuts, cuts + [n]))
    F0 = torch.rand(r, d, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    F = F0.clone() if not first else torch.full((r, d), math.nan, device="cuda")
    tb.check(tb.act8_fisher(c.s, dy.data_ptr(), code(tb, torch, dy.dtype), dy.stride(0), r, pairs(torch, samples).data_ptr(),
                            S, F.data_ptr(), alpha=0.01, beta=0.99, first_step=first))
    torch.cuda.synchronize()
    ga = ref.gradients(torch, dy, c.values(torch), samples)
    alpha, beta = 0.01, 0.99
    want = ref.fisher(torch, [G for G, _ in ga], alpha, beta, None if first else F0.double())
    slack = n * PARTS[dy_t] * 2.0 ** -23
    worst = ref.fisher(torch, [G.abs() + slack * A for G, A in ga], alpha, beta, None if first else F0.double())
    bar = (worst - want) + 6 * S * 2.0 ** -24 * worst + 1e-40  # four roundings and the two factors' own
    assert float(((F.double() - want).abs() - bar).max()) <= 0
    assert float((F.double() - want).norm() / want.norm()) <= 4e-6


@pytest.mark.parametrize("n", [500, 513, 1000, 1024])
@pytest.mark.parametrize("d", [256, 512])
def test_fisher_of_terms_of_one_sign(cuda, tblib, n, d):
    """The tensor core cuts its sums off, which terms of one sign do not even out.  Fisher's g are the very sums that the
    gradients are, groups of 512 tokens (32 steps) added in FP32: a step cuts off half of 2^-23 of the sum so far on
    average, and those are half the group's on average, so g loses at most 32 2^-25 of itself, and a rounding.  (74 and
    148 tiles, so that neither call shares a sum out; with 512 features the values are written out first.)"""
    torch, tb = cuda, tblib
    r = 74 * 256
    c = packed(torch, tb, rows(torch, n, d, torch.float32, 1, heavy=0).abs())
    dy = rows(torch, n, r, torch.bfloat16, 2, r, 1e-2, 0).abs()
    F, G = torch.empty(r, d, device="cuda"), torch.empty(r, d, device="cuda")
    tb.check(tb.act8_fisher(c.s, dy.data_ptr(), tb.BF16, r, r, None, 1, F.data_ptr(), alpha=1.0))
    tb.check(tb.act8_weight_grad(c.s, dy.data_ptr(), tb.BF16, r, r, None, 1, G.data_ptr(), tb.F32))
    assert torch.equal(F, G * G)
    want = dy.double().t() @ c.values(torch)
    assert float((G.double() - want).norm() / want.norm()) <= 32 * 2.0 ** -25 + 2.0 ** -24


def test_fisher_equals_its_steps(cuda, tblib):
    """One fused call and tb_fisher_ema_step over the FP32 gradients of the same call's family agree to rounding of g."""
    torch, tb = cuda, tblib
    n, r, d, S = 500, 256, 384, 5
    c = packed(torch, tb, rows(torch, n, d, torch.float32, 4))
    dy = rows(torch, n, r, torch.bfloat16, 5, 256, 1e-2, 0)
    sp = pairs(torch, [(i * 100, i * 100 + 100) for i in range(S)])
    G = torch.empty(S, r, d, device="cuda")
    tb.check(tb.act8_weight_grad(c.s, dy.data_ptr(), tb.BF16, 256, r, sp.data_ptr(), S, G.data_ptr(), tb.F32))
    F, F2 = torch.empty(r, d, device="cuda"), torch.zeros(r, d, device="cuda")
    f32 = lambda v: float(torch.tensor(v, dtype=torch.float32))  # what the step's float arguments hold
    tb.check(tb.act8_fisher(c.s, dy.data_ptr(), tb.BF16, 256, r, sp.data_ptr(), S, F.data_ptr(), alpha=f32(0.01),
                            beta=f32(0.99)))
    for s in range(S):
        tb.check(tb.lib().tb_fisher_ema_step(F2.data_ptr(), G[s].data_ptr(), tb.F32, r * d, 0.01, 0.99, int(s == 0), None))
    assert float((F - F2).norm() / F2.norm()) <= 1e-6


@pytest.mark.parametrize("n,d,acc", [(1, 1, False), (64, 128, False), (130, 200, True), (1000, 640, False),
                                     (777, 515, True), (0, 96, False), (0, 96, True), (4096, 256, False), (300, 1100, True),
                                     (5000, 300, True), (9000, 130, False), (4000, 2900, True), (4000, 2899, False)])
def test_hessian(cuda, tblib, n, d, acc):
    torch, tb = cuda, tblib
    x = rows(torch, n, d, torch.float32, n + d)
    c = packed(torch, tb, x) if n else Checkpoint(torch, tb, 0, d)
    H = rows(torch, d, d, torch.float32, 9, heavy=0).contiguous()
    H0 = H.clone()
    scale = 1.0 / max(1, n)
    tb.check(tb.act8_hessian(c.s, scale, H.data_ptr(), accumulate=acc))
    torch.cuda.synchronize()
    tb.check(tb.lib().tb_gemm_status(None))
    t = torch.arange(d, device="cuda") // 128
    lower = t[:, None] >= t[None]
    assert torch.equal(H[~lower], H0[~lower])
    xh = c.values(torch) if n else torch.zeros(0, d, device="cuda", dtype=torch.float64)
    s32 = float(torch.tensor(scale, dtype=torch.float32))
    want = s32 * (xh.t() @ xh) + (H0.double() if acc else 0)
    mag = s32 * (xh.abs().t() @ xh.abs()) + (H0.double().abs() if acc else 0)
    err = (H.double() - want).abs() - (n + 3) * 2.0 ** -23 * mag
    assert float(err[lower].max()) <= 0
    if not acc and n:
        assert float((H.double() - want)[lower].norm() / want[lower].norm()) <= 1e-6


def test_hessian_of_a_block_without_numbers(cuda, tblib):
    torch, tb = cuda, tblib
    x = rows(torch, 200, 150, torch.float32, 3)
    x[150, 7] = math.inf
    c = packed(torch, tb, x)
    H = torch.zeros(150, 150, device="cuda")
    tb.check(tb.act8_hessian(c.s, 1.0, H.data_ptr()))
    t = torch.arange(150, device="cuda")
    hit = ((t[:, None] == 7) | (t[None] == 7)) & (t[:, None] // 128 >= t[None] // 128)
    assert bool(torch.isnan(H[hit]).all()) and bool(torch.isfinite(H[~hit]).all())


def test_hessian_matches_the_bf16_entry(cuda, tblib):
    """xhat is exact in BF16: tb_obs_hessian of the values read back gives the same matrix to FP32 rounding."""
    torch, tb = cuda, tblib
    n, d = 640, 512
    c = packed(torch, tb, rows(torch, n, d, torch.float32, 12))
    H, H2 = torch.zeros(d, d, device="cuda"), torch.zeros(d, d, device="cuda")
    xt = c.values(torch).t().contiguous().bfloat16()
    tb.check(tb.lib().tb_obs_hessian(xt.data_ptr(), d, n, H2.data_ptr(), None))
    tb.check(tb.act8_hessian(c.s, 1.0 / n, H.data_ptr()))
    torch.cuda.synchronize()
    assert float((H - H2).norm() / H2.norm()) <= 1e-6


def test_two_streams_and_two_graphs(cuda, tblib):
    """Calls on two streams at once, and two captured graphs replayed in turn with changed inputs, give what single calls give."""
    torch, tb = cuda, tblib
    n, r, d = 700, 264, 520
    sets = []
    for i in range(2):
        c = packed(torch, tb, rows(torch, n, d, torch.float32, 20 + i))
        dy = rows(torch, n, r, torch.float32, 30 + i, 264, 1e-2, 0)  # FP32: takes scratch
        sp = pairs(torch, [(0, 300 + i), (300 + i, n)])
        out = [torch.empty(2, r, d, device="cuda"), torch.empty(r, d, device="cuda"), torch.zeros(d, d, device="cuda")]
        sets.append((c, dy, sp, out))

    def go(k, stream):
        c, dy, sp, (G, F, H) = sets[k]
        tb.check(tb.act8_weight_grad(c.s, dy.data_ptr(), tb.F32, 264, r, sp.data_ptr(), 2, G.data_ptr(), tb.F32, stream=stream))
        tb.check(tb.act8_fisher(c.s, dy.data_ptr(), tb.F32, 264, r, sp.data_ptr(), 2, F.data_ptr(), stream=stream))
        tb.check(tb.act8_hessian(c.s, 1.0, H.data_ptr(), stream=stream))

    def single(k):
        go(k, None)
        torch.cuda.synchronize()
        return [t.clone() for t in sets[k][3]]

    want = [single(0), single(1)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for t in sets[0][3] + sets[1][3]:
            t.fill_(-1.0)
        torch.cuda.synchronize()
        for k in (0, 1):
            go(k, streams[k].cuda_stream)
        torch.cuda.synchronize()
        for k in (0, 1):
            low = [torch.tril(a) for a in sets[k][3][2:]], [torch.tril(a) for a in want[k][2:]]
            assert all(torch.equal(a, b) for a, b in zip(sets[k][3][:2] + low[0], want[k][:2] + low[1]))
    graphs = []
    for k in (0, 1):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            go(k, torch.cuda.current_stream().cuda_stream)
        graphs.append(g)
    for t in sets[0][3] + sets[1][3]:
        t.fill_(-1.0)
    for k in (0, 1, 0, 1):
        graphs[k].replay()
    torch.cuda.synchronize()
    for k in (0, 1):
        assert all(torch.equal(a, b) for a, b in zip(sets[k][3][:2], want[k][:2]))
    sets[0][2].copy_(pairs(torch, [(0, 1), (1, 1)]))  # new sample bounds under the captured graph
    graphs[0].replay()
    torch.cuda.synchronize()
    assert not bool(sets[0][3][0][1].any()) and not torch.equal(sets[0][3][0][0], want[0][0][0])


def test_calibration_end_to_end(cuda, tblib):
    """A layer's calibration from one checkpoint: the Fisher state scored and masked by the fused pass equals the pass
    over the materialised gradients' own EMA, and the Hessian prunes the layer."""
    import ctypes as C
    torch, tb = cuda, tblib
    n, r, d, S = 512, 256, 512, 4
    c = packed(torch, tb, rows(torch, n, d, torch.bfloat16, 40))
    dy = rows(torch, n, r, torch.bfloat16, 41, 256, 1e-2, 0)
    sp = pairs(torch, [(i * 128, i * 128 + 128) for i in range(S)])
    W = rows(torch, r, d, torch.float32, 42, scale=0.02, heavy=0).contiguous()
    F = torch.empty(r, d, device="cuda")
    tb.check(tb.act8_fisher(c.s, dy.data_ptr(), tb.BF16, 256, r, sp.data_ptr(), S, F.data_ptr()))
    G = torch.empty(S, r, d, device="cuda")
    tb.check(tb.act8_weight_grad(c.s, dy.data_ptr(), tb.BF16, 256, r, sp.data_ptr(), S, G.data_ptr(), tb.F32))
    outs = []
    for kw in (dict(grads=None, S=0, fisher_in=F.data_ptr(), fisher_steps_in=S), dict(grads=G.data_ptr(), S=S)):
        w, m = torch.empty(r, d, device="cuda"), torch.empty(r * d // 4, device="cuda", dtype=torch.uint8)
        a = tb.prune_args(weights=W.data_ptr(), w_dtype=tb.F32, g_dtype=tb.F32, N=r * d, w_out=w.data_ptr(),
                          mask_out=m.data_ptr(), **kw)
        tb.check(tb.score_mask_pack(a))
        outs.append((w, m))
    torch.cuda.synchronize()
    assert float((outs[0][1] != outs[1][1]).float().mean()) <= 1e-3  # near ties only: F differs by rounding
    H = torch.zeros(d, d, device="cuda")
    tb.check(tb.act8_hessian(c.s, 1.0 / n, H.data_ptr()))
    mask = torch.empty(r * d // 4, device="cuda", dtype=torch.uint8)
    tb.check(tb.lib().tb_obs_sparsegpt(W.data_ptr(), r, d, H.data_ptr(), 0.01, 2, 4, mask.data_ptr(), None, None))
    assert float((W == 0).float().mean()) == 0.5


def test_corners_of_the_state(cuda, tblib):
    """No tokens added to H leave it, subnormals too; a first step does not read F, whatever beta's powers."""
    torch, tb = cuda, tblib
    H = torch.full((40, 40), 1e-40, device="cuda")
    H[3, 4] = math.nan
    before = H.clone()
    ck = packed(torch, tb, rows(torch, 4, 40, torch.float32, 0))
    ck.s.n = 0
    tb.check(tb.act8_hessian(ck.s, 1.0, H.data_ptr(), accumulate=True))
    torch.cuda.synchronize()
    assert torch.equal(H.view(torch.int32), before.view(torch.int32))
    ck = packed(torch, tb, rows(torch, 150, 24, torch.float32, 1))
    dy = rows(torch, 150, 16, torch.bfloat16, 2, 16, 1e-3)
    sp = torch.tensor([[i, i + 1] for i in range(150)], device="cuda")
    for beta in (0.0, 2.0):
        F = torch.full((16, 24), math.nan, device="cuda")
        S = 150 if beta == 0.0 else 128  # (beta^S alone is beyond FP32)
        tb.check(tb.act8_fisher(ck.s, dy.data_ptr(), tb.BF16, 16, 16, sp.data_ptr(), S, F.data_ptr(), alpha=0.5, beta=beta))
        want = torch.zeros(16, 24, device="cuda", dtype=torch.float64)
        xh = ck.values(torch)
        for s in range(S):
            g = torch.outer(dy[s].double(), xh[s])
            want = 0.5 * g * g if s == 0 else beta * want + 0.5 * (1 - beta) * g * g
        # terms of both signs (1 - beta = -1): S additions and a few roundings of each term, of their magnitudes
        mag = torch.zeros_like(want)
        for s in range(S):
            g = torch.outer(dy[s].double(), xh[s])
            mag = 0.5 * g * g if s == 0 else beta * mag + 0.5 * abs(1 - beta) * g * g
        assert bool(((F.double() - want).abs() <= (S + 8) * 2.0 ** -23 * mag + 1e-38).all())


@pytest.mark.parametrize("n,r,d,S,first", [(40, 60, 52, 8, True), (700, 264, 300, 5, False), (3000, 200, 136, 2, False),
                                           (900, 2600, 2600, 6, True), (1500, 2600, 2304, 3, False)])
def test_fisher_of_few_tiles_and_of_last_waves(cuda, tblib, n, r, d, S, first):
    """Tiles whose samples are shared out (all of few, the last ones of 110 or 90), long samples among them."""
    torch, tb = cuda, tblib
    ck = packed(torch, tb, rows(torch, n, d, torch.float32, 7))
    dy = rows(torch, n, r, torch.bfloat16, 8, ref.up(r, 8), 0.1)
    cuts = [0] + [n * (i + 1) * (i + 2) // (S * (S + 1)) for i in range(S)]
    sp = torch.tensor([[a, b] for a, b in zip(cuts, cuts[1:])], device="cuda")
    F = torch.rand(r, d, device="cuda")
    old = F.double()
    tb.check(tb.act8_fisher(ck.s, dy.data_ptr(), tb.BF16, dy.stride(0), r, sp.data_ptr(), S, F.data_ptr(), first_step=first))
    again = old.float()
    tb.check(tb.act8_fisher(ck.s, dy.data_ptr(), tb.BF16, dy.stride(0), r, sp.data_ptr(), S, again.data_ptr(), first_step=first))
    torch.cuda.synchronize()
    tb.check(tb.lib().tb_gemm_status(None))
    xh = ck.values(torch)
    want, bar = (None, torch.zeros_like(old)) if first else (old, old * 0.0)
    for a, b in sp.tolist():
        g, m = dy[a:b].double().t() @ xh[a:b], dy[a:b].double().abs().t() @ xh[a:b].abs()
        e = (b - a) * 2.0 ** -23 * m
        w = 0.01 if want is None else 0.01 * 0.01
        bar = 0.99 * bar + w * (2 * m * e + e * e)
        want = 0.01 * g * g if want is None else 0.99 * want + w * g * g
    bar = bar + (2 * S + 6) * 2.0 ** -23 * want  # the state's own multiplications and additions, at most
    assert bool(((F.double() - want).abs() <= bar * 1.01 + 1e-40).all())
    assert float((F.double() - want).norm() / want.norm()) <= 2e-6
    assert torch.equal(F, again)


def test_a_cut_slice_behind_seconds_of_whole_ones(cuda, tblib):
    """65534 samples of 128 whole slices, then one that ends inside a slice: what cuts that slice waits for all the others,
    several seconds, longer than a bounded wait for one slice lasts.  74 tiles, so that no sample is shared out, and
    enough rows that the values are written out first.

    All samples but the last have one gradient g, so the state is alpha (c g^2 + (1 - beta) g_last^2) with c = beta (1 -
    beta) (1 + beta + ...) + beta^(S-1), whose sum is beta up to terms below 1e-280.  The additions' roundings: each is 2^-24
    of the state so far, and those are F beta^(S-j), which add to F / (1 - beta) = 100 F."""
    torch, tb = cuda, tblib
    n, r, d, S, whole = 65536, 74 * 256, 256, 65535, 128 * 64
    ck = packed(torch, tb, rows(torch, n, d, torch.float32, 50, heavy=0))
    dy = rows(torch, n, r, torch.bfloat16, 51, r, 0.1, 0)
    sp = torch.tensor([[0, whole]], device="cuda").repeat(S, 1)
    sp[S - 1, 1] = whole + 37
    F = torch.full((r, d), math.nan, device="cuda")
    tb.check(tb.act8_fisher(ck.s, dy.data_ptr(), tb.BF16, dy.stride(0), r, sp.data_ptr(), S, F.data_ptr()))
    torch.cuda.synchronize()
    tb.check(tb.lib().tb_gemm_status(None))
    xh, part = ck.values(torch), dy[:whole + 37].double()
    g, last = part[:whole].t() @ xh[:whole], part.t() @ xh[:whole + 37]
    mag = part.abs().t() @ xh[:whole + 37].abs()
    want = 0.01 * (0.99 * g * g + 0.01 * last * last)
    e = whole * 2.0 ** -23 * mag
    bar = 0.01 * (2 * mag * e + e * e) + (100 + 8) * 2.0 ** -24 * want
    assert bool(((F.double() - want).abs() <= bar).all())
    assert float((F.double() - want).norm() / want.norm()) <= 2e-5  # 100 2^-24, and twice g's own 2e-6


@pytest.mark.parametrize("n,r,d,S", [(2100, 2600, 2600, 1), (1100, 500, 1300, 9)])
@pytest.mark.parametrize("g_t", ["float32", "bfloat16"])
def test_gradients_of_last_waves(cuda, tblib, n, r, d, S, g_t):
    """121 and 108 units: those behind the first wave have their K shared out, rows on 16 bytes or not."""
    torch, tb = cuda, tblib
    ck = packed(torch, tb, rows(torch, n, d, torch.float32, 9))
    dy = rows(torch, n, r, torch.bfloat16, 10, ref.up(r, 8), 0.1)
    sp = torch.tensor([[n * i // S, n * (i + 1) // S] for i in range(S)], device="cuda")
    dt = getattr(torch, g_t)
    for pad in (0, 1):
        G = torch.full((S, r * d + pad), 3.0, device="cuda", dtype=dt)
        tb.check(tb.act8_weight_grad(ck.s, dy.data_ptr(), tb.BF16, dy.stride(0), r, sp.data_ptr(), S, G.data_ptr(), code(tb, torch, dt),
                                     g_stride=r * d + pad))
        torch.cuda.synchronize()
        tb.check(tb.lib().tb_gemm_status(None))
        xh = ck.values(torch)
        for s, (a, b) in enumerate(sp.tolist()):
            g, m = dy[a:b].double().t() @ xh[a:b], dy[a:b].double().abs().t() @ xh[a:b].abs()
            half = 2.0 ** -8 if g_t == "bfloat16" else 0.0
            got = G[s, :r * d].view(r, d).double()
            assert bool(((got - g).abs() <= half * g.abs() + (b - a) * 2.0 ** -23 * 1.01 * m + 1e-40).all())
        assert pad == 0 or bool((G[:, r * d] == 3).all())


@pytest.mark.parametrize("dy_t", ["float32", "bfloat16"])
@pytest.mark.parametrize("d", [200, 10000])
def test_samples_of_many_rows_leave_other_tokens_out(cuda, tblib, dy_t, d):
    """NaN before, between and behind the samples reaches none; with 10000 features the values are written out first."""
    torch, tb = cuda, tblib
    n, r = 600, 1100
    samples = [(3, 130), (131, 200), (210, 211), (220, 539)]
    x, dy = rows(torch, n, d, torch.float32, 30), rows(torch, n, r, getattr(torch, dy_t), 31, ref.up(r, 8), 0.1, 0)
    inside = torch.zeros(n, dtype=torch.bool, device="cuda")
    for a, b in samples:
        inside[a:b] = True
    dy[~inside] = math.nan
    x[560:] = math.nan  # blocks 0 .. 3 stay numbers
    x[512:560] = 0.0
    ck = packed(torch, tb, x, (torch.arange(n, device="cuda") < 560).to(torch.uint8))
    sp = pairs(torch, samples)
    G = torch.full((4, r, d), 3.0, device="cuda")
    tb.check(tb.act8_weight_grad(ck.s, dy.data_ptr(), code(tb, torch, dy.dtype), dy.stride(0), r, sp.data_ptr(), 4, G.data_ptr(), tb.F32))
    F = torch.full((r, d), math.nan, device="cuda")
    tb.check(tb.act8_fisher(ck.s, dy.data_ptr(), code(tb, torch, dy.dtype), dy.stride(0), r, sp.data_ptr(), 4, F.data_ptr()))
    torch.cuda.synchronize()
    tb.check(tb.lib().tb_gemm_status(None))
    want = None
    for s, (g, m) in enumerate(ref.gradients(torch, dy, ck.values(torch), samples)):
        check_sums(torch, G[s], g, m, n * PARTS[dy_t])
        want = 0.01 * g * g if want is None else 0.99 * want + 0.01 * 0.01 * g * g
    assert float((F.double() - want).norm() / want.norm()) <= 4e-6  # a square doubles g's 2e-6
    x[225, 7] = math.nan  # a number no longer in block 1: the feature of that block is NaN, for the samples in it
    ck = packed(torch, tb, x, (torch.arange(n, device="cuda") < 560).to(torch.uint8))
    tb.check(tb.act8_weight_grad(ck.s, dy.data_ptr(), code(tb, torch, dy.dtype), dy.stride(0), r, sp.data_ptr(), 4, G.data_ptr(), tb.F32))
    assert not bool(torch.isnan(G[0][:, :7]).any()) and bool(torch.isnan(G[1][:, 7]).all()) and bool(torch.isnan(G[3][:, 7]).all())
    assert int(torch.isnan(G).sum()) == sum(r for a, b in samples if a < 256 and b > 128)


def test_first_call_of_a_host_thread(cuda, tblib):
    """A thread that has made no CUDA call before: every entry that encodes tensor maps, among them products that allocate no
    scratch first (an aligned BF16 dy, 74 or fewer tiles of one K step; adapters' forward without adapters; a GEMM)."""
    import threading
    torch, tb = cuda, tblib
    c = packed(torch, tb, rows(torch, 64, 256, torch.float32, 100))
    dy = rows(torch, 64, 256, torch.bfloat16, 101, None, 0.1, 0)
    x, w = rows(torch, 64, 256, torch.bfloat16, 102, heavy=0), rows(torch, 256, 256, torch.bfloat16, 103, None, 0.05, 0)
    outs = [torch.empty(256, 256, device="cuda") for _ in range(4)] + [torch.empty(64, 256, device="cuda", dtype=torch.bfloat16)]
    G, F, H, P, y = outs
    calls = [
        lambda: tb.act8_weight_grad(c.s, dy.data_ptr(), tb.BF16, 256, 256, None, 1, G.data_ptr(), tb.F32),
        lambda: tb.act8_fisher(c.s, dy.data_ptr(), tb.BF16, 256, 256, None, 1, F.data_ptr()),
        lambda: tb.act8_hessian(c.s, 1.0, H.data_ptr()),
        lambda: tb.lib().tb_gemm_nt_bf16(w.data_ptr(), 256, w.data_ptr(), 256, 256, 256, 256, 1.0, 0.0, None, 0, P.data_ptr(), 256, 0, None),
        lambda: tb.adapter_forward(tb.adapter_args(n=64, d=256, r=256, rank=0, n_adapters=0, w=w.data_ptr(), ldw=256,
                                                   x=x.data_ptr(), ldx=256, y=y.data_ptr(), ldy=256))]

    def all_outs():
        torch.cuda.synchronize()
        return [torch.tril(t) if t is H else t.clone() for t in outs]

    for f in calls:
        tb.check(f())
    want = all_outs()
    for t in outs:
        t.zero_()
    torch.cuda.synchronize()
    codes = []
    for f in calls:
        t = threading.Thread(target=lambda: codes.append(f()))
        t.start()
        t.join()
    assert codes == [tb.TB_OK] * len(calls)
    assert all(torch.equal(a, b) for a, b in zip(all_outs(), want))


@pytest.mark.parametrize("r,d,first", [(264, 264, True), (1300, 300, False), (256, 74 * 256, False), (74 * 256, 256, True)])
def test_fisher_of_more_samples_than_factors_are_kept(cuda, tblib, r, d, first):
    """1500 samples, factors from the 1025th on formed as they are needed: shared out over blocks or not (74 tiles), from
    codes or from values written out first (1300 and 18944 rows).  The bars of test_fisher; the state's additions are
    2^-24 of the state so far, and those are F beta^(S-j), which add to 100 F."""
    torch, tb = cuda, tblib
    n, S = 3000, 1500
    c = packed(torch, tb, rows(torch, n, d, torch.float32, 60, heavy=0))
    dy = rows(torch, n, r, torch.bfloat16, 61, ref.up(r, 8), 0.1, 0)
    samples = [(2 * i, 2 * i + 2) for i in range(S - 1)] + [(700, 1100)]
    F = torch.full((r, d), math.nan, device="cuda") if first else torch.rand(r, d, device="cuda")
    want = None if first else F.double()
    mag = torch.zeros(r, d, device="cuda", dtype=torch.float64)
    tb.check(tb.act8_fisher(c.s, dy.data_ptr(), tb.BF16, dy.stride(0), r, pairs(torch, samples).data_ptr(), S, F.data_ptr(),
                            first_step=first))
    torch.cuda.synchronize()
    tb.check(tb.lib().tb_gemm_status(None))
    xh, dyd = c.values(torch), dy.double()
    for a, b in samples:
        g = dyd[a:b].t() @ xh[a:b]
        e = (b - a) * 2.0 ** -23 * (dyd[a:b].abs().t() @ xh[a:b].abs())
        w = 0.01 if want is None else 0.01 * 0.01
        want = w * g * g if want is None else want.mul_(0.99).addcmul_(g, g, value=w)
        mag.mul_(0.99).add_(2 * g.abs() * e + e * e, alpha=w)
    bar = mag + (100 + 8) * 2.0 ** -24 * want
    assert bool(((F.double() - want).abs() <= bar * 1.01 + 1e-40).all())
    assert float((F.double() - want).norm() / want.norm()) <= 4e-6 + (100 + 8) * 2.0 ** -24


def test_values_beyond_their_scratch_are_decoded_in_the_product(cuda, tblib):
    """140000 tokens of 8192 features are more than 2 GiB as BF16: 1300 rows of gradients read the codes all the same."""
    torch, tb = cuda, tblib
    n, d, r, m = 140000, 8192, 1300, 333
    c = Checkpoint(torch, tb, n, d)
    c.codes.zero_()
    c.exps.fill_(1)
    dy = torch.zeros(n, ref.up(r, 8), device="cuda", dtype=torch.bfloat16)[:, :r]
    at = [(128 * 50 + 3, 128 * 50 + 3 + m), (n - m, n)]
    for i, (a, b) in enumerate(at):
        x = rows(torch, 512, d, torch.float32, 70 + i, heavy=0)
        q, e = ref.pack(torch, x)
        lo, k = a // 128 * 128, min(512, n - a // 128 * 128)
        c.codes[lo:lo + k] = q[:k]
        c.exps[lo // 128:lo // 128 + -(-k // 128)] = e[:-(-k // 128)]
        dy[a:b] = rows(torch, m, r, torch.bfloat16, 72 + i, None, 0.1, 0)
    G, F = torch.empty(2, r, d, device="cuda"), torch.empty(r, d, device="cuda")
    sp = pairs(torch, at)
    tb.check(tb.act8_weight_grad(c.s, dy.data_ptr(), tb.BF16, dy.stride(0), r, sp.data_ptr(), 2, G.data_ptr(), tb.F32))
    tb.check(tb.act8_fisher(c.s, dy.data_ptr(), tb.BF16, dy.stride(0), r, sp.data_ptr(), 2, F.data_ptr()))
    torch.cuda.synchronize()
    tb.check(tb.lib().tb_gemm_status(None))
    grads = []
    for s, (a, b) in enumerate(at):
        lo = a // 128 * 128
        xh = ref.values(torch, c.codes[lo:b], c.exps[lo // 128:])[a - lo:]
        g, A = dy[a:b].double().t() @ xh, dy[a:b].double().abs().t() @ xh.abs()
        check_sums(torch, G[s], g, A, m)
        grads.append(g)
    want = ref.fisher(torch, grads, 0.01, 0.99)
    assert float((F.double() - want).norm() / want.norm()) <= 4e-6


def test_hessian_of_more_tiles_than_a_grid_has_rows(cuda, tblib):
    """92417 features, whose rows of H do not start on 16 bytes: all 65703 tiles of 256 x 256 go through scratch and are
    written by a second kernel in two launches.  Spot rows; what is above the diagonal stays."""
    torch, tb = cuda, tblib
    n, d = 3, 361 * 256 + 1
    c = packed(torch, tb, rows(torch, n, d, torch.float32, 80))
    H = torch.full((d, d), 7.0, device="cuda")
    tb.check(tb.act8_hessian(c.s, 0.5, H.data_ptr()))
    torch.cuda.synchronize()
    tb.check(tb.lib().tb_gemm_status(None))
    xh = c.values(torch)
    for i in (0, 127, 128, 255, 256, 40000, 65535, 92159, 92160, 92415, 92416):
        k = min(d, i // 128 * 128 + 128)
        want, mag = 0.5 * xh[:, i] @ xh[:, :k], 0.5 * xh[:, i].abs() @ xh[:, :k].abs()
        assert bool(((H[i, :k].double() - want).abs() <= (n + 3) * 2.0 ** -23 * mag).all())
        assert bool((H[i, k:] == 7).all())


def test_two_host_threads(cuda, tblib):
    """Calls from two threads at once, each on a stream of its own, give what the same calls give one behind another."""
    import threading
    torch, tb = cuda, tblib
    n, d = 700, 520
    work = []
    for i in range(2):
        r = (264, 1500)[i]  # the latter's values are written out first
        c = packed(torch, tb, rows(torch, n, d, torch.float32, 90 + i))
        dy = rows(torch, n, r, torch.bfloat16, 92 + i, ref.up(r, 8), 0.1, 0)
        sp = pairs(torch, [(j * n // 40, (j + 1) * n // 40) for j in range(40)])
        out = [torch.zeros(40, r, d, device="cuda"), torch.zeros(r, d, device="cuda"), torch.zeros(d, d, device="cuda"),
               torch.zeros(n, d, device="cuda", dtype=torch.bfloat16), torch.zeros(n, r, device="cuda", dtype=torch.bfloat16)]
        w = rows(torch, r, d, torch.bfloat16, 94 + i, None, 0.05, 0)
        a, b = rows(torch, 16, d, torch.bfloat16, 96, None, 0.05, 0), rows(torch, 2 * r, 8, torch.bfloat16, 97, None, 0.3, 0)
        who = (torch.arange(n, device="cuda") % 3 - 1).to(torch.int32)
        work.append((r, c, dy, sp, out, w, a, b, who, torch.ones(2, device="cuda"), torch.cuda.Stream()))
    torch.cuda.synchronize()

    def go(k):
        r, c, dy, sp, (G, F, H, X, Y), w, a, b, who, scale, st = work[k]
        s = st.cuda_stream
        tb.check(tb.act8_weight_grad(c.s, dy.data_ptr(), tb.BF16, dy.stride(0), r, sp.data_ptr(), 40, G.data_ptr(), tb.F32, stream=s))
        tb.check(tb.act8_fisher(c.s, dy.data_ptr(), tb.BF16, dy.stride(0), r, sp.data_ptr(), 40, F.data_ptr(), stream=s))
        tb.check(tb.act8_hessian(c.s, 1.0, H.data_ptr(), stream=s))
        tb.check(tb.act8_unpack(c.s, X.data_ptr(), tb.BF16, d, stream=s))
        for m in (20, n):
            tb.check(tb.adapter_forward(tb.adapter_args(
                n=m, d=d, r=r, rank=8, n_adapters=2, w=w.data_ptr(), ldw=d, a=a.data_ptr(), lda=d, b=b.data_ptr(), ldb=8,
                scale=scale.data_ptr(), token_adapter=who.data_ptr(), x=X.data_ptr(), ldx=d, y=Y.data_ptr(), ldy=r), stream=s))

    want = []
    for k in (0, 1):
        go(k)
        torch.cuda.synchronize()
        want.append([t.clone() for t in work[k][4]])
    failed = []

    def loop(k):
        try:
            for _ in range(30):
                go(k)
            work[k][10].synchronize()
        except Exception as e:  # (handed to the test's own thread)
            failed.append(e)

    for _ in range(3):
        for k in (0, 1):
            for t in work[k][4]:
                t.zero_()
        torch.cuda.synchronize()
        threads = [threading.Thread(target=loop, args=(k,)) for k in (0, 1)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        torch.cuda.synchronize()
        assert not failed, failed
        assert all(torch.equal(x, y) for k in (0, 1) for x, y in zip(work[k][4], want[k]))
    tb.check(tb.lib().tb_gemm_status(None))


def test_values_written_out_first_under_graphs(cuda, tblib):
    """Two captured graphs whose calls write their values to scratch first, replayed on two streams at once with new sample
    bounds and new dy, against single calls."""
    torch, tb = cuda, tblib
    n, r, d, S = 900, 1400, 1300, 4
    sets, graphs = [], []
    for i in range(2):
        c = packed(torch, tb, rows(torch, n, d, torch.float32, 110 + i))
        dy = rows(torch, n, r, torch.float32, 112 + i, r, 1e-2, 0)
        sp = pairs(torch, [(j * 200, j * 200 + 190 + i) for j in range(S)])
        sets.append((c, dy, sp, torch.empty(S, r, d, device="cuda"), torch.empty(r, d, device="cuda")))

    def go(k, stream=None):
        c, dy, sp, G, F = sets[k]
        tb.check(tb.act8_weight_grad(c.s, dy.data_ptr(), tb.F32, r, r, sp.data_ptr(), S, G.data_ptr(), tb.F32, stream=stream))
        tb.check(tb.act8_fisher(c.s, dy.data_ptr(), tb.F32, r, r, sp.data_ptr(), S, F.data_ptr(), stream=stream))

    for k in (0, 1):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            go(k, torch.cuda.current_stream().cuda_stream)
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for t in range(3):
        for k, (c, dy, sp, G, F) in enumerate(sets):
            dy.copy_(rows(torch, n, r, torch.float32, 120 + 2 * t + k, r, 1e-2, 0))
            sp.copy_(pairs(torch, [(j * 210 + t, j * 210 + 130 + 9 * t + k) for j in range(S)]))
            G.fill_(-1.0)
            F.fill_(-1.0)
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        got = [(G.clone(), F.clone()) for _, _, _, G, F in sets]
        for k in (0, 1):
            go(k)
            torch.cuda.synchronize()
            assert torch.equal(got[k][0], sets[k][3]) and torch.equal(got[k][1], sets[k][4])
            xh = sets[k][0].values(torch)
            for s, (G, A) in enumerate(ref.gradients(torch, sets[k][1], xh, sets[k][2].tolist())):
                check_sums(torch, got[k][0][s], G, A, 200 * 3)


def test_scratch_that_cannot_be_had_fails_its_call_alone(cuda, tblib):
    """A call whose scratch (here 2 PB) is refused by the allocator returns before any launch; the next call is fine."""
    torch, tb = cuda, tblib
    c = packed(torch, tb, rows(torch, 40, 64, torch.float32, 130))
    unread = torch.zeros(64, device="cuda", dtype=torch.uint8).data_ptr()
    big = tb.act8(n=1 << 30, d=16, codes=unread, ldq=16, exps=unread, lde=16)
    assert tb.act8_weight_grad(big, unread + 2, tb.BF16, 1 << 20, 1 << 20, None, 1, unread, tb.F32) == tb.TB_ERR_CUDA
    assert b"memory" in tb.lib().tb_last_error()
    out = torch.zeros(40, 64, device="cuda")
    assert tb.act8_unpack(c.s, out.data_ptr(), tb.F32, 64) == tb.TB_OK
    assert torch.equal(out.double(), c.values(torch))


FIRST_CALL_CAPTURED = """
import sys
import torch
import tbabi as tb
n, d, r, what = 700, 512, 256, sys.argv[1]
g = torch.Generator(device="cuda").manual_seed(1)
codes = torch.randint(-127, 128, (n, d), device="cuda", generator=g, dtype=torch.int8)
exps = torch.full((6, d), 120, device="cuda", dtype=torch.uint8)
ck = tb.act8(n=n, d=d, codes=codes.data_ptr(), ldq=d, exps=exps.data_ptr(), lde=d)
half = lambda *s: torch.randn(*s, device="cuda", generator=g).bfloat16()
x, w, a, b = half(n, d), half(r, d), half(16, d), half(2 * r, 8)
dy, G, H = torch.randn(n, r, device="cuda", generator=g), torch.zeros(r, d, device="cuda"), torch.zeros(d, d, device="cuda")
who, scale = torch.zeros(n, device="cuda", dtype=torch.int32), torch.ones(2, device="cuda")
y = torch.zeros(n, r, device="cuda", dtype=torch.bfloat16)
def go():
    s = torch.cuda.current_stream().cuda_stream
    if what == "gradient":
        tb.check(tb.act8_weight_grad(ck, dy.data_ptr(), tb.F32, r, r, None, 1, G.data_ptr(), tb.F32, stream=s))
    elif what == "hessian":
        tb.check(tb.act8_hessian(ck, 1.0, H.data_ptr(), stream=s))
    else:
        tb.check(tb.adapter_forward(tb.adapter_args(n=int(what), d=d, r=r, rank=8, n_adapters=2, w=w.data_ptr(), ldw=d, a=a.data_ptr(),
            lda=d, b=b.data_ptr(), ldb=8, scale=scale.data_ptr(), token_adapter=who.data_ptr(), x=x.data_ptr(), ldx=d,
            y=y.data_ptr(), ldy=r), stream=s))
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    go()
graph.replay()
torch.cuda.synchronize()
got = [t.clone() for t in (G, H, y)]
go()
torch.cuda.synchronize()
assert all(torch.equal(p, q) for p, q in zip(got, (G, H, y))) and any(bool(t.any()) for t in got)
"""


@pytest.mark.parametrize("what", ["gradient", "hessian", "20", "700"])
def test_a_process_first_call_may_be_captured(cuda, tblib, what):
    """In a process of its own: the library's pool and its kernels' settings are made while a stream captures."""
    import os
    import subprocess
    import sys
    env = dict(os.environ, PYTHONPATH=os.path.dirname(tblib.__file__))
    p = subprocess.run([sys.executable, "-c", FIRST_CALL_CAPTURED, what], env=env, capture_output=True, text=True, timeout=300)
    assert p.returncode == 0, p.stderr[-2000:]


def test_more_blocks_of_tokens_than_a_grid_has_rows(cuda, tblib):
    """65535 blocks of 128 tokens and 300 tokens more: packing and reading back in two launches, and sums over all of them.
    A sum's groups (512 tokens; the Hessian's 128 are exact) lose at most 32 2^-23 of their terms' magnitudes in the tensor
    core; the one tile has 74 to 148 shares, the additions of whose groups, and of the shares, round by 2^-24 of the
    magnitudes each."""
    torch, tb = cuda, tblib
    n, d, r = 65535 * 128 + 300, 9, 5
    x = rows(torch, n, d, torch.float32, 140, heavy=0)
    keep = (torch.arange(n, device="cuda") % 1000 < 990).to(torch.uint8)
    c = packed(torch, tb, x, keep)
    lo = 65533 * 128  # the last blocks of the first launch, and the second
    q, e = ref.pack(torch, x[lo:], keep[lo:])
    assert torch.equal(c.codes[lo:n, :d], q) and torch.equal(c.exps[65533:, :d], e)
    q, e = ref.pack(torch, x[:1024], keep[:1024])
    assert torch.equal(c.codes[:1024, :d], q) and torch.equal(c.exps[:8, :d], e)
    xh = c.values(torch)
    out = torch.full((n, d), 9.0, device="cuda")
    tb.check(tb.act8_unpack(c.s, out.data_ptr(), tb.F32, d))
    assert torch.equal(out.double(), xh)
    dy = rows(torch, n, r, torch.bfloat16, 141, 8, 1e-2, 0)
    G, H = torch.empty(r, d, device="cuda"), torch.empty(d, d, device="cuda")
    tb.check(tb.act8_weight_grad(c.s, dy.data_ptr(), tb.BF16, 8, r, None, 1, G.data_ptr(), tb.F32))
    tb.check(tb.act8_hessian(c.s, 1.0, H.data_ptr()))
    torch.cuda.synchronize()
    tb.check(tb.lib().tb_gemm_status(None))
    for got, a, groups in ((G, dy.double(), n // 512), (H, xh, n // 128)):
        want, mag = a.t() @ xh, a.abs().t() @ xh.abs()
        bar = (64 + groups // 74 + 1 + 148 + 2) * 2.0 ** -24 * mag
        assert bool(((got.double() - want).abs() <= bar).all())
