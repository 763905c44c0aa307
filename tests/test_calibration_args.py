"""CPU: argument checks of the checkpoint and adapter entries that return before
any device work, and the layout of their structures."""
import ctypes as C

import pytest

import tbabi as tb

P = 1 << 20  # a 16-byte aligned address that is never read


def ck(**kw):
    a = dict(n=256, d=64, codes=P, ldq=64, exps=P, lde=64)
    a.update(kw)
    return tb.act8(**a)


def test_struct_layouts():
    assert C.sizeof(tb.Act8) == 48
    assert C.sizeof(tb.AdapterArgs) == 184  # 32 of sizes, 48 of w, a, b, 16 of scale and tokens, 32 forward, 56 backward


@pytest.mark.parametrize("kw,code", [
    (dict(d=0), tb.TB_ERR_ZERO_SIZE), (dict(n=-1), tb.TB_ERR_SHAPE), (dict(n=1 << 31), tb.TB_ERR_SHAPE),
    (dict(ldq=48), tb.TB_ERR_ARG), (dict(ldq=72), tb.TB_ERR_ARG), (dict(lde=65), tb.TB_ERR_ARG),
    (dict(codes=None), tb.TB_ERR_ARG), (dict(exps=P + 8), tb.TB_ERR_ARG)])
def test_checkpoint_refusals(tblib, kw, code):
    c = ck(**kw)
    assert tb.act8_pack(c, P, tb.F32, 64) == code
    assert tb.act8_unpack(c, P, tb.F32, 64) == code
    assert tb.act8_hessian(c, 1.0, P) == code
    assert tb.act8_weight_grad(c, P, tb.BF16, 64, 64, None, 1, P, tb.F32) == code
    assert tb.act8_fisher(c, P, tb.BF16, 64, 64, None, 1, P) == code


def test_struct_size_is_checked(tblib):
    c = ck()
    c.struct_size = 40
    assert tb.act8_pack(c, P, tb.F32, 64) == tb.TB_ERR_ARG
    a = tb.adapter_args(n=1, d=64, r=64, rank=8, n_adapters=0, w=P, ldw=64, x=P, ldx=64, y=P, ldy=64)
    a.struct_size = 8
    assert tb.adapter_forward(a) == tb.TB_ERR_ARG
    assert b"struct_size" in tb.lib().tb_last_error()


def test_call_refusals(tblib):
    c = ck()
    assert tb.act8_pack(c, P, 7, 64) == tb.TB_ERR_ARG
    assert tb.act8_pack(c, None, tb.F32, 64) == tb.TB_ERR_ARG
    assert tb.act8_pack(c, P, tb.F32, 63) == tb.TB_ERR_ARG
    assert tb.act8_unpack(c, P, tb.BF16, 60) == tb.TB_ERR_ARG
    assert tb.act8_weight_grad(c, P, tb.BF16, 64, 64, None, 2, P, tb.F32) == tb.TB_ERR_ARG  # two samples, none named
    assert tb.act8_weight_grad(c, P, tb.BF16, 64, 64, P, -1, P, tb.F32) == tb.TB_ERR_ARG
    assert tb.act8_weight_grad(c, P, 5, 64, 64, P, 1, P, tb.F32) == tb.TB_ERR_ARG
    assert tb.act8_weight_grad(c, P, tb.BF16, 63, 64, P, 1, P, tb.F32) == tb.TB_ERR_ARG
    assert tb.act8_weight_grad(c, P, tb.BF16, 64, 0, P, 1, P, tb.F32) == tb.TB_ERR_ZERO_SIZE
    assert tb.act8_weight_grad(c, P, tb.BF16, 64, 64, P, 1, P, tb.F16) == tb.TB_ERR_UNSUPPORTED
    assert tb.act8_weight_grad(c, P, tb.BF16, 64, 64, P, 1, P, tb.F32, g_stride=64 * 64 - 1) == tb.TB_ERR_SHAPE
    assert tb.act8_weight_grad(c, P, tb.BF16, 64, 64, P, 1, None, tb.F32) == tb.TB_ERR_ARG
    assert tb.act8_fisher(c, P, tb.BF16, 64, 64, P, 1, None) == tb.TB_ERR_ARG
    assert tb.act8_hessian(c, 1.0, None) == tb.TB_ERR_ARG
    # nothing to do, nothing touched
    assert tb.act8_pack(ck(n=0), None, tb.F32, 64) == tb.TB_OK
    assert tb.act8_unpack(ck(n=0), None, tb.F32, 64) == tb.TB_OK
    assert tb.act8_weight_grad(c, P, tb.BF16, 64, 64, P, 0, None, tb.F32) == tb.TB_OK
    assert tb.act8_fisher(c, P, tb.BF16, 64, 64, P, 0, None) == tb.TB_OK


def adapters(**kw):
    a = dict(n=4, d=64, r=32, rank=8, n_adapters=2, w=P, ldw=64, a=P, lda=64, b=P, ldb=8, scale=P, token_adapter=P, x=P,
             ldx=64, y=P, ldy=32)
    a.update(kw)
    return tb.adapter_args(**a)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=tb.F32), tb.TB_ERR_UNSUPPORTED), (dict(dtype=tb.F16), tb.TB_ERR_UNSUPPORTED),
    (dict(d=0), tb.TB_ERR_ZERO_SIZE), (dict(r=0), tb.TB_ERR_ZERO_SIZE), (dict(n=-1), tb.TB_ERR_SHAPE),
    (dict(rank=0), tb.TB_ERR_SHAPE), (dict(rank=129, ldb=136), tb.TB_ERR_SHAPE), (dict(n_adapters=-1), tb.TB_ERR_ARG),
    (dict(w=P + 2), tb.TB_ERR_ARG), (dict(ldw=60), tb.TB_ERR_ARG), (dict(ldw=66), tb.TB_ERR_ARG),
    (dict(a=None), tb.TB_ERR_ARG), (dict(ldb=4), tb.TB_ERR_ARG), (dict(scale=None), tb.TB_ERR_ARG),
    (dict(token_adapter=None), tb.TB_ERR_ARG), (dict(x=P + 8), tb.TB_ERR_ARG), (dict(ldx=65), tb.TB_ERR_ARG),
    (dict(y=None), tb.TB_ERR_ARG), (dict(ldy=31), tb.TB_ERR_ARG)])
def test_adapter_forward_refusals(tblib, kw, code):
    assert tb.adapter_forward(adapters(**kw)) == code


def test_adapter_backward_refusals(tblib):
    c = tb.act8(n=4, d=64, codes=P, ldq=64, exps=P, lde=64)
    ok = dict(dy=P, lddy=32, x8=c, dx=P, lddx=64, da=P, db=P)
    for kw, code in [(dict(dy=None), tb.TB_ERR_ARG), (dict(lddy=36), tb.TB_ERR_ARG), (dict(x8=None), tb.TB_ERR_ARG),
                     (dict(da=None), tb.TB_ERR_ARG), (dict(lddx=63), tb.TB_ERR_ARG), (dict(w=None), tb.TB_ERR_ARG),
                     (dict(x8=ck(n=5)), tb.TB_ERR_SHAPE), (dict(x8=ck(n=4, d=48)), tb.TB_ERR_SHAPE)]:
        assert tb.adapter_backward(adapters(**{**ok, **kw})) == code, kw
    assert tb.adapter_forward(adapters(n=0, x=None, y=None, token_adapter=None)) == tb.TB_OK


@pytest.mark.parametrize("n", [(1 << 31) - 127, (1 << 31) - 65])
def test_hessian_refuses_tokens_that_its_steps_cannot_count(tblib, n):
    """Tokens whose number, rounded up to the Hessian's step of 128, passes 31 bits (the other entries take them)."""
    assert tb.act8_hessian(ck(n=n), 1.0, P) == tb.TB_ERR_SHAPE
    assert tb.act8_hessian(ck(n=n), 1.0, P, accumulate=True) == tb.TB_ERR_SHAPE


@pytest.mark.parametrize("many", [(1 << 31) - 255, (1 << 31) - 1])
def test_features_that_tiles_cannot_count_are_refused(tblib, many):
    """In or out features whose number, rounded up to a tile of 256, passes 31 bits."""
    ld = 1 << 31
    c = ck(n=1, d=many, ldq=ld, lde=ld)
    assert tb.act8_pack(c, P, tb.F32, ld) == tb.TB_ERR_SHAPE
    assert tb.act8_unpack(c, P, tb.F32, ld) == tb.TB_ERR_SHAPE
    assert tb.act8_hessian(c, 1.0, P) == tb.TB_ERR_SHAPE
    for k, r in ((c, 8), (ck(n=1), many)):
        assert tb.act8_weight_grad(k, P, tb.F32, ld, r, None, 1, P, tb.F32) == tb.TB_ERR_SHAPE
        assert tb.act8_fisher(k, P, tb.F32, ld, r, None, 1, P) == tb.TB_ERR_SHAPE
    for kw in (dict(d=many, ldw=ld, lda=ld, ldx=ld), dict(r=many, ldy=ld, lddy=ld)):
        assert tb.adapter_forward(adapters(**kw)) == tb.TB_ERR_SHAPE
        assert tb.adapter_backward(adapters(dy=P, lddy=ld, dx=P, lddx=ld, **{k: v for k, v in kw.items() if k != "lddy"})) == tb.TB_ERR_SHAPE


def test_adapters_refuse_tokens_beyond_their_limit(tblib):
    """The largest batch is 2^31 - 65537 tokens, as the header states."""
    text = open(tb.HEADER).read()
    assert "tokens, up to 2^31 - 65537 " in text[text.index("typedef struct tb_adapter_args"):]
    for n in ((1 << 31) - 65536, (1 << 31) - 256, 1 << 31):
        assert tb.adapter_forward(adapters(n=n)) == tb.TB_ERR_SHAPE
        assert tb.adapter_backward(adapters(n=n, dy=P, lddy=32, dx=P, lddx=64)) == tb.TB_ERR_SHAPE


def test_samples_end_at_their_limit(tblib):
    """At most 65535 samples in a call, as the header states."""
    text = open(tb.HEADER).read()
    assert "S at most 65535" in text[text.index("Weight gradients of y"):text.index("int tb_act8_weight_grad")]
    c = ck()
    assert tb.act8_weight_grad(c, P, tb.BF16, 64, 64, P, 65536, P, tb.F32) == tb.TB_ERR_ARG
    assert tb.act8_fisher(c, P, tb.BF16, 64, 64, P, 65536, P) == tb.TB_ERR_ARG
