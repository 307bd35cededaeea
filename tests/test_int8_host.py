"""What quantize and linear_int8 refuse, and what their C entry points check before they touch CUDA (no GPU needed)."""
import pytest
import torch as th

BF, I8 = th.bfloat16, th.int8


@pytest.fixture(scope='module')
def lib():
    import __graft_entry__ as ge
    ge.build()
    from wind_rwkv.rwkv7 import _lib
    return _lib.lib()


def fwd(lib, M=4, N=16, K=64, ldx=64, ldw=64, ldr=16, ldy=16, act=0, flags=0, x=0x1000, xs=0x1000, w=0x1000, s=0x1000, bias=None, r=None, y=0x1000, ws=None):
    return lib.wkv7_linear_int8(x, xs, w, s, bias, r, y, M, N, K, ldx, ldw, ldr, ldy, act, flags, ws, None)


def test_product_checks(lib):
    assert fwd(lib, M=-1) == fwd(lib, N=0) == fwd(lib, K=0) == fwd(lib, act=7) == fwd(lib, act=-1) == fwd(lib, flags=4) == fwd(lib, flags=8) == -1
    assert fwd(lib, ldx=48) == fwd(lib, ldw=48) == fwd(lib, ldy=15) == fwd(lib, r=0x1000, ldr=15) == -1
    assert fwd(lib, ldx=72) == fwd(lib, ldw=72) == -4
    assert fwd(lib, x=0x1008) == fwd(lib, w=0x1008) == fwd(lib, xs=0x1002) == fwd(lib, s=0x1002) == fwd(lib, y=0x1001) == fwd(lib, r=0x1001) == fwd(lib, ws=0x1008) == -4
    assert fwd(lib, flags=1, y=0x1002) == fwd(lib, flags=2, bias=0x1002) == -4
    assert fwd(lib, x=None) == fwd(lib, w=None) == fwd(lib, xs=None) == fwd(lib, s=None) == fwd(lib, y=None) == -6
    assert fwd(lib, M=1 << 31) == fwd(lib, ldx=1 << 31) == fwd(lib, K=1 << 17, ldx=1 << 17, ldw=1 << 17) == -8
    assert fwd(lib, M=0, x=None, w=None, y=None) == 0
    assert lib.wkv7_linear_int8_workspace_bytes(0, 5, 8) == lib.wkv7_linear_int8_workspace_bytes(-1, 5, 8) == 0


def test_quantize_checks(lib):
    f = lib.wkv7_quantize
    assert f(0x1000, 0x1000, 0x1000, -1, 8, 8, 8, 0, None) == f(0x1000, 0x1000, 0x1000, 1, 0, 8, 8, 0, None) == f(0x1000, 0x1000, 0x1000, 1, 8, 7, 8, 0, None) == -1
    assert f(0x1000, 0x1000, 0x1000, 1, 8, 8, 7, 0, None) == f(0x1000, 0x1000, 0x1000, 1, 8, 8, 8, 2, None) == -1
    assert f(None, 0x1000, 0x1000, 1, 8, 8, 8, 0, None) == f(0x1000, None, 0x1000, 1, 8, 8, 8, 0, None) == f(0x1000, 0x1000, None, 1, 8, 8, 8, 0, None) == -6
    assert f(0x1001, 0x1000, 0x1000, 1, 8, 8, 8, 0, None) == f(0x1002, 0x1000, 0x1000, 1, 8, 8, 8, 1, None) == f(0x1000, 0x1000, 0x1002, 1, 8, 8, 8, 0, None) == -4
    assert f(0x1000, 0x1000, 0x1000, 1, (1 << 30) + 1, 1 << 31, 1 << 31, 0, None) == -8
    assert f(None, None, None, 0, 8, 8, 8, 0, None) == 0


def refusals(linear_int8, quantize):
    x, w = (th.zeros(4, 64, dtype=I8), th.zeros(4)), (th.zeros(16, 64, dtype=I8), th.zeros(16))
    for bad in (dict(act='swish'), dict(bias=th.zeros(15)), dict(bias=th.zeros(16, dtype=th.float64)), dict(residual=th.zeros(4, 15, dtype=BF)), dict(residual=th.zeros(4, 16)),
                dict(residual=th.zeros(16, dtype=BF)), dict(residual=th.zeros(4, 16, dtype=BF), out_dtype=th.float32)):
        with pytest.raises(ValueError, match='linear_int8'):
            linear_int8(x, w, **bad)
    long = 1 << 17
    for bx, bw in ((x, (w[0][:, :56], w[1])), (x, (w[0][None], w[1][None])), (x, (w[0][:0], w[1][:0])), ((x[0], x[1][:3]), w), (x, (w[0], w[1][:1])), (x, (w[0], w[1][:, None])),
                   ((x[0][:, :0], x[1]), (w[0][:, :0], w[1])), ((th.zeros(1, long, dtype=I8), th.zeros(1)), (th.zeros(1, long, dtype=I8), th.zeros(1)))):
        with pytest.raises(ValueError, match='linear_int8'):
            linear_int8(bx, bw)
    for bx, bw, out in ((x[0], w, None), (x, w[0], None), ((x[0].float(), x[1]), w, None), (x, (w[0], w[1].bfloat16()), None), (x, w, th.float16), (x, w, I8)):
        with pytest.raises(TypeError, match='linear_int8'):
            linear_int8(bx, bw, out_dtype=out)
    for more in (dict(bias=th.zeros(16).requires_grad_()), dict(residual=th.zeros(4, 16, dtype=BF).requires_grad_())):
        with pytest.raises(RuntimeError, match='no backward'):
            linear_int8(x, w, **more)
    with pytest.raises(RuntimeError, match='CUDA'):
        linear_int8(x, w)
    with pytest.raises(TypeError, match='quantize'):
        quantize(th.zeros(4, 64).half())
    for bad in (th.zeros(4, 0), th.zeros(()), th.zeros(1).expand(2, (1 << 30) + 1)):
        with pytest.raises(ValueError, match='quantize'):
            quantize(bad)
    with pytest.raises(RuntimeError, match='CUDA'):
        quantize(th.zeros(4, 64))


def test_python_refusals(lib):
    from wind_rwkv.rwkv7 import linear_int8, quantize
    refusals(linear_int8, quantize)


def test_refusals_while_torch_compile_traces(lib):
    from wind_rwkv.rwkv7 import linear_int8, quantize

    def traced(f):
        def call(*a, **k):
            th.compiler.reset()
            return th.compile(lambda: f(*a, **k), backend='eager')()
        return call

    refusals(traced(linear_int8), traced(quantize))


def test_operands_on_16_byte_boundaries():
    from wind_rwkv.rwkv7.rwkv7_int8 import operand8, pitch8
    assert [pitch8(n) for n in (1, 16, 17, 203)] == [16, 16, 32, 208]
    t = th.arange(6 * 40, dtype=th.int16).to(I8).view(6, 40)
    wide = th.zeros(6, 48, dtype=I8)
    wide[:, :40] = t
    for view in (wide[:, :40], wide[:, 16:40], wide):
        r, ld = operand8(view)
        assert r is view and ld == 48
    for view in (t, wide[:, 1:30], t.t()):
        r, ld = operand8(view)
        assert th.equal(r, view) and ld % 16 == 0 and r.data_ptr() % 16 == 0 and r.stride(0) == ld


def test_forward_mode_tangents_are_refused(lib):
    import torch.autograd.forward_ad as fw
    from wind_rwkv.rwkv7 import linear_int8, quantize, rms_norm
    x, w = (th.zeros(4, 64, dtype=I8), th.zeros(4)), (th.zeros(16, 64, dtype=I8), th.zeros(16))
    with fw.dual_level(), th.no_grad():
        def dual(t):
            return fw.make_dual(t, th.ones_like(t))
        for call in (lambda: linear_int8(x, w, residual=dual(th.zeros(4, 16, dtype=BF))), lambda: linear_int8(x, w, dual(th.zeros(16))), lambda: linear_int8((x[0], dual(x[1])), w),
                     lambda: linear_int8(x, (w[0], dual(w[1]))), lambda: quantize(dual(th.zeros(4, 64))), lambda: rms_norm(dual(th.zeros(4, 64)), out_dtype=I8),
                     lambda: rms_norm(th.zeros(4, 64), dual(th.zeros(64)), out_dtype=I8), lambda: rms_norm(th.zeros(4, 64), residual=dual(th.zeros(4, 64)), out_dtype=I8)):
            with pytest.raises(RuntimeError, match='tangent'):
                call()
        with pytest.raises(RuntimeError, match='CUDA'):  # (a level alone refuses nothing)
            linear_int8(x, w)
