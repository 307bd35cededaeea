"""What linear refuses, and what its C entry points check before they touch CUDA (no GPU needed)."""
import pytest
import torch as th

BF = th.bfloat16


@pytest.fixture(scope='module')
def lib():
    import __graft_entry__ as ge
    ge.build()
    from wind_rwkv.rwkv7 import _lib
    return _lib.lib()


def fwd(lib, M=4, N=16, K=64, ldx=64, ldw=64, ldr=16, ldy=16, ldz=16, act=0, flags=0, x=0x1000, w=0x1000, bias=None, r=None, y=0x1000, z=None, ws=None):
    return lib.wkv7_linear_fwd(x, w, bias, r, y, z, M, N, K, ldx, ldw, ldr, ldy, ldz, act, flags, ws, None)


def bwd(lib, M=4, N=16, K=64, lds=16, lddy=16, act=2, flags=0, saved=0x1000, dy=0x1000, dx=0x1000, dw=0x1000, db=None, ws=0x1000):
    return lib.wkv7_linear_bwd(0x1000, 0x1000, saved, dy, dx, dw, db, M, N, K, K, K, lds, lddy, act, flags, ws, None)


def test_forward_checks(lib):
    assert fwd(lib, M=-1) == fwd(lib, N=0) == fwd(lib, K=0) == -1
    assert fwd(lib, act=7) == fwd(lib, act=-1) == fwd(lib, flags=16) == fwd(lib, flags=4) == -1
    assert fwd(lib, ldx=56) == fwd(lib, ldw=56) == fwd(lib, ldy=15) == fwd(lib, r=0x1000, ldr=15) == -1
    assert fwd(lib, N=17, ldy=17, z=0x1000, ldz=17) == -1                     # z's rows hold the next multiple of 8
    assert fwd(lib, K=60) == fwd(lib, ldx=68) == fwd(lib, ldw=68) == -4
    assert fwd(lib, x=0x1008) == fwd(lib, w=0x1008) == fwd(lib, y=0x1001) == fwd(lib, r=0x1001) == fwd(lib, z=0x1008) == fwd(lib, ws=0x1008) == -4
    assert fwd(lib, flags=1, y=0x1002) == fwd(lib, flags=2, bias=0x1002) == -4
    assert fwd(lib, x=None) == fwd(lib, w=None) == fwd(lib, y=None) == -6
    assert fwd(lib, M=1 << 31) == fwd(lib, ldx=1 << 31) == -8
    assert fwd(lib, M=0, x=None, w=None, y=None) == 0


def test_backward_checks(lib):
    assert bwd(lib, flags=4, act=3) == bwd(lib, flags=5, act=2) == bwd(lib, flags=2) == bwd(lib, flags=12) == -1   # a derivative from y: relu and relu2, bf16
    assert bwd(lib, lds=15) == bwd(lib, lddy=15) == -1
    assert bwd(lib, dy=None) == bwd(lib, saved=None) == bwd(lib, ws=None) == -6
    assert bwd(lib, dx=0x1008) == bwd(lib, dw=0x1008) == bwd(lib, ws=0x1008) == bwd(lib, db=0x1002) == bwd(lib, saved=0x1001) == -4
    assert bwd(lib, M=0, dx=None, dw=None) == 0
    assert lib.wkv7_linear_bwd_workspace_bytes(0, 5, 8) == lib.wkv7_linear_bwd_workspace_bytes(-1, 5, 8) == lib.wkv7_linear_fwd_workspace_bytes(0, 5, 8) == 0
    for M, N in ((1, 1), (333, 77), (70000, 5)):
        assert lib.wkv7_linear_bwd_workspace_bytes(M, N, 64) >= M * ((N + 7) // 8 * 8) * 2 + 4 * N


def test_python_refusals(lib):
    from wind_rwkv.rwkv7 import linear
    x, w = th.zeros(4, 64, dtype=BF), th.zeros(16, 64, dtype=BF)
    for bad in (dict(act='swish'), dict(bias=th.zeros(15)), dict(bias=th.zeros(16, dtype=th.float64)), dict(residual=th.zeros(4, 15, dtype=BF)),
                dict(residual=th.zeros(4, 16)), dict(residual=th.zeros(16, dtype=BF))):
        with pytest.raises(ValueError, match='linear'):
            linear(x, w, **bad)
    for bx, bw in ((x, w[:, :56]), (x, w[None]), (x[:, :60], w[:, :60]), (x, w[:0])):
        with pytest.raises(ValueError, match='linear'):
            linear(bx, bw)
    for bx, bw, out in ((x.float(), w, None), (x, w.half(), None), (x, w, th.float16)):
        with pytest.raises(TypeError, match='linear'):
            linear(bx, bw, out_dtype=out)
    with pytest.raises(RuntimeError, match='CUDA'):
        linear(x, w)


@pytest.mark.parametrize('dynamic', [False, True])
def test_refusals_while_torch_compile_traces(lib, dynamic):
    from wind_rwkv.rwkv7 import linear
    x, w, b, r = th.zeros(4, 64, dtype=BF), th.zeros(16, 64, dtype=BF), th.zeros(16), th.zeros(4, 16, dtype=BF)

    def call(x, w, bias=None, residual=None, **how):
        th.compiler.reset()
        return th.compile(lambda *t: linear(t[0], t[1], t[2], residual=t[3], **how) * 1, backend='eager', dynamic=dynamic)(x, w, bias, residual)

    for bad in (dict(act='swish'), dict(bias=b[:15]), dict(bias=b[:1]), dict(bias=b.double()), dict(residual=r[:, :15]), dict(residual=r[:3]), dict(residual=r.float()),
                dict(residual=r, out_dtype=th.float32), dict(bias=b[None])):
        with pytest.raises(ValueError, match='linear'):
            call(x, w, **bad)
    for bx, bw in ((x, w[:, :56]), (x[:, :56], w), (x, w[None]), (x[:, :60], w[:, :60]), (x, w[:0])):
        with pytest.raises(ValueError, match='linear'):
            call(bx, bw)
    for bx, bw, out in ((x.float(), w, None), (x, w.half(), None), (x.half(), w, None), (x, w, th.float16)):
        with pytest.raises(TypeError, match='linear'):
            call(bx, bw, out_dtype=out)
    with pytest.raises(RuntimeError, match='CUDA'):
        call(x, w, b, r, act='relu2')


def test_rows_are_taken_as_they_lie():
    from wind_rwkv.rwkv7.rwkv7_linear import operand_of, rows_of
    t = th.zeros(4, 6, 32, dtype=BF)
    for view, ld in ((t, 32), (t[..., :16], 32), (t[0], 32), (t[:, 0], 192), (t[0, 0], 32), (t[:1, 2:3], 32)):
        r, p = rows_of(view)
        assert r is view and p == ld
    for view in (t.transpose(0, 1), t[:, :3], t[..., ::2], t[:, :1].expand(4, 6, 32)):
        r, p = rows_of(view)
        assert r.is_contiguous() and p == view.shape[-1]
    assert operand_of(t[..., :16])[1] == 32 and operand_of(t[..., 1:17])[1] == 16 and operand_of(t[0, :, 8:24])[0].data_ptr() == t.data_ptr() + 16
