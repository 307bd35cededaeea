"""What rms_norm and dropout refuse, what their C entry points check before they touch CUDA, and the generator's words (no GPU needed)."""
import pytest
import torch as th

BF = th.bfloat16


@pytest.fixture(scope='module')
def lib():
    import __graft_entry__ as ge
    ge.build()
    from wind_rwkv.rwkv7 import _lib
    return _lib.lib()


def fwd(lib, M=4, D=64, ldx=64, ldr=64, ldy=64, ldh=64, eps=1e-5, p=0., flags=0, x=0x1000, r=0x1000, w=0x1000, y=0x1000, h=0x1000, rstd=None, scale=None, seed_ptr=None):
    return lib.wkv7_rms_norm_fwd(x, r, w, y, h, rstd, scale, M, D, ldx, ldr, ldy, ldh, eps, p, 1, seed_ptr, flags, None)


def bwd(lib, M=4, D=64, ldh=64, lddy=64, lddh=64, lddx=64, lddr=64, p=0., flags=0, h=0x1000, rstd=0x1000, w=0x1000, dy=0x1000, dh=0x1000, dx=0x1000, dr=0x1000, dw=0x1000,
        ws=0x1000, seed_ptr=None):
    return lib.wkv7_rms_norm_bwd(h, rstd, w, dy, dh, dx, dr, dw, M, D, ldh, lddy, lddh, lddx, lddr, p, 1, seed_ptr, flags, ws, None)


def test_norm_checks(lib):
    assert fwd(lib, M=-1) == fwd(lib, D=0) == fwd(lib, ldx=63) == fwd(lib, ldr=63) == fwd(lib, ldy=63) == fwd(lib, ldh=63) == -1
    assert fwd(lib, eps=-1.) == fwd(lib, eps=float('nan')) == fwd(lib, p=-0.1) == fwd(lib, p=1.1) == fwd(lib, p=float('nan')) == fwd(lib, flags=32) == -1
    assert fwd(lib, flags=24, scale=0x1000) == -1                                   # y in one type
    assert fwd(lib, p=0.5, r=None, h=None) == -1                                    # dropout of what joins the stream
    assert fwd(lib, x=None) == fwd(lib, y=None) == fwd(lib, h=None) == fwd(lib, r=None) == fwd(lib, flags=16) == fwd(lib, scale=0x1000) == -6
    assert fwd(lib, x=0x1001) == fwd(lib, flags=1, x=0x1002) == fwd(lib, flags=2, r=0x1002) == fwd(lib, flags=2, h=0x1002) == fwd(lib, flags=4, w=0x1002) == -4
    assert fwd(lib, flags=8, y=0x1002) == fwd(lib, rstd=0x1002) == fwd(lib, flags=16, scale=0x1002) == fwd(lib, seed_ptr=0x1004) == -4
    big = 16385
    assert fwd(lib, D=big, ldx=big, ldr=big, ldy=big, ldh=big) == -8
    assert fwd(lib, M=0, x=None, y=None, h=None, r=None) == 0


def test_norm_backward_checks(lib):
    assert bwd(lib, M=-1) == bwd(lib, D=0) == bwd(lib, ldh=63) == bwd(lib, lddy=63) == bwd(lib, lddh=63) == bwd(lib, lddx=63) == bwd(lib, lddr=63) == -1
    assert bwd(lib, p=2.) == bwd(lib, flags=16) == -1
    assert bwd(lib, h=None) == bwd(lib, rstd=None) == bwd(lib, dy=None) == bwd(lib, ws=None) == -6
    assert bwd(lib, h=0x1001) == bwd(lib, flags=2, dh=0x1002) == bwd(lib, flags=1, dx=0x1002) == bwd(lib, flags=2, dr=0x1002) == bwd(lib, flags=8, dy=0x1002) == -4
    assert bwd(lib, dw=0x1002) == bwd(lib, ws=0x1008) == bwd(lib, flags=4, w=0x1002) == bwd(lib, rstd=0x1002) == bwd(lib, seed_ptr=0x1004) == -4
    assert bwd(lib, M=0, dw=None, h=None, dy=None, rstd=None) == 0
    n = lib.wkv7_rms_norm_bwd_workspace_bytes
    assert n(0, 64) == n(-1, 64) == n(4, 0) == n(4, 16385) == 0
    for M, D in ((1, 1), (5, 333), (100000, 16), (70000, 2048), (1000, 16384)):
        assert n(M, D) % (4 * D) == 0 and 4 * D <= n(M, D) <= 16 * 148 * 256 * 4 * D


def test_dropout_checks(lib):
    f = lib.wkv7_dropout
    assert f(0x1000, None, 0x1000, -1, 0.5, 1, None, 0, None) == f(0x1000, None, 0x1000, 8, 1.5, 1, None, 0, None) == f(0x1000, None, 0x1000, 8, 0.5, 1, None, 4, None) == -1
    assert f(None, None, 0x1000, 8, 0.5, 1, None, 0, None) == f(0x1000, None, None, 8, 0.5, 1, None, 0, None) == -6
    assert f(0x1008, None, 0x1000, 8, 0.5, 1, None, 0, None) == f(0x1000, 0x1008, 0x1000, 8, 0.5, 1, None, 0, None) == f(0x1000, None, 0x1008, 8, 0.5, 1, None, 0, None) == -4
    assert f(0x1000, None, 0x1000, 8, 0.5, 1, 0x1004, 0, None) == -4
    assert f(None, None, None, 0, 0.5, 1, None, 0, None) == 0


def refusals(call_norm, call_drop):
    x, w, r = th.zeros(4, 64, dtype=BF), th.zeros(64), th.zeros(4, 64, dtype=BF)
    for bad in (dict(weight=w[:63]), dict(weight=w[:1]), dict(residual=r[:3]), dict(residual=r[:, :1]), dict(eps=-1e-5), dict(residual=r, p=0.1), dict(residual=r, p=1.5, seed=1),
                dict(residual=r, p=0.1, seed=-1), dict(residual=r, p=0.1, seed=1 << 63), dict(residual=r, p=0.1, seed=th.zeros(2, dtype=th.int64)),
                dict(residual=r, p=0.1, seed=th.zeros(1, dtype=th.int32)), dict(p=0.1, seed=1)):
        with pytest.raises(ValueError, match='rms_norm'):
            call_norm(x, **bad)
    for bad in (dict(x=x.half()), dict(weight=w.double()), dict(residual=r.half()), dict(out_dtype=th.float16)):
        with pytest.raises(TypeError, match='rms_norm'):
            call_norm(**{'x': x, **bad})
    for bad in (x[:, :0], th.zeros(2, 16385, dtype=BF)):
        with pytest.raises(ValueError, match='rms_norm'):
            call_norm(bad)
    for leaf in (dict(x=x.clone().requires_grad_()), dict(x=x, weight=w.clone().requires_grad_()), dict(x=x, residual=r.clone().requires_grad_())):
        with pytest.raises(RuntimeError, match='no backward'):
            call_norm(**leaf, out_dtype=th.int8)
    with pytest.raises(RuntimeError, match='CUDA'):
        call_norm(x, weight=w, residual=r)
    for bad in (dict(p=-0.1), dict(p=1.1), dict(seed=None), dict(seed=-1), dict(seed=1 << 63), dict(residual=r[:3]), dict(seed=th.zeros(2, dtype=th.int64))):
        with pytest.raises(ValueError, match='dropout'):
            call_drop(**{'x': x, 'p': 0.1, 'seed': 1, **bad})
    for bad in (dict(x=x.half()), dict(residual=r.double())):
        with pytest.raises(TypeError, match='dropout'):
            call_drop(**{'x': x, 'p': 0.1, 'seed': 1, **bad})
    with pytest.raises(RuntimeError, match='CUDA'):
        call_drop(x, 0.1, 1)


def test_python_refusals(lib):
    from wind_rwkv.rwkv7 import dropout, rms_norm
    refusals(rms_norm, dropout)


def test_refusals_while_torch_compile_traces(lib):
    from wind_rwkv.rwkv7 import dropout, rms_norm

    def traced(f):
        def call(*a, **k):
            th.compiler.reset()
            return th.compile(lambda: f(*a, **k), backend='eager')()
        return call

    refusals(traced(rms_norm), traced(dropout))


def test_the_generators_words():
    """The tests' own Philox4x32-10 against the published vectors (Random123's known answers)."""
    from philox import words
    assert [int(w) for w in words(0, 4, 0)] == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]
    assert [int(w) for w in words(0, 4, 0, counter=(0xffffffff,) * 4, key=(0xffffffff,) * 2)] == [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]
    assert [int(w) for w in words(0, 4, 0, counter=(0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344), key=(0xa4093822, 0x299f31d0))] == [0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1]
    assert (words(6, 3, 5) == words(0, 12, 5)[6:9]).all()


def test_seeds_are_integers_whether_or_not_they_are_used(lib):
    from wind_rwkv.rwkv7 import dropout, rms_norm
    x = th.zeros(4, 64, dtype=BF)
    for seed in (-1, -2, 1 << 63, 1.5, th.zeros(2, dtype=th.int64), th.zeros(1)):
        for p in (0., 0.5):
            with pytest.raises(ValueError, match='rms_norm: a seed'):
                rms_norm(x, residual=x, p=p, seed=seed)
            with pytest.raises(ValueError, match='dropout: a seed'):
                dropout(x, p, seed)
    for seed in (0, 7, (1 << 63) - 1):
        with pytest.raises(RuntimeError, match='CUDA'):
            rms_norm(x, residual=x, seed=seed)
