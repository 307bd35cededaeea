"""quantize, rms_norm in 8 bits and linear_int8 against their formulas in 64 bits.

Tolerances.  e = 2^-24; u: half a step of the result's type (bf16 2^-8, fp32 2^-24), relative.
  quantize: of bf16 rows q is exact, ties to even (127 x / a is a quotient of 15 by 8 bits); of fp32 rows it may be off by one where 127 x / a is within 127 * 4 e of a half
     (127 x, 1 / a, their product, the remainder's).  scale: a / 127, two roundings.
  linear_int8: the sum is exact; its conversion and each scale one rounding: 3 e |z0|; the bias one e of the sum; activations as in the tests of linear (2^-18 of max(|value|,
     |argument|), |act'| <= L times the argument's error); the residual one e; then u.
  rms_norm in 8 bits: y64 = norm(h) in 64 bits; scale within 42 e of max |y64| / 127; |q scale - y64| <= scale / 2 + 42 e |y64| + 127 * 42 e scale.
"""
import pytest
import torch as th

pytestmark = pytest.mark.gpu

E, U = 2.0 ** -24, {th.bfloat16: 2.0 ** -8, th.float32: 2.0 ** -24}
BF, F32 = th.bfloat16, th.float32
L1 = {None: 1, 'relu': 1, 'tanh': 1, 'sigmoid': 0.25, 'silu': 1.1, 'gelu': 1.13}
F64 = {None: lambda z: z, 'relu': th.relu, 'relu2': lambda z: th.relu(z).square(), 'tanh': th.tanh, 'sigmoid': th.sigmoid,
       'silu': th.nn.functional.silu, 'gelu': lambda z: th.nn.functional.gelu(z, approximate='tanh')}


def check(name, got, want, bound):
    assert got.shape == want.shape, name
    e = (got.double() - want).abs() - bound
    assert bool((e <= 0).all()), f'{name}: {int((e > 0).sum())} of {e.numel()} beyond the bound, the worst by {float(e.max()):.2e}'


def rn(*shape, seed, dtype=F32, std=1.):
    g = th.Generator(device='cuda').manual_seed(seed)
    return (th.randn(*shape, generator=g, device='cuda') * std).to(dtype)


def ints(*shape, seed, lo=-127):
    g = th.Generator(device='cuda').manual_seed(seed)
    t = th.zeros(*shape[:-1], (shape[-1] + 15) // 16 * 16, dtype=th.int8, device='cuda')
    t[..., :shape[-1]] = th.randint(lo, 128, shape, generator=g, device='cuda')
    return t[..., :shape[-1]]


def check_quantized(q8, x):
    q, scale = q8
    assert q.shape == x.shape and q.dtype == th.int8 and scale.shape == x.shape[:-1] and q.stride(-1) == 1 and q.data_ptr() % 16 == 0
    X = x.double()
    a = X.abs().amax(-1, keepdim=True)
    live = a > 2.0 ** -100
    exact = th.where(live, 127 * X / a, 0.)
    off = (q.double() - exact.round()).abs()
    if x.dtype == BF:
        assert not off.any()
    else:
        assert bool((off <= ((exact - exact.floor() - 0.5).abs() <= 127 * 4 * E)).all())
    check('scale', scale, th.where(live, a / 127, 0.)[..., 0], 2 * E * a[..., 0] / 127)


@pytest.mark.parametrize('M,K', [(1, 1), (3, 7), (1, 2048), (5, 16), (700, 24), (257, 203), (40, 333), (24, 8192), (301, 2560), (700, 2047), (350, 4099), (400, 9001), (3, 10000), (2, 16384), (2, 16392), (3, 40001), (1, 131071)])
@pytest.mark.parametrize('dtype', [BF, F32])
def test_quantize(M, K, dtype):
    from wind_rwkv.rwkv7 import quantize
    check_quantized(quantize(rn(M, K, seed=M + K, dtype=dtype)), rn(M, K, seed=M + K, dtype=dtype))
    x = rn(M, K, seed=M * K, dtype=dtype).relu().square()  # the channel mixer's
    check_quantized(quantize(x), x)


def test_quantize_decides_ties_to_even():
    """All bf16 values of two binades beside every maximum of one: 127 x / a meets halves exactly."""
    from wind_rwkv.rwkv7 import quantize
    v = (1 + th.arange(128, device='cuda') / 128)
    rows = th.cat([v, v / 2, v / 4, v / 8, -v / 2], 0)[None].repeat(128, 1)
    rows = th.cat([th.where(rows.abs() <= v[:, None], rows, 0.), v[:, None]], 1).bfloat16()
    half = (127 * rows.double() / rows.double().abs().amax(1, keepdim=True)) % 1 == 0.5
    assert int(half.sum()) > 100
    check_quantized(quantize(rows), rows)


def test_quantize_far_magnitudes_and_what_is_no_number():
    from wind_rwkv.rwkv7 import quantize
    x = rn(12, 100, seed=1)
    x[0] = 0
    x[1] *= 2.0 ** -110
    x[2] *= 2.0 ** -98
    x[3] *= 1e30
    x[4] *= 3.4e38 / x[4].abs().max()
    x[5] = 0
    x[5, 3] = -3.4028234663852886e38
    x[6, 1:] = 0
    check_quantized(quantize(x), x)
    b = x[:7].bfloat16()
    b[4] = b[4].clamp(-3.3e38, 3.3e38)
    b[5, 3] = -3.3e38
    check_quantized(quantize(b), b)
    x[7, 5], x[8, 6], x[9, 7] = float('nan'), float('inf'), -float('inf')
    q, s = quantize(x)
    assert bool(s[7:10].isnan().all()) and not q[7:10].any() and bool(s[10:].isfinite().all()) and bool(s[:7].isfinite().all())


def test_quantize_layouts():
    from wind_rwkv.rwkv7 import quantize
    wide = rn(20, 700, seed=1, dtype=BF)
    for view in (wide[:, 8:264], wide[:, 1:300], wide[::3], wide.t(), wide[:, ::2], wide[:1].expand(20, 700), wide[0], wide.view(4, 5, 700), wide[:0]):
        q, s = quantize(view)
        a, b = quantize(view.clone(memory_format=th.contiguous_format))
        assert th.equal(q, a) and th.equal(s, b) and q.shape == view.shape
    leaf = rn(8, 64, seed=2).requires_grad_()
    q, s = quantize(leaf)
    assert not s.requires_grad


@pytest.mark.parametrize('M,D', [(1, 2048), (3, 7), (700, 16), (500, 2047), (320, 8199), (257, 203), (301, 4096), (2, 16384), (5000, 333)])
@pytest.mark.parametrize('x_t', [BF, F32])
@pytest.mark.parametrize('r_t', [None, BF, F32])
def test_norm_in_8_bits(M, D, x_t, r_t):
    from wind_rwkv.rwkv7 import rms_norm
    x, w = rn(M, D, seed=1, dtype=x_t), 1 + rn(D, seed=2, std=0.3)
    r = None if r_t is None else rn(M, D, seed=3, dtype=r_t, std=2.)
    got = rms_norm(x, w, residual=r, out_dtype=th.int8)
    (q, s), h = got if r is not None else (got, x)
    if r is not None:
        assert th.equal(h, rms_norm(x, w, residual=r)[1])
    H = h.double()
    Y = H / (H.square().mean(-1, keepdim=True) + 1e-5).sqrt() * w.double()
    top = Y.abs().amax(-1)
    check('scale', s, top / 127, 42 * E * top / 127)
    S = s.double()[:, None]
    check('y', q.double() * S, Y, S / 2 + 42 * E * Y.abs() + 127 * 42 * E * S)
    assert q.shape == x.shape and bool((q.abs().amax(-1) == 127).all())


def test_norm_in_8_bits_of_rows_without_numbers():
    from wind_rwkv.rwkv7 import rms_norm
    x = rn(5, 64, seed=1)
    x[0], x[1, 3], x[2, 4] = 0, float('nan'), float('inf')
    q, s = rms_norm(x, out_dtype=th.int8)
    assert float(s[0]) == 0 and not q[:3].any() and bool(s[1:3].isnan().all()) and bool(s[3:].isfinite().all())


def compare(M, N, K, act=None, bias=None, residual=False, out=BF, seed=1, lo=-127, x=None, w=None):
    from wind_rwkv.rwkv7 import linear_int8
    xq, wq = x if x is not None else ints(M, K, seed=seed, lo=lo), w if w is not None else ints(N, K, seed=seed + 1, lo=lo)
    xs, ws = rn(M, seed=seed + 2).abs() * 0.01, rn(N, seed=seed + 3).abs() * 0.3 / (73 * 73 * K ** 0.5 * 0.01)
    b = None if bias is None else rn(N, seed=seed + 4).to(bias)
    r = rn(M, N, seed=seed + 5, dtype=out) if residual else None
    y = linear_int8((xq, xs), (wq, ws), b, act=act, residual=r, out_dtype=out)
    assert y.dtype == out
    acc = xq.double() @ wq.double().T
    z0 = acc * xs.double()[:, None] * ws.double()
    B = 0. if b is None else b.double()
    Z = z0 + B
    ez = 3 * E * z0.abs() + (0. if b is None else E * (Z.abs() + 3 * E * z0.abs()))
    A = F64[act](Z)
    l1 = 2 * (Z.abs() + ez) if act == 'relu2' else L1[act]
    own = 0. if act is None else 2.0 ** -18 * (A.abs() + (0. if act in ('relu', 'relu2') else Z.abs()))
    e = l1 * ez + own
    Y = A + (0. if r is None else r.double())
    e = e + (0. if r is None else E * (Y.abs() + e))
    check('y', y, Y, e + U[out] * (Y.abs() + e))
    return y


SHAPES = [  # rows, columns, k
    (1, 1, 1), (1, 8192, 2048), (3, 77, 203), (16, 129, 1024), (17, 2048, 8192), (33, 1000, 64), (64, 257, 4111), (2, 50001, 96),
    (65, 64, 64), (100, 130, 72), (333, 77, 200), (513, 200, 768), (700, 1000, 136), (40, 1000, 8192), (200, 40, 20000),
    (1, 77, 63), (1, 1000, 203), (2, 33, 4111), (1, 40, 131071), (2, 129, 20000), (1, 50001, 2048),
    (1300, 4096, 80), (1283, 4001, 207), (2500, 2053, 1032), (5000, 96, 2048), (20000, 40, 24), (3328, 1536, 8192), (1536, 8192, 3336)]


@pytest.mark.parametrize('M,N,K', SHAPES)
def test_shapes(M, N, K):
    compare(M, N, K, 'relu2')
    compare(M, N, K, bias=F32, residual=True)
    compare(M, N, K, out=F32)


@pytest.mark.parametrize('act', list(F64))
@pytest.mark.parametrize('M,N,K', [(5, 100, 128), (200, 264, 128), (1400, 3333, 128)])
@pytest.mark.parametrize('residual', [False, True])
def test_activations(act, M, N, K, residual):
    compare(M, N, K, act, BF, residual)


@pytest.mark.parametrize('bias,residual,out', [(None, False, BF), (F32, True, BF), (BF, True, F32), (F32, True, F32)])
@pytest.mark.parametrize('M,N,K', [(1283, 10240, 512), (1283, 10236, 512), (1283, 10235, 512), (8192, 2048, 512)])
def test_wide_results(M, N, K, bias, residual, out):
    compare(M, N, K, 'silu', bias, residual, out)


def test_sums_at_the_ends_of_32_bits():
    """All operands at -128 and at 127, the longest sums: +- 2^31 is nearly reached and nothing wraps or saturates."""
    for M, N in ((1, 40), (3, 70), (130, 70), (300, 2100)):
        K = 131071
        for a, b in ((-128, -128), (-128, 127), (127, 127)):
            x, w = (th.full((n, 131072), v, dtype=th.int8, device='cuda')[:, :K] for n, v in ((M, a), (N, b)))
            compare(M, N, K, out=F32, x=x, w=w)


def test_what_lies_behind_the_rows_does_not_count():
    """k beyond K in wider rows, rows beyond the last: operands inside buffers of other values."""
    from wind_rwkv.rwkv7 import linear_int8
    for M, N, K in ((1, 50, 203), (2, 77, 90), (3, 77, 203), (130, 200, 130), (1283, 4100, 72)):
        x, w = ints(M, K, seed=1), ints(N, K, seed=2)
        X, W = (th.full((n + 4, K + 150 - K % 16 - 6 + 16 & ~15), 99, dtype=th.int8, device='cuda') for n in (M, N))
        X[2:2 + M, 16:16 + K], W[2:2 + N, 16:16 + K] = x, w
        xs, ws = rn(M, seed=3), rn(N, seed=4)
        assert th.equal(linear_int8((X[2:2 + M, 16:16 + K], xs), (W[2:2 + N, 16:16 + K], ws)), linear_int8((x, xs), (w, ws)))
        assert th.equal(linear_int8((X[2:2 + M, 16:16 + K], xs), (w.contiguous(), ws)), linear_int8((x, xs), (w, ws)))   # rows that are copied


def test_results_go_where_they_belong():
    from wind_rwkv.rwkv7 import _lib
    L = _lib.lib()
    for M, N, K in ((1, 77, 64), (2, 40, 72), (5, 77, 64), (40, 264, 64), (130, 77, 72), (200, 264, 512), (1283, 4100, 64), (1283, 4101, 64), (3000, 3333, 64)):
        x, w = ints(M, K, seed=1), ints(N, K, seed=2)
        xs, ws = rn(M, seed=3), rn(N, seed=4)
        Y = (x.double() @ w.double().T) * xs.double()[:, None] * ws.double()
        for f32 in (0, 1):
            for ldy in ((N + 7) // 8 * 8 + 16, N + 3):
                y = th.full((M + 2, ldy), 7., dtype=F32 if f32 else BF, device='cuda')
                work = th.empty(max(16, L.wkv7_linear_int8_workspace_bytes(M, N, K)), dtype=th.uint8, device='cuda')
                to = y.data_ptr() + ldy * y.element_size()
                assert L.wkv7_linear_int8(x.data_ptr(), xs.data_ptr(), w.data_ptr(), ws.data_ptr(), None, None, to, M, N, K, x.stride(0), w.stride(0), 0, ldy, 0, f32,
                                          work.data_ptr(), _lib.stream_of(x)) == 0
                assert bool((y[0] == 7).all()) and bool((y[-1] == 7).all()) and bool((y[:, N:] == 7).all())
                check('y', y[1:-1, :N], Y, (3 * E + U[y.dtype] * (1 + 3 * E)) * Y.abs())


def test_scales_of_zero_and_no_number():
    from wind_rwkv.rwkv7 import linear_int8
    for M, N in ((5, 100), (200, 264), (1400, 3333)):
        x, w = ints(M, 64, seed=1), ints(N, 64, seed=2)
        x[3] = 0
        xs, ws = th.ones(M, device='cuda'), th.ones(N, device='cuda')
        xs[2], xs[3], ws[7] = 0, float('nan'), 0
        y = linear_int8((x, xs), (w, ws))
        assert not y[2].any() and bool(y[3].isnan().all()) and not y[:3, 7].any() and bool(y[[0, 1, 4]].isfinite().all())


def test_large_offsets():
    """Results beyond 2^31 elements, in a weight beyond 2^31 bytes."""
    from wind_rwkv.rwkv7 import linear_int8
    M, N, K = 66000, 33000, 32
    x, w, xs, ws = ints(M, K, seed=1), ints(N, K, seed=2), rn(M, seed=3), rn(N, seed=4)
    y = linear_int8((x, xs), (w, ws))
    for rows in (slice(0, 3), slice(M - 3, M)):
        Y = (x[rows].double() @ w.double().T) * xs[rows].double()[:, None] * ws.double()
        check('y', y[rows], Y, (3 * E + U[BF] * (1 + 3 * E)) * Y.abs())
    del y
    N, K = 40000, 65536
    w = th.zeros(N, K, dtype=th.int8, device='cuda')
    w[-2:] = ints(2, K, seed=5)
    x = ints(2, K, seed=6)
    y = linear_int8((x, xs[:2]), (w, th.ones(N, device='cuda')), out_dtype=F32)
    Y = (x.double() @ w[-2:].double().T) * xs[:2].double()[:, None]
    check('y', y[:, -2:], Y, 3 * E * Y.abs())
    assert not y[:, :-2].any()


def test_streams_graphs_and_call_to_call():
    from wind_rwkv.rwkv7 import linear_int8, quantize, rms_norm
    for M, N, K in ((5, 8192, 2048), (37, 77, 203), (3328, 1536, 4096)):
        x, r, w8 = rn(M, K, seed=1, dtype=BF), rn(M, K, seed=2, dtype=BF), (ints(N, K, seed=3), rn(N, seed=4).abs())

        def step():
            q8, h = rms_norm(x, residual=r, out_dtype=th.int8)
            return linear_int8(q8, w8, act='relu2'), linear_int8(quantize(h), w8)

        want = step()
        sides = [th.cuda.Stream() for _ in range(2)]
        for s in sides:
            s.wait_stream(th.cuda.current_stream())
        outs = []
        for _ in range(3):
            for s in sides:
                with th.cuda.stream(s):
                    outs.append(step())
        th.cuda.synchronize()
        graphs, caught = [th.cuda.CUDAGraph() for _ in range(2)], []
        for g in graphs:
            with th.cuda.graph(g):
                caught.append(step())
        for g in graphs + graphs:
            g.replay()
        for got in outs + caught:
            assert all(th.equal(a, b) for a, b in zip(got, want))
        x.copy_(x.flip(0))
        want = step()
        for g, got in zip(graphs, caught):
            g.replay()
            assert all(th.equal(a, b) for a, b in zip(got, want))


def test_batch_dimensions_and_empty():
    from wind_rwkv.rwkv7 import linear_int8, quantize
    w8 = quantize(rn(40, 100, seed=1))
    x = rn(3, 5, 100, seed=2, dtype=BF)
    y = linear_int8(quantize(x), w8, residual=th.zeros(3, 5, 40, dtype=BF, device='cuda'))
    assert th.equal(y.view(15, 40), linear_int8(quantize(x.view(15, 100)), w8)) and th.equal(linear_int8(quantize(x[1, 2]), w8), y[1, 2])
    assert linear_int8(quantize(x[:0]), w8).shape == (0, 5, 40)


def test_torch_compile_and_the_python_form():
    from wind_rwkv.rwkv7 import linear_int8, quantize, rms_norm
    from wind_rwkv.rwkv7.rwkv7_int8 import fw_int8, rows8
    x, r, w, b = rn(9, 203, seed=1, dtype=BF), rn(9, 203, seed=2, dtype=BF), quantize(rn(70, 203, seed=3)), rn(70, seed=4)

    def f(x, r, b):
        q8, h = rms_norm(x, residual=r, out_dtype=th.int8)
        return linear_int8(q8, w, b, act='relu2') * 2, linear_int8(quantize(h), w, out_dtype=F32), h

    want = f(x, r, b)
    th.compiler.reset()
    got = th.compile(f, backend='aot_eager', fullgraph=True)(x, r, b)
    assert all(th.equal(p, q) for p, q in zip(want, got))
    q, s = rows8(x)
    assert th.equal(q[:, :203], quantize(x).q) and th.equal(s, quantize(x).scale)
    assert th.equal(fw_int8(q[:, :203], s, *w, b, None, 6, False), linear_int8(quantize(x), w, b, act='gelu'))


def test_a_block_in_8_bits():
    """As a program runs them: norm, channel mixer in 8 bits, the stream going on; against the same quantized steps in 64 bits."""
    from wind_rwkv.rwkv7 import linear_int8, quantize, rms_norm
    for M in (1, 24, 700):
        D, F = 512, 2048
        h = rn(M, D, seed=1, dtype=BF)
        gain, wk, wv = 1 + rn(D, seed=2, std=0.2), quantize(rn(F, D, seed=3, std=D ** -0.5)), quantize(rn(D, F, seed=4, std=F ** -0.5))
        mixed = rn(M, D, seed=5, dtype=BF)
        H = h.double()
        for _ in range(2):
            q8, h = rms_norm(mixed, gain, residual=h, out_dtype=th.int8)
            k = linear_int8(q8, wk, act='relu2')
            h = linear_int8(quantize(k), wv, residual=h)
            H = H + mixed.double()
            Y = H / (H.square().mean(-1, keepdim=True) + 1e-5).sqrt() * gain.double()
            W = [t.q.double() * t.scale.double()[:, None] for t in (wk, wv)]
            H = H + th.relu(Y @ W[0].T).square() @ W[1].T
        # 8 bits of y and of relu2's values: a rounding of scale / 2 in each of D and F terms; the bf16 stream's two roundings a step
        assert float((h.double() - H).norm() / H.norm()) < 2e-2


BATCHES = (1, 2, 5, 24, 64, 70, 130, 300, 700, 1283, 4096, 8192)  # the rows' kernel, tiles along the columns and the rows, cut or whole, pairs both ways


@pytest.mark.parametrize('N,K', [(4096, 1024), (4001, 1024), (1000, 8192)])
def test_a_row_has_the_same_bits_in_every_batch(N, K):
    from wind_rwkv.rwkv7 import linear_int8
    x, w, xs, ws, b = ints(8192, K, seed=1), ints(N, K, seed=2), rn(8192, seed=3), rn(N, seed=4), rn(N, seed=5)
    for bias in (None, b):
        want = linear_int8((x, xs), (w, ws), bias, out_dtype=F32)
        for M in BATCHES[:-1]:
            assert th.equal(linear_int8((x[:M], xs[:M]), (w, ws), bias, out_dtype=F32), want[:M]), M


@pytest.mark.parametrize('act', [a for a in F64 if a])
@pytest.mark.parametrize('N', [4096, 4001])
def test_a_row_has_the_same_bits_behind_the_epilogue(act, N):
    from wind_rwkv.rwkv7 import linear_int8
    K = 1024
    x, w, xs, ws, b = ints(8192, K, seed=1), ints(N, K, seed=2), rn(8192, seed=3, std=1e-3), rn(N, seed=4, std=1e-2), rn(N, seed=5)
    for out in (F32, BF):
        r = rn(8192, N, seed=6, dtype=out)
        want = linear_int8((x, xs), (w, ws), b, act=act, residual=r, out_dtype=out)
        for M in BATCHES[:-1]:
            assert th.equal(linear_int8((x[:M], xs[:M]), (w, ws), b, act=act, residual=r[:M], out_dtype=out), want[:M]), M


@pytest.mark.parametrize('N,K', [(4096, 1024), (4001, 1024), (1000, 8192)])
def test_rows_near_the_end_of_fp32(N, K):
    """Scales of 1e36: sum xs is beyond fp32, the result with the weight's scales is not."""
    from wind_rwkv.rwkv7 import linear_int8, quantize
    w8 = quantize(rn(N, K, seed=2, std=1e-4))
    x = rn(8192, K, seed=1)
    x[0] *= 2e37
    x[1] = 3e38
    x8 = quantize(x)
    assert float(x8.scale[1]) > 2e36
    for M in BATCHES:
        rows = slice(0, min(M, 3))
        Y = (x8.q[rows].double() @ w8.q.double().T) * w8.scale.double() * x8.scale[rows].double()[:, None]  # (the sums of integers are exact)
        assert float(Y[:1].abs().max()) > 1e33 and float(Y.abs().max()) < 2.0 ** 127
        check('y', linear_int8((x8.q[:M], x8.scale[:M]), w8, out_dtype=F32)[rows], Y, 3.01 * E * Y.abs())


def test_forward_mode_tangents_are_refused():
    import torch.autograd.forward_ad as fw
    from wind_rwkv.rwkv7 import linear_int8, quantize, rms_norm
    x8, w8, x, r = (ints(4, 64, seed=1), rn(4, seed=2)), (ints(16, 64, seed=3), rn(16, seed=4)), rn(4, 64, seed=5), rn(4, 16, seed=6, dtype=BF)
    want = linear_int8(x8, w8, residual=r), *quantize(x), *rms_norm(x, out_dtype=th.int8)
    with fw.dual_level(), th.no_grad():
        def dual(t):
            return fw.make_dual(t, th.ones_like(t))
        for call in (lambda: linear_int8(x8, w8, residual=dual(r)), lambda: linear_int8((x8[0], dual(x8[1])), w8), lambda: linear_int8(x8, (w8[0], dual(w8[1]))),
                     lambda: linear_int8(x8, w8, dual(rn(16, seed=7))), lambda: quantize(dual(x)), lambda: rms_norm(dual(x), out_dtype=th.int8),
                     lambda: rms_norm(x, residual=dual(x), out_dtype=th.int8), lambda: rms_norm(x, dual(rn(64, seed=8)), out_dtype=th.int8)):
            with pytest.raises(RuntimeError, match='tangent'):
                call()
        got = linear_int8(x8, w8, residual=r), *quantize(x), *rms_norm(x, out_dtype=th.int8)
    assert all(th.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize('M,N,K', [(1, 77, 64), (2, 1000, 203), (24, 2048, 8192), (64, 257, 4111), (70, 1000, 8192), (130, 4096, 1024), (200, 40, 20000), (300, 4001, 8192), (700, 4096, 1024),
                                   (700, 4001, 1024), (1283, 1000, 8192), (4096, 1000, 8192), (4096, 4001, 1024), (4096, 4096, 1024)])
def test_y_may_be_its_own_residual(M, N, K):
    from wind_rwkv.rwkv7 import _lib
    L = _lib.lib()
    x, w, xs, ws = ints(M, K, seed=1), ints(N, K, seed=2), rn(M, seed=3), rn(N, seed=4)
    work = th.empty(max(16, L.wkv7_linear_int8_workspace_bytes(M, N, K)), dtype=th.uint8, device='cuda')
    for f32 in (0, 1):
        for ld in (N, N + 3, (N + 15) // 8 * 8):
            r = rn(M, ld, seed=5, std=1e3, dtype=F32 if f32 else BF)
            out = []
            for y in (th.zeros_like(r), r.clone()):
                residual = r if not out else y
                assert L.wkv7_linear_int8(x.data_ptr(), xs.data_ptr(), w.data_ptr(), ws.data_ptr(), None, residual.data_ptr(), y.data_ptr(), M, N, K, x.stride(0), w.stride(0), ld, ld,
                                          2, f32, work.data_ptr(), _lib.stream_of(x)) == 0
                out.append(y)
            assert th.equal(out[0][:, :N], out[1][:, :N]) and th.equal(out[1][:, N:], r[:, N:])
