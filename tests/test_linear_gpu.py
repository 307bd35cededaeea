"""linear = act(x w^T + bias) + residual and its gradients against the formula in 64 bits on the same bf16 values.

Tolerances, element by element.  u = 2^-8: a rounding to bf16, relative.  A sum of K products on the tensor core, K/16 steps of 16 with fp32 rounding
or cutting (2^-22 of the running magnitude, two steps more for bias and residual): acc(K) = (K/16 + 2) 2^-22 of the sum of the products' magnitudes.
Activations are formed with errors of a few 2^-21 of max(|value|, |argument|) (hardware exponential and reciprocal): 2^-18 is allowed.
  y:  |act'| <= L times the error of z, the activation's own, u |y| for its rounding (fp32 y: 2^-22 |y|)
  dz: |dy| times the error of act': L2 >= |act''| times that of z (bf16 z: u |z| more), from y (relu2): 2 sqrt(y (1 + u)), i.e. u/2 relative;
      u |dz| for its rounding to bf16
  dx, dw: the sums of the bounds on dz times the other operand's magnitudes, acc of the sum, u of the result;  dbias: dz's without its rounding, fp32 with z in fp32
"""
import pytest
import torch as th

pytestmark = pytest.mark.gpu

U = 2.0 ** -8
L1 = {None: 1, 'relu': 1, 'tanh': 1, 'sigmoid': 0.25, 'silu': 1.1, 'gelu': 1.13}
L2 = {None: 0, 'relu': 0, 'tanh': 0.77, 'sigmoid': 0.1, 'silu': 0.5, 'gelu': 1.13}
F64 = {None: lambda z: z, 'relu': th.relu, 'relu2': lambda z: th.relu(z).square(), 'tanh': th.tanh, 'sigmoid': th.sigmoid,
       'silu': th.nn.functional.silu, 'gelu': lambda z: th.nn.functional.gelu(z, approximate='tanh')}


def acc(K):
    return (K / 16 + 2) * 2.0 ** -22


def inputs(M, N, K, bias, residual, out, seed):
    g = th.Generator(device='cuda').manual_seed(seed)

    def rn(*s):
        return th.randn(*s, generator=g, device='cuda')

    x, w = rn(M, K).bfloat16(), (rn(N, K) / K ** 0.5).bfloat16()
    return x, w, rn(N).to(bias) if bias else None, rn(M, N).to(out) if residual else None, rn(M, N).to(out)


def check(name, got, want, bound):
    assert got.shape == want.shape, name
    e = (got.double() - want).abs() - bound
    assert bool((e <= 0).all()), f'{name}: {int((e > 0).sum())} of {e.numel()} beyond the bound, the worst by {float(e.max()):.2e}'


def compare(x, w, b, r, dy, act, out=th.bfloat16, call=None):
    """One call with its backward against the formula."""
    from wind_rwkv.rwkv7 import linear
    K = w.shape[1]
    leaves = [None if t is None else t.detach().requires_grad_() for t in (x, w, b, r)]
    y = (call or linear)(leaves[0], leaves[1], leaves[2], act=act, residual=leaves[3], out_dtype=out)
    assert y.dtype == out
    grads = iter(th.autograd.grad(y, [t for t in leaves if t is not None], dy))
    X, W = x.detach().double().reshape(-1, K), w.detach().double()
    N = W.shape[0]
    Z = X @ W.T + (0 if b is None else b.detach().double())
    mag = X.abs() @ W.abs().T + (0 if b is None else b.detach().double().abs())
    Zr = Z.clone().requires_grad_()
    A = F64[act](Zr)
    R = 0 if r is None else r.detach().double().reshape(-1, N)
    Y = A.detach() + R
    D, = th.autograd.grad(A.sum(), Zr)
    ez = acc(K) * mag
    l1 = 2 * (Z.abs() + ez) if act == 'relu2' else L1[act]
    own = 0 if act is None else 2.0 ** -18 * (A.detach().abs() + (0 if act in ('relu', 'relu2') else Z.abs()))
    e = l1 * ez + own
    round_y = U if out == th.bfloat16 else 2.0 ** -22
    check('y', y.reshape(-1, N), Y, e + round_y * (Y.abs() + e) + (0 if r is None else 2.0 ** -22 * R.abs()))
    DY = dy.double().reshape(-1, N)
    DZ = DY * D
    if act == 'relu2':
        ed = 2 * ez + D * U + 2 * (Z.abs() <= ez) * ez
    elif act == 'relu':
        ed = (Z.abs() <= ez).double()
    else:
        ed = L2[act] * (ez + U * Z.abs()) + (0 if act is None else 2.0 ** -18 * (1 + Z.abs()))
    # a bias in fp32: its gradient's terms from an argument in fp32
    edb = 2 * ez + 2.0 ** -22 * Z.abs() if act == 'relu2' else (ed if act == 'relu' else L2[act] * ez + (0 if act is None else 2.0 ** -18 * (1 + Z.abs())))
    edb = DY.abs() * (edb if b is not None and b.dtype == th.float32 else ed)
    edz = DY.abs() * ed
    edzr = edz + U * (DZ.abs() + edz)
    M = X.shape[0]
    dx = next(grads)
    check('dx', dx.reshape(-1, K), DZ @ W, (edzr @ W.abs()) * (1 + U) + acc(N) * (DZ.abs() @ W.abs()) + U * (DZ @ W).abs())
    check('dw', next(grads), DZ.T @ X, (edzr.T @ X.abs()) * (1 + U) + acc(M) * (DZ.abs().T @ X.abs()) + U * (DZ.T @ X).abs())
    if b is not None:
        s = DZ.sum(0)
        round_b = U if b.dtype == th.bfloat16 else 0
        check('dbias', next(grads), s, edb.sum(0) * (1 + U) + (M + 8) * 2.0 ** -24 * DZ.abs().sum(0) + round_b * s.abs())
    if r is not None:
        assert th.equal(next(grads), dy)
    return y


SHAPES = [  # rows, columns, k
    (1, 1, 8), (1, 8192, 2048), (3, 77, 200), (16, 129, 1024), (17, 2048, 8192), (33, 1000, 64), (64, 257, 4104),   # few rows
    (65, 64, 64), (100, 130, 72), (333, 77, 200), (513, 200, 768), (700, 1000, 136),                                # tiles
    (1300, 4096, 72), (1283, 4001, 200), (2500, 2053, 1032), (5000, 96, 2048), (20000, 40, 24), (9000, 40, 200)]                     # pairs, and mixtures in the backward


@pytest.mark.parametrize('M,N,K', SHAPES)
def test_shapes(M, N, K):
    compare(*inputs(M, N, K, None, False, th.bfloat16, M + N + K), 'relu2')
    compare(*inputs(M, N, K, th.float32, True, th.bfloat16, M + N + K + 1), None)


@pytest.mark.parametrize('act', list(F64))
@pytest.mark.parametrize('M,N,K', [(5, 100, 128), (200, 264, 128), (1400, 3333, 128)])
@pytest.mark.parametrize('residual', [False, True])
def test_activations(act, M, N, K, residual):
    compare(*inputs(M, N, K, th.bfloat16, residual, th.bfloat16, 7), act)


@pytest.mark.parametrize('act', [None, 'relu2', 'tanh'])
@pytest.mark.parametrize('M,N,K', [(7, 50001, 64), (300, 203, 256), (1400, 3333, 64), (1536, 4096, 64)])
def test_fp32_output(act, M, N, K):
    compare(*inputs(M, N, K, th.float32, True, th.float32, 9), act, out=th.float32)


@pytest.mark.parametrize('M,N,K', [(3328, 1536, 8192), (1536, 8192, 3336), (60000, 80, 200), (30000, 33, 264), (40, 1000, 8192)])
def test_long_sums(M, N, K):
    """Sums that are shared out: over the clusters of a tile, over the units of the tiles of the last round, and both in the backward."""
    compare(*inputs(M, N, K, th.float32, True, th.bfloat16, 21), 'silu')
    compare(*inputs(M, N, K, None, False, th.bfloat16, 22), None)


@pytest.mark.parametrize('act', ['relu2', 'tanh'])
@pytest.mark.parametrize('bias,residual,out', [(None, False, th.bfloat16), (th.float32, True, th.bfloat16), (th.bfloat16, True, th.float32), (th.float32, True, th.float32)])
@pytest.mark.parametrize('M,N,K', [(1283, 10240, 256), (1283, 10236, 256), (1283, 10235, 256)])
def test_columns_of_y_along_the_accumulators_rows(M, N, K, act, bias, residual, out):
    """Shapes that the pairs take turned over, with every kind of result: aligned rows (bulk stores), rows that only fp32 ones are, odd ones."""
    compare(*inputs(M, N, K, bias, residual, out, 31), act, out=out)


def test_results_go_where_they_belong():
    """Nothing is written beside y, z, dx or dw: C entry points with outputs inside larger buffers."""
    from wind_rwkv.rwkv7 import _lib
    L = _lib.lib()
    for M, N, K in ((5, 77, 64), (40, 264, 64), (130, 77, 72), (200, 264, 512), (1283, 4100, 64), (1283, 4101, 64), (3000, 3333, 64)):
        x, w, _, _, dy = inputs(M, N, K, None, False, th.bfloat16, 2)
        n8 = (N + 7) // 8 * 8
        for f32 in (0, 1):
            ldy = n8 + 16
            y = th.full((M + 2, ldy), 7., dtype=th.float32 if f32 else th.bfloat16, device='cuda')
            z = th.full((M + 2, n8 + 8), 7., dtype=th.bfloat16, device='cuda')
            ws = th.empty(max(16, L.wkv7_linear_fwd_workspace_bytes(M, N, K)), dtype=th.uint8, device='cuda')
            rc = L.wkv7_linear_fwd(x.data_ptr(), w.data_ptr(), None, None, y[1:].data_ptr(), z[1:].data_ptr(), M, N, K, K, K, 0, ldy, n8 + 8, 5, f32, ws.data_ptr(),
                                   _lib.stream_of(x))
            assert rc == 0
            ref = x.double() @ w.double().T
            assert bool((y[0] == 7).all()) and bool((y[-1] == 7).all()) and bool((y[:, N:] == 7).all())
            assert bool((z[0] == 7).all()) and bool((z[-1] == 7).all()) and bool((z[:, n8:] == 7).all())
            tol = U * ref.abs() + acc(K) * (x.double().abs() @ w.double().abs().T)
            assert bool(((z[1:-1, :N].double() - ref).abs() <= tol).all())
            check('y', y[1:-1, :N], F64['silu'](ref), U * F64['silu'](ref).abs() + 1.1 * acc(K) * (x.double().abs() @ w.double().abs().T) + 2. ** -17 * (1 + ref.abs()))
        d = th.full((M + N + 3, K), 7., dtype=th.bfloat16, device='cuda')
        dx, dw = d[1:M + 1], d[M + 2:M + N + 2]
        ws = th.empty(L.wkv7_linear_bwd_workspace_bytes(M, N, K), dtype=th.uint8, device='cuda')
        rc = L.wkv7_linear_bwd(x.data_ptr(), w.data_ptr(), None, dy.data_ptr(), dx.data_ptr(), dw.data_ptr(), None, M, N, K, K, K, N, N, 0, 0, ws.data_ptr(), _lib.stream_of(x))
        assert rc == 0
        assert bool((d[0] == 7).all()) and bool((d[M + 1] == 7).all()) and bool((d[-1] == 7).all())
        D, X, W = dy.double(), x.double(), w.double()
        check('dx', dx, D @ W, U * (D @ W).abs() + (U + acc(N)) * (D.abs() @ W.abs()) * (1 if N % 8 else 0.5))
        check('dw', dw, D.T @ X, U * (D.T @ X).abs() + acc(M) * (D.abs().T @ X.abs()))


def test_large_offsets():
    """Results and gradients beyond 2^31 elements."""
    from wind_rwkv.rwkv7 import linear
    M, N, K = 66000, 33000, 16
    x, w = [inputs(n, 1, K, None, False, th.bfloat16, n)[0] for n in (M, N)]
    x.requires_grad_()
    y = linear(x, w, act='relu2')
    for rows in (slice(0, 3), slice(M - 3, M)):
        ref = th.relu(x.detach()[rows].double() @ w.double().T).square()
        check('y', y[rows], ref, U * ref + 2.0 ** -18 * (1 + ref) * K)
    dy = th.zeros_like(y)
    dy[M - 2, N - 5:] = 1.
    dx, = th.autograd.grad(y, x, dy)
    z = th.relu(x.detach()[M - 2].double() @ w[N - 5:].double().T)
    ref = (2 * z) @ w[N - 5:].double()
    check('dx', dx[M - 2], ref, 3 * U * ((2 * z) @ w[N - 5:].double().abs()) + 1e-6)
    assert not dx[:M - 2].any() and not dx[M - 1].any()


def test_without_workspace():
    """wkv7_linear_fwd with a null workspace: the same sums in another order."""
    from wind_rwkv.rwkv7 import _lib
    L = _lib.lib()
    M, N, K = 3328, 1536, 8192
    x, w, _, _, _ = inputs(M, N, K, None, False, th.bfloat16, 2)
    y = th.empty(M, N, dtype=th.bfloat16, device='cuda')
    assert L.wkv7_linear_fwd(x.data_ptr(), w.data_ptr(), None, None, y.data_ptr(), None, M, N, K, K, K, N, N, 0, 0, 0, None, _lib.stream_of(x)) == 0
    ref = x.double() @ w.double().T
    check('y', y, ref, U * ref.abs() + acc(K) * (x.double().abs() @ w.double().abs().T))


def test_training_step_in_a_graph():
    """Forward and backward captured together and replayed on other inputs."""
    from wind_rwkv.rwkv7 import linear
    for M, N, K in ((37, 77, 200), (1300, 4096, 512)):
        x, w, b, r, dy = inputs(M, N, K, th.float32, True, th.bfloat16, 5)

        def step(x, w, b, r):
            leaves = [t.detach().requires_grad_() for t in (x, w, b, r)]
            y = linear(leaves[0], leaves[1], leaves[2], act='gelu', residual=leaves[3])
            return [y.detach(), *th.autograd.grad(y, leaves, dy)]

        side = th.cuda.Stream()
        side.wait_stream(th.cuda.current_stream())
        with th.cuda.stream(side):
            step(x, w, b, r)
        th.cuda.current_stream().wait_stream(side)
        graph = th.cuda.CUDAGraph()
        with th.cuda.graph(graph):
            out = step(x, w, b, r)
        for _ in range(2):
            x.copy_(x.flip(0))
            graph.replay()
            assert all(th.equal(a, c) for a, c in zip(out, step(x, w, b, r)))


def test_large_arguments():
    """Activations far out on both sides: exponentials that overflow and vanish."""
    x, w, _, _, dy = inputs(70, 96, 64, None, False, th.bfloat16, 3)
    for act in F64:
        compare(x * 64, w, None, None, dy, act)
        if act != 'relu2':  # (whose values leave the range)
            compare(x * 1e19, w, None, None, dy, act)


@pytest.mark.parametrize('act', ['sigmoid', 'silu', 'gelu', 'tanh'])
def test_derivatives_to_their_own_size(act):
    """act' where it is small, relative to it: z is an fp32 bias alone, and its gradient, of one row, is act'(z) in fp32.  With s = sigmoid(u), q = 1 - s, in units of 2^-24: the exponential 4,
    its argument a |u| (product and constant 1.25; gelu's u 7 more, tanh's the same), reciprocal 2 and its argument 1, products; each of s and q is off by E = 13 + a |u| at most."""
    from wind_rwkv.rwkv7 import linear
    z = th.linspace(-6, 6, 4001) if act == 'gelu' else th.linspace(-24, 24, 4001)
    b = z.cuda().requires_grad_()
    x, w = th.zeros(1, 8, dtype=th.bfloat16, device='cuda'), th.zeros(4001, 8, dtype=th.bfloat16, device='cuda')
    y = linear(x, w, b, act=act, out_dtype=th.float32)
    got, = th.autograd.grad(y, b, th.ones_like(y))
    z = b.detach().double()
    C = 2 * (2 / th.pi) ** 0.5
    u = {'gelu': C * (z + 0.044715 * z ** 3), 'tanh': 2 * z}.get(act, z)
    E = (13 + (8.25 if act == 'gelu' else 1.25) * u.abs()) * 2.0 ** -24
    s, q = th.sigmoid(u), th.sigmoid(-u)
    if act in ('sigmoid', 'tanh'):
        want = s * q * (4 if act == 'tanh' else 1)
        bound = 2 * E * want
    else:
        du = C * (1 + 3 * 0.044715 * z ** 2) if act == 'gelu' else 1
        want = s + z * s * q * du
        bound = (2 * E + 8 * 2.0 ** -24) * (s + z.abs() * s * q * du)
    check(act, got, want, bound)


def test_layouts():
    """Rows that lie in wider tensors, batch dimensions, orders and alignments that are copied."""
    x, w, b, r, dy = inputs(60, 72, 64, th.float32, True, th.bfloat16, 5)
    wide = th.zeros(60, 160, dtype=th.bfloat16, device='cuda')
    wide[:, 8:72] = x
    off = th.zeros(60, 160, dtype=th.bfloat16, device='cuda')
    off[:, 1:65] = x
    ww = th.zeros(72, 96, dtype=th.bfloat16, device='cuda')
    ww[:, :64] = w
    rr = th.zeros(60, 75, dtype=th.bfloat16, device='cuda')
    rr[:, 3:] = r
    first = compare(x, w, b, r, dy, 'silu')
    for xs in (wide[:, 8:72], off[:, 1:65], x.t().contiguous().t()):
        for ws in (ww[:, :64], w.t().contiguous().t()):
            assert th.equal(compare(xs, ws, b, rr[:, 3:], dy, 'silu'), first)
    assert th.equal(compare(x, w, b, r.t().contiguous().t(), dy.t().contiguous().t(), 'silu'), first)
    y3 = compare(x.view(3, 20, 64), w, b, r.view(3, 20, 72), dy.view(3, 20, 72), 'silu')
    assert y3.shape == (3, 20, 72) and th.equal(y3.view(60, 72), first)
    x4 = x.view(3, 20, 64).transpose(0, 1)
    y4 = compare(x4, w, b, r.view(3, 20, 72).transpose(0, 1), dy.view(3, 20, 72).transpose(0, 1), 'silu')
    assert th.equal(y4.transpose(0, 1).reshape(60, 72), first)
    one = compare(x[0], w, b, r[0], dy[0], 'silu')
    assert one.shape == (72,)
    bb = th.zeros(144, device='cuda')
    bb[::2] = b
    assert th.equal(compare(x, w, bb[::2], r, dy, 'silu'), first)


@pytest.mark.parametrize('M,N,K', [(20, 77, 64), (200, 77, 72), (1300, 4099, 72)])
def test_what_lies_beside_rows_is_not_read(M, N, K):
    """NaN behind the rows of x, w, the residual and dy, whose pitches the copies can take as they are."""
    x, w, b, r, dy = inputs(M, N, K, th.float32, True, th.bfloat16, 5)

    def wide(t):
        n = (t.shape[1] + 7) // 8 * 8 + 8
        o = th.full((t.shape[0] + 1, n), float('nan'), dtype=t.dtype, device='cuda')
        o[:-1, :t.shape[1]] = t
        return o[:-1, :t.shape[1]]

    for act in (None, 'relu2'):
        first = compare(x, w, b, r, dy, act)
        assert th.equal(compare(wide(x), wide(w), b, wide(r), wide(dy), act), first)


def test_empty():
    from wind_rwkv.rwkv7 import linear
    x = th.zeros(0, 64, dtype=th.bfloat16, device='cuda', requires_grad=True)
    w = th.ones(9, 64, dtype=th.bfloat16, device='cuda', requires_grad=True)
    b = th.ones(9, device='cuda', requires_grad=True)
    y = linear(x, w, b, act='gelu')
    assert y.shape == (0, 9)
    dx, dw, db = th.autograd.grad(y, (x, w, b), th.zeros_like(y))
    assert dx.shape == (0, 64) and not dw.any() and not db.any()


def test_only_what_is_wanted():
    from wind_rwkv.rwkv7 import linear
    x, w, b, r, dy = inputs(40, 24, 64, th.float32, True, th.bfloat16, 5)
    full = [t.clone().requires_grad_() for t in (x, w, b, r)]
    want = th.autograd.grad(linear(full[0], full[1], full[2], act='tanh', residual=full[3]), full, dy)
    for i in range(4):
        ins = [t.clone() for t in (x, w, b, r)]
        ins[i].requires_grad_()
        got, = th.autograd.grad(linear(ins[0], ins[1], ins[2], act='tanh', residual=ins[3]), ins[i], dy)
        assert th.equal(got, want[i])
    ins = [t.clone() for t in (x, w, r)]
    ins[2].requires_grad_()
    got, = th.autograd.grad(linear(ins[0], ins[1], act='tanh', residual=ins[2]), ins[2], dy)
    assert th.equal(got, dy)


def test_gradient_against_differences():
    """The derivative along one direction of all inputs: a central difference of the 64-bit formula against the gradients.  Each gradient is off by
    at most the bounds above, of which the largest part, a few u relative to the sum of the terms' magnitudes, is allowed here."""
    x, w, b, r, dy = inputs(48, 40, 64, th.float32, True, th.bfloat16, 11)
    from wind_rwkv.rwkv7 import linear
    for act in F64:
        leaves = [t.clone().requires_grad_() for t in (x, w, b, r)]
        grads = th.autograd.grad(linear(leaves[0], leaves[1], leaves[2], act=act, residual=leaves[3]), leaves, dy)
        g = th.Generator(device='cuda').manual_seed(1)
        dirs = [th.randn(t.shape, generator=g, device='cuda', dtype=th.float64) for t in leaves]

        def f(h):
            X, W, B, R = [t.detach().double() + h * d for t, d in zip(leaves, dirs)]
            return ((F64[act](X @ W.T + B) + R) * dy.double()).sum()

        num = (f(1e-5) - f(-1e-5)) / 2e-5
        got = sum((a.double() * d).sum() for a, d in zip(grads, dirs))
        scale = sum((a.double() * d).abs().sum() for a, d in zip(grads, dirs))
        assert abs(float(got - num)) <= 4 * U * float(scale)


@pytest.mark.parametrize('B,T,C,F', [(1, 1, 128, 512), (3, 77, 192, 640), (2, 700, 512, 2048)])
def test_channel_mixer_training(B, T, C, F):
    """Both halves of a channel mixer, as a model trains them: x + relu2(x wk^T) wv^T.  Between the inputs and each gradient lie at most six roundings to bf16
    (h, y; dh and its dz; the gradient's two terms and their sum), of u each relative to what is rounded: 6 u in the L2 norm, relative to the norm of the
    larger of the result and its terms."""
    from wind_rwkv.rwkv7 import linear
    g = th.Generator(device='cuda').manual_seed(B + T)

    def rn(*s, std=1.0):
        return (th.randn(*s, generator=g, device='cuda') * std).bfloat16()

    x, wk, wv, dy = rn(B, T, C), rn(F, C, std=C ** -0.5), rn(C, F, std=F ** -0.5), rn(B, T, C)
    leaves = [t.clone().requires_grad_() for t in (x, wk, wv)]
    y = linear(linear(leaves[0], leaves[1], act='relu2'), leaves[2], residual=leaves[0])
    grads = th.autograd.grad(y, leaves, dy)
    ref = [t.double().requires_grad_() for t in (x, wk, wv)]
    Y = ref[0] + th.relu(ref[0] @ ref[1].T).square() @ ref[2].T
    want = th.autograd.grad(Y, ref, dy.double())
    for a, b in ((y.detach(), Y.detach()), *zip(grads, want)):
        assert float((a.double() - b).norm()) <= 6 * U * float(b.norm())


def test_same_results_every_time_and_in_a_graph():
    from wind_rwkv.rwkv7 import linear
    for M, N, K in ((1, 2048, 2048), (300, 96, 2048), (1400, 3328, 512)):
        x, w, b, r, dy = inputs(M, N, K, th.float32, True, th.bfloat16, 5)
        first = linear(x, w, b, act='gelu', residual=r)
        for _ in range(3):
            assert th.equal(linear(x, w, b, act='gelu', residual=r), first)
        graph = th.cuda.CUDAGraph()
        with th.cuda.graph(graph):
            again = linear(x, w, b, act='gelu', residual=r)
        again.zero_()
        graph.replay()
        assert th.equal(again, first)
        x.copy_(x.flip(0))
        graph.replay()
        assert th.equal(again, linear(x, w, b, act='gelu', residual=r))


def test_streams_and_calls_that_follow_one_another():
    """Two streams at once, and a call that reads what the one ahead of it writes."""
    from wind_rwkv.rwkv7 import linear
    x, w, b, r, _ = inputs(400, 512, 512, th.float32, True, th.bfloat16, 5)
    want = x
    for _ in range(6):
        want = linear(want, w, b, act='tanh', residual=r)
        th.cuda.synchronize()
    side = th.cuda.Stream()
    side.wait_stream(th.cuda.current_stream())
    a = c = x
    for _ in range(6):
        a = linear(a, w, b, act='tanh', residual=r)
        with th.cuda.stream(side):
            c = linear(c, w, b, act='tanh', residual=r)
    th.cuda.synchronize()
    assert th.equal(a, want) and th.equal(c, want)


@pytest.mark.parametrize('M', [4, 100, 3000])
def test_in_a_thread_that_has_made_no_call_yet(M):
    """Such a thread has no current context; the tensor maps' encoding needs one."""
    import threading
    from wind_rwkv.rwkv7 import linear
    x, w, b, r, _ = inputs(M, 3328, 64, th.float32, True, th.bfloat16, 5)
    want, got = linear(x, w, b, residual=r), []
    t = threading.Thread(target=lambda: got.append(linear(x, w, b, residual=r)))
    t.start()
    t.join()
    assert th.equal(got[0], want)


def test_python_form_agrees():
    """The form that torch.compile traces, called directly."""
    from wind_rwkv.rwkv7.rwkv7_linear import ACTS, Linear
    for act, residual, out in (('relu2', False, th.bfloat16), ('relu2', True, th.bfloat16), ('gelu', True, th.float32), (None, True, th.bfloat16)):
        x, w, b, r, dy = inputs(90, 51, 72, th.bfloat16, residual, out, 5)
        compare(x, w, b, r, dy, act, out, call=lambda x, w, b, act, residual, out_dtype: Linear.apply(x, w, b, residual, ACTS[act], out_dtype == th.float32))


def test_compiles():
    from wind_rwkv.rwkv7 import linear
    x, w, b, r, dy = inputs(90, 56, 72, th.float32, True, th.bfloat16, 5)

    def f(x, w, b, r):
        return linear(linear(x, w, b, act='relu2'), w.t(), act=None).float().sum() + linear(x, w, b, act='gelu', residual=r).float().sum()

    grads = []
    for g in (f, th.compile(f, fullgraph=True)):
        leaves = [t.clone().requires_grad_() for t in (x, w, b, r)]
        g(*leaves).backward()
        grads.append([t.grad for t in leaves])
    for a, c in zip(*grads):
        assert th.allclose(a.float(), c.float(), rtol=2 * U, atol=2 * U * float(a.float().abs().max()))


def test_device_status_is_clean():
    from wind_rwkv.rwkv7 import _lib
    assert _lib.device_status() == 0
