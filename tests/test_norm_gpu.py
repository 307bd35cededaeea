"""rms_norm and dropout against their formulas in 64 bits, element by element.

Tolerances, counted in roundings: e = 2^-24 for fp32, u = half a step of the type that is stored (bf16 2^-8, fp32 2^-24), relative.
  h: x / (1 - p) takes two roundings (the factor's and the product's), the sum one, all of |residual| + |x / (1 - p)|; then u.
  y, from the kernel's own h: the sum of squares (all positive) passes at most 32 additions in a thread, 5 in a warp and 16 over warps, plus each square's: 54 e, of which
     the root halves 27; mean, eps, root, reciprocal, two products: 6; 36 e allowed.  Then u.
  dr: g = dy w one rounding; S = sum g h over the row, its error 54 e of sum |g h|; c = S / D rstd^2 takes 3 more and twice rstd's 33 e; rstd (g - c h) 3 more and rstd's.
     Together |rstd g| 40 e + |rstd h| rstd^2 / D (60 e sum |g h| + 80 e |S|); the addition of dh one e of the result and of |dh|; then u.
  dx: dr's before its rounding, two roundings more, times 1 / (1 - p); u.
  dw: a term's three roundings and rstd's 33; n = M / parts + parts / 32 + 64 additions (a thread's rows, a CTA's, the parts): (40 + n) e of the sum of magnitudes.
Which elements are dropped has to be exact.
"""
import pytest
import torch as th

from philox import kept

pytestmark = pytest.mark.gpu

E, U = 2.0 ** -24, {th.bfloat16: 2.0 ** -8, th.float32: 2.0 ** -24}
BF, F32 = th.bfloat16, th.float32


def check(name, got, want, bound):
    assert got.shape == want.shape, name
    e = (got.double() - want).abs() - bound
    assert bool((e <= 0).all()), f'{name}: {int((e > 0).sum())} of {e.numel()} beyond the bound, the worst by {float(e.max()):.2e}'


def rn(*shape, seed, dtype=F32, std=1.):
    g = th.Generator(device='cuda').manual_seed(seed)
    return (th.randn(*shape, generator=g, device='cuda') * std).to(dtype)


def mask_of(shape, p, seed):
    n = 1
    for s in shape:
        n *= s
    return th.from_numpy(kept(0, n, p, seed)).cuda().view(shape)


def check_stream(h, x, r, p, seed):
    X, R = x.detach().double(), r.detach().double()
    X = th.where(mask_of(x.shape, p, seed), X / (1 - p), 0.) if p else X
    assert h.dtype == r.dtype
    check('h', h, R + X, (3 * E * (X.abs() + R.abs())) * (1 + U[h.dtype]) + U[h.dtype] * (R + X).abs())


def check_norm(y, h, w, eps):
    H = h.detach().double()
    W = 1. if w is None else w.detach().double()
    Y = H / (H.square().mean(-1, keepdim=True) + eps).sqrt() * W
    check('y', y, Y, (36 * E + U[y.dtype] * (1 + 36 * E)) * Y.abs())


def parts_of(M, D):
    from wind_rwkv.rwkv7 import _lib
    return _lib.lib().wkv7_rms_norm_bwd_workspace_bytes(M, D) // (4 * D)


def check_grads(h, w, dy, dh, eps, p, mask, dx, dr, dw):
    D = h.shape[-1]
    H, DY = h.detach().double().reshape(-1, D), dy.double().reshape(-1, D)
    W = th.ones(D, dtype=th.float64, device='cuda') if w is None else w.detach().double()
    rstd = (H.square().mean(-1, keepdim=True) + eps).rsqrt()
    G = DY * W
    S, mag = (G * H).sum(-1, keepdim=True), (G * H).abs().sum(-1, keepdim=True)
    d = rstd * (G - H * rstd.square() * S / D)
    bound = E * (40 * (rstd * G).abs() + (rstd * H).abs() * rstd.square() / D * (60 * mag + 80 * S.abs()))
    if dh is not None:
        DH = dh.double().reshape(-1, D)
        d = d + DH
        bound = bound + E * (DH.abs() + d.abs())
    if dr is not None:
        assert dr.dtype == h.dtype
        check('dr', dr.reshape(-1, D), d, bound + U[dr.dtype] * (d.abs() + bound))
    if dx is not None:
        k = mask.reshape(-1, D).double() / (1 - p) if p else 1.
        b = k * (bound + 2 * E * d.abs())
        check('dx', dx.reshape(-1, D), d * k, b + U[dx.dtype] * ((d * k).abs() + b))
    if dw is not None:
        T = DY * H * rstd
        M = H.shape[0]
        n = M / parts_of(M, D) + parts_of(M, D) / 32 + 64
        check('dw', dw, T.sum(0), (40 + n) * E * T.abs().sum(0) + U[dw.dtype] * T.sum(0).abs() * (1 if dw.dtype == BF else 2))


def compare(M, D, x_t, r_t, w_t, p=0., out=None, eps=1e-5, seed=3, std=1., lead=None, only=None):
    """One call with its backward."""
    from wind_rwkv.rwkv7 import rms_norm
    shape = (*(lead or (M,)), D)
    x = rn(*shape, seed=seed, dtype=x_t, std=std).requires_grad_()
    r = None if r_t is None else rn(*shape, seed=seed + 1, dtype=r_t, std=2 * std).requires_grad_()
    w = None if w_t is None else (1 + rn(D, seed=seed + 2, std=0.3)).to(w_t).requires_grad_()
    number = (1 << 40) + 77 * seed
    got = rms_norm(x, w, residual=r, eps=eps, p=p, seed=number if p else None, out_dtype=out)
    y, h = got if r is not None else (got, None)
    assert y.dtype == (out or x_t)
    if r is not None:
        check_stream(h, x, r, p, number)
    base = x if h is None else h
    check_norm(y, base, w, eps)
    dy = rn(*shape, seed=seed + 3, dtype=y.dtype)
    dh = None if h is None or only == 'y' else rn(*shape, seed=seed + 4, dtype=h.dtype)
    leaves = [t for t in (x, w, r) if t is not None]
    outs, grads = ([y], [dy]) if dh is None else ([h], [dh]) if only == 'h' else ([y, h], [dy, dh])
    g = iter(th.autograd.grad(outs, leaves, grads, allow_unused=only == 'h'))
    if only == 'h':
        dy = th.zeros_like(dy)
    dx, dw, dr = next(g), next(g) if w is not None else None, next(g) if r is not None else None
    assert dx.dtype == x_t and dx.shape == x.shape
    check_grads(base, w, dy, dh, eps, p, mask_of(shape, p, number) if p else None, dx, dr, dw)
    return y


SIZES = [(1, 1), (1, 2048), (3, 7), (5, 8), (700, 16), (4100, 24), (257, 100), (33, 256), (1003, 333), (64, 512), (9, 2047), (2000, 2048), (7, 2056), (301, 4096), (5, 5001), (3, 8192), (40, 8200),
         (2, 16383), (11, 16384)]


@pytest.mark.parametrize('M,D', SIZES)
def test_sizes(M, D):
    compare(M, D, BF, BF, BF)
    compare(M, D, BF, BF, F32, p=0.1)
    compare(M, D, F32, F32, F32, p=0.25)
    compare(M, D, F32, None, F32)


@pytest.mark.parametrize('M,D', [(300, 1), (5000, 3), (9000, 8), (3000, 9), (700, 257), (600, 2041), (400, 2047), (350, 4097), (310, 8185), (330, 8199), (500, 16383)])
def test_teams(M, D):
    """Two pieces a thread, several teams a CTA, rows whose first and last pieces have a part, more rows than teams."""
    compare(M, D, BF, BF, F32, p=0.1)
    compare(M, D, BF, F32, BF)
    compare(M, D, F32, F32, F32, p=0.3)
    compare(M, D, BF, None, None)


@pytest.mark.parametrize('D', [64, 333, 2048, 4096])
@pytest.mark.parametrize('x_t', [BF, F32])
@pytest.mark.parametrize('r_t', [None, BF, F32])
@pytest.mark.parametrize('w_t', [None, BF, F32])
def test_types(D, x_t, r_t, w_t):
    for out in (BF, F32):
        compare(37, D, x_t, r_t, w_t, out=out)
        if r_t is not None:
            compare(37, D, x_t, r_t, w_t, p=0.5, out=out)


@pytest.mark.parametrize('M,D', [(20000, 64), (100000, 24), (9000, 2048), (3000, 4100)])
def test_many_rows(M, D):
    """More rows than teams: the persistent loops, and sums over many rows."""
    compare(M, D, BF, F32, F32, p=0.1)
    compare(M, D, F32, BF, None)


def test_one_output_alone_has_a_gradient():
    for only in ('y', 'h'):
        compare(50, 333, BF, BF, F32, p=0.2, only=only)
        compare(50, 512, F32, F32, F32, only=only)


def test_batch_dimensions():
    compare(0, 512, BF, BF, F32, p=0.1, lead=(3, 5))
    compare(0, 100, BF, None, F32, lead=(2, 1, 7))
    from wind_rwkv.rwkv7 import rms_norm
    v = rn(512, seed=1, dtype=BF)
    assert th.equal(rms_norm(v), rms_norm(v[None])[0])


@pytest.mark.parametrize('D', [256, 333, 9000])
@pytest.mark.parametrize('p', [0., 0.2])
def test_some_inputs_alone_have_gradients(D, p):
    """What is not asked for is not formed; what is has the values of the whole."""
    from wind_rwkv.rwkv7 import rms_norm
    x, r, w = rn(40, D, seed=1, dtype=BF), rn(40, D, seed=2, dtype=BF), 1 + rn(D, seed=3, std=0.2)
    dy, dh = rn(40, D, seed=4, dtype=BF), rn(40, D, seed=5, dtype=BF)
    leaves = [t.clone().requires_grad_() for t in (x, w, r)]
    whole = th.autograd.grad(rms_norm(leaves[0], leaves[1], residual=leaves[2], p=p, seed=3), leaves, [dy, dh])
    for keep in ((0,), (1,), (2,), (0, 1), (0, 2), (1, 2)):
        t = [a.clone().requires_grad_() if i in keep else a for i, a in enumerate((x, w, r))]
        got = th.autograd.grad(rms_norm(t[0], t[1], residual=t[2], p=p, seed=3), [t[i] for i in keep], [dy, dh])
        assert all(th.equal(g, whole[i]) for g, i in zip(got, keep))
        y, h = rms_norm(t[0], residual=t[2], p=p, seed=3)     # without a weight
        assert (y.requires_grad and h.requires_grad) == (keep != (1,))


def test_gradient_against_differences():
    """The formula itself: differences of the formula in 64 bits along random directions."""
    M, D, eps, p, seed = 6, 40, 1e-3, 0.3, 11
    x, r, w = rn(M, D, seed=1).requires_grad_(), rn(M, D, seed=2).requires_grad_(), (1 + rn(D, seed=3)).requires_grad_()
    dy, dh = rn(M, D, seed=4), rn(M, D, seed=5)
    from wind_rwkv.rwkv7 import rms_norm
    grads = th.autograd.grad(rms_norm(x, w, residual=r, eps=eps, p=p, seed=seed), [x, w, r], [dy, dh])
    mask = mask_of((M, D), p, seed)

    def loss(x, w, r):
        h = r + th.where(mask, x / (1 - p), 0.)
        return float(((h / (h.square().mean(-1, keepdim=True) + eps).sqrt() * w) * dy.double()).sum() + (h * dh.double()).sum())

    at = [t.detach().double() for t in (x, w, r)]
    for i in range(3):
        for s in range(4):
            d = rn(*at[i].shape, seed=20 + s).double()
            hi, lo = ([t + sign * 1e-5 * d if j == i else t for j, t in enumerate(at)] for sign in (1, -1))
            diff = (loss(*hi) - loss(*lo)) / 2e-5
            # differences: 1e-10 times a third derivative of some 1e3, and 1e-16 of the loss over 2e-5; gradients: fp32 of M D terms
            assert abs(diff - float((grads[i].double() * d).sum())) < 1e-5 * float((grads[i].double() * d).abs().sum()) + 1e-6


def test_zero_rows_and_far_magnitudes():
    from wind_rwkv.rwkv7 import rms_norm
    x = rn(6, 256, seed=1)
    x[0] = 0
    x[1] *= 1e-15
    x[2] *= 1e15
    x[3, 1:] = 0
    x[4] *= 1e-30
    check_norm(rms_norm(x), x, None, 1e-5)
    check_norm(rms_norm(x[:4], eps=1e-12), x[:4], None, 1e-12)
    y = rms_norm(x[:1], eps=0.)
    assert bool(y.isnan().all())                                        # 0 / 0, as the formula has it
    bad = rn(4, 300, seed=2, dtype=BF)
    bad[1, 7], bad[2, 9] = float('nan'), float('inf')
    y = rms_norm(bad)
    assert bool(y[0].isfinite().all()) and bool(y[3].isfinite().all()) and bool(y[1].isnan().all())
    assert bool(y[2, 9].isnan()) and not y[2, :9].any()                 # inf / inf, finite / inf


@pytest.mark.parametrize('D', [2048, 333])
def test_layouts(D):
    """Rows that lie in wider tensors, at any alignment; orders that are copied."""
    from wind_rwkv.rwkv7 import rms_norm
    w = 1 + rn(D, seed=9, std=0.2)
    wide = [rn(12, 2 * D + 24, seed=s, dtype=BF) for s in (1, 2)]
    views = [lambda t: t[:, 8:8 + D], lambda t: t[:, 1:1 + D], lambda t: t[::2, 16:16 + D], lambda t: t[:, :2 * D:2], lambda t: t[:1, 3:3 + D].expand(12, D), lambda t: t[:0, :D]]
    for view in views:
        for other in views:
            x, r = view(wide[0]), other(wide[1])
            if x.shape != r.shape:
                continue
            want = rms_norm(x.clone(memory_format=th.contiguous_format), w, residual=r.clone(memory_format=th.contiguous_format))
            got = rms_norm(x, w, residual=r)
            assert all(th.equal(a, b) for a, b in zip(got, want))
    flat = rn(12 * D + 8, seed=6, dtype=BF)
    for off in (1, 3, 4, 8):  # rows back to back, at any alignment
        x = flat[off:off + 12 * D].view(12, D)
        assert th.equal(rms_norm(x, w), rms_norm(x.clone(), w))
    # gradients that come in other layouts
    x, r = (t[:, :D].clone().requires_grad_() for t in wide)
    y, h = rms_norm(x, w, residual=r, p=0.1, seed=5)
    dy, dh = rn(D, 12, seed=3, dtype=BF).t(), rn(1, 1, seed=4, dtype=BF).expand(12, D)
    got = th.autograd.grad([y, h], [x, r], [dy, dh], retain_graph=True)
    want = th.autograd.grad([y, h], [x, r], [dy.contiguous(), dh.contiguous()])
    assert all(th.equal(a, b) for a, b in zip(got, want))


def test_same_results_from_call_to_call_and_on_other_streams():
    from wind_rwkv.rwkv7 import rms_norm
    x, r, w = rn(4000, 1000, seed=1, dtype=BF).requires_grad_(), rn(4000, 1000, seed=2, dtype=BF).requires_grad_(), rn(1000, seed=3).requires_grad_()
    dy = rn(4000, 1000, seed=4, dtype=BF)

    def step():
        y, h = rms_norm(x, w, residual=r, p=0.1, seed=9)
        return [y.detach(), h.detach(), *th.autograd.grad([y, h], [x, w, r], [dy, dy])]

    want = step()
    sides = [th.cuda.Stream() for _ in range(2)]
    outs = []
    for s in sides:
        s.wait_stream(th.cuda.current_stream())
    for _ in range(3):
        for s in sides:
            with th.cuda.stream(s):
                outs.append(step())
    th.cuda.synchronize()
    for got in outs:
        assert all(th.equal(a, b) for a, b in zip(got, want))


def test_results_go_where_they_belong():
    """Nothing is written beside y, h, dx, dr, dw, q: C entry points with outputs inside larger buffers."""
    from wind_rwkv.rwkv7 import _lib
    L = _lib.lib()
    for M, D in ((3, 77), (5, 64), (300, 333), (700, 2050), (9, 9000)):
        x, r, dy = (rn(M, D, seed=s, dtype=BF) for s in (1, 2, 3))
        for ld in (D + 3, (D + 23) // 8 * 8):
            y, h, dx, dr = (th.full((M + 2, ld), 7., dtype=BF, device='cuda') for _ in range(4))
            rstd, scale = (th.full((M + 2,), 7., device='cuda') for _ in range(2))
            dw = th.full((D + 8,), 7., device='cuda')
            q = th.full((M + 2, ld), 7, dtype=th.int8, device='cuda')
            s = _lib.stream_of(x)
            at = lambda t: t.data_ptr() + t.stride(0) * t.element_size()  # noqa: E731
            assert L.wkv7_rms_norm_fwd(x.data_ptr(), r.data_ptr(), None, at(y), at(h), at(rstd), None, M, D, D, D, ld, ld, 1e-5, 0.1, 3, None, 0, s) == 0
            assert L.wkv7_rms_norm_fwd(x.data_ptr(), r.data_ptr(), None, at(q), at(h), None, at(scale), M, D, D, D, ld, ld, 1e-5, 0.1, 3, None, 16, s) == 0
            ws = th.empty(L.wkv7_rms_norm_bwd_workspace_bytes(M, D), dtype=th.uint8, device='cuda')
            assert L.wkv7_rms_norm_bwd(at(h), at(rstd), None, dy.data_ptr(), None, at(dx), at(dr), dw[4:].data_ptr(), M, D, ld, D, D, ld, ld, 0.1, 3, None, 0, ws.data_ptr(), s) == 0
            for t in (y, h, dx, dr, q):
                assert bool((t[0] == 7).all()) and bool((t[-1] == 7).all()) and bool((t[:, D:] == 7).all())
            assert float(rstd[0]) == float(rstd[-1]) == float(scale[0]) == float(scale[-1]) == 7 and bool((dw[:4] == 7).all()) and bool((dw[-4:] == 7).all())
            check_stream(h[1:-1, :D], x, r, 0.1, 3)
            check_norm(y[1:-1, :D], h[1:-1, :D], None, 1e-5)
            check_grads(h[1:-1, :D], None, dy, None, 1e-5, 0.1, mask_of((M, D), 0.1, 3), dx[1:-1, :D], dr[1:-1, :D], dw[4:-4])
    # the stream in place
    x, r = rn(500, 333, seed=1, dtype=BF), rn(500, 333, seed=2, dtype=BF)
    keep, y = r.clone(), th.empty_like(x)
    assert L.wkv7_rms_norm_fwd(x.data_ptr(), r.data_ptr(), None, y.data_ptr(), r.data_ptr(), None, None, 500, 333, 333, 333, 333, 333, 1e-5, 0., 0, None, 0, _lib.stream_of(x)) == 0
    check_stream(r, x, keep, 0., 0)
    check_norm(y, r, None, 1e-5)


def test_empty():
    from wind_rwkv.rwkv7 import dropout, rms_norm
    x, r, w = (th.zeros(0, 64, dtype=BF, device='cuda').requires_grad_() for _ in range(2)), None, rn(64, seed=1).requires_grad_()
    x, r = x
    y, h = rms_norm(x, w, residual=r, p=0.1, seed=1)
    assert y.shape == h.shape == (0, 64)
    dx, dw, dr = th.autograd.grad([y, h], [x, w, r], [th.zeros_like(y), th.zeros_like(h)])
    assert dx.shape == dr.shape == (0, 64) and dw.shape == (64,) and not dw.any()
    assert dropout(x, 0.5, 1).shape == (0, 64)


# ---- dropout -----------------------------------------------------------------------------------------------
@pytest.mark.parametrize('shape', [(1,), (3,), (4,), (7, 13), (512, 768), (2, 3, 1000), (100003,)])
@pytest.mark.parametrize('x_t', [BF, F32])
@pytest.mark.parametrize('r_t', [None, BF, F32])
@pytest.mark.parametrize('p', [0., 0.1, 0.5, 1.])
def test_dropout(shape, x_t, r_t, p):
    from wind_rwkv.rwkv7 import dropout
    seed = (1 << 45) + 12345
    x = rn(*shape, seed=1, dtype=x_t).requires_grad_()
    r = None if r_t is None else rn(*shape, seed=2, dtype=r_t).requires_grad_()
    y = dropout(x, p, seed, residual=r)
    assert y.dtype == (r_t or x_t) and y.shape == x.shape
    mask = mask_of(shape, p, seed)
    X = th.where(mask, x.detach().double() / (1 - p) if p < 1 else 0., 0.)
    R = 0. if r is None else r.detach().double()
    u = U[y.dtype]
    e = 3 * E * (X.abs() + (0. if r is None else R.abs()))
    check('y', y, X + R, e + u * ((X + R).abs() + e))
    dy = rn(*shape, seed=3, dtype=y.dtype)
    g = th.autograd.grad(y, [t for t in (x, r) if t is not None], dy)
    D = th.where(mask, dy.double() / (1 - p) if p < 1 else 0., 0.)
    assert g[0].dtype == x_t
    check('dx', g[0], D, (2 * E + U[x_t]) * (1 + 2 * E) * D.abs())
    assert r is None or th.equal(g[1], dy)


def test_dropped_infinities_and_nan():
    from wind_rwkv.rwkv7 import dropout, rms_norm
    x = th.full((1000,), float('inf'), device='cuda')
    x[::2] = float('nan')
    mask = mask_of((1000,), 0.5, 3)
    y = dropout(x, 0.5, 3)
    assert not y[~mask].any() and bool((y[mask].isnan() == x[mask].isnan()).all()) and bool((y[mask].isinf() == x[mask].isinf()).all())
    one = rms_norm(x[None], residual=th.ones(1, 1000, device='cuda'), p=1., seed=3)
    assert bool((one[1] == 1).all())


def test_rates_and_seeds():
    from wind_rwkv.rwkv7 import dropout
    x = th.ones(1 << 22, device='cuda')
    seen = []
    for p in (0.1, 0.5, 0.9):
        y = dropout(x, p, 5)
        n = float((y == 0).sum())
        assert abs(n / x.numel() - p) < 6 * (p * (1 - p) / x.numel()) ** 0.5
        seen.append(y == 0)
    assert bool((seen[0] <= seen[1]).all()) and bool((seen[1] <= seen[2]).all())      # one word an element
    a, b = dropout(x, 0.5, 5) == 0, dropout(x, 0.5, 6) == 0
    assert abs(float((a & b).sum()) / x.numel() - 0.25) < 6 * (0.1875 / x.numel()) ** 0.5
    assert th.equal(dropout(x, 0.5, th.tensor([5], device='cuda')) == 0, a) and th.equal(dropout(x, 0.5, th.tensor(5, device='cuda')) == 0, a)


def test_layouts_of_dropout():
    from wind_rwkv.rwkv7 import dropout
    wide = rn(64, 200, seed=1)
    for view in (wide[:, 1:100], wide.t(), wide[:, ::2], wide[:1].expand(64, 200), wide.view(-1)[1:1001]):
        x = view.detach().requires_grad_()
        y = dropout(x, 0.3, 7, residual=view)
        flat = dropout(view.clone(memory_format=th.contiguous_format), 0.3, 7, residual=view.clone(memory_format=th.contiguous_format))
        assert th.equal(y, flat)
        g, = th.autograd.grad(y, x, th.ones_like(y))
        assert bool(((g != 0) == mask_of(view.shape, 0.3, 7)).all())


def test_beyond_32_bits():
    """Elements behind the 2^32nd: their places, and the words' counters."""
    from wind_rwkv.rwkv7 import dropout
    n = (1 << 32) + 4099
    x = th.ones(n, dtype=BF, device='cuda')
    y = dropout(x, 0.5, 21)
    for first in (0, (1 << 31) - 8, (1 << 32) - 8, n - 4000):
        part = y[first:first + 4000] != 0
        assert th.equal(part.cpu(), th.from_numpy(kept(first, part.numel(), 0.5, 21)))


def test_counters_beyond_32_bits():
    """Elements behind the 2^34th, whose counters leave 32 bits."""
    from wind_rwkv.rwkv7 import dropout
    n = (1 << 34) + 4099
    if th.cuda.mem_get_info()[0] < 5 * n:
        pytest.skip('two tensors of 32 GB do not fit')
    y = dropout(th.ones(n, dtype=BF, device='cuda'), 0.5, 21)
    for first in (0, (1 << 32) - 8, (1 << 34) - 2000, n - 4000):
        part = y[first:first + 4000] != 0
        assert th.equal(part.cpu(), th.from_numpy(kept(first, part.numel(), 0.5, 21)))
    del y
    th.cuda.empty_cache()


def test_rows_beyond_32_bits():
    from wind_rwkv.rwkv7 import rms_norm
    M, D = 70000, 32768 + 8
    x = th.empty(M, D, dtype=BF, device='cuda')[:, :16384]  # rows of a wider tensor: 2.3e9 elements apart at the end
    x[-3:] = rn(3, 16384, seed=1, dtype=BF)
    x[:-3] = 1.
    check_norm(rms_norm(x)[-3:], x[-3:], None, 1e-5)


def test_a_captured_step_draws_anew():
    """Forward and backward captured together; the seed lies on the device and is changed between replays."""
    from wind_rwkv.rwkv7 import dropout, rms_norm
    x, r, w, dy = rn(300, 512, seed=1, dtype=BF), rn(300, 512, seed=2, dtype=BF), rn(512, seed=3), rn(300, 512, seed=4, dtype=BF)
    seed = th.tensor([100], dtype=th.int64, device='cuda')

    def step(seed):
        leaves = [t.detach().requires_grad_() for t in (x, w, r)]
        y, h = rms_norm(leaves[0], leaves[1], residual=leaves[2], p=0.2, seed=seed)
        z = dropout(y, 0.3, seed, residual=h)
        return [z.detach(), *th.autograd.grad(z, leaves, dy)]

    side = th.cuda.Stream()
    side.wait_stream(th.cuda.current_stream())
    with th.cuda.stream(side):
        step(seed)
    th.cuda.current_stream().wait_stream(side)
    graph = th.cuda.CUDAGraph()
    with th.cuda.graph(graph):
        out = step(seed)
    for number in (100, 101, (1 << 62) + 3):
        seed.fill_(number)
        x.copy_(x.flip(0))
        graph.replay()
        assert all(th.equal(a, c) for a, c in zip(out, step(number)))


def test_a_seed_changed_before_its_backward_is_noticed():
    from wind_rwkv.rwkv7 import dropout
    x = rn(100, seed=1).requires_grad_()
    seed = th.tensor([1], dtype=th.int64, device='cuda')
    y = dropout(x, 0.5, seed)
    seed += 1
    with pytest.raises(RuntimeError, match='modified by an inplace'):
        y.sum().backward()


def test_torch_compile():
    from wind_rwkv.rwkv7 import dropout, rms_norm
    x, r, w = rn(40, 333, seed=1, dtype=BF).requires_grad_(), rn(40, 333, seed=2, dtype=F32).requires_grad_(), rn(333, seed=3).requires_grad_()

    def f(x, r, w):
        y, h = rms_norm(x, w, residual=r, p=0.1, seed=4)
        return dropout(y, 0.2, 9) * 2, h

    want = f(x, r, w)
    wg = th.autograd.grad([t.float().sum() for t in want], [x, r, w])
    th.compiler.reset()
    got = th.compile(f, backend='aot_eager', fullgraph=True)(x, r, w)
    gg = th.autograd.grad([t.float().sum() for t in got], [x, r, w])
    assert all(th.equal(a, b) for a, b in zip([*want, *wg], [*got, *gg]))


@pytest.mark.parametrize('dynamic', [False, True])
def test_torch_compile_without_a_residual(dynamic):
    from wind_rwkv.rwkv7 import rms_norm
    w = (1 + rn(333, seed=3, std=0.2)).requires_grad_()
    th.compiler.reset()
    f = th.compile(lambda x, w: rms_norm(x, w, out_dtype=F32) * 2, backend='aot_eager', fullgraph=True, dynamic=dynamic)
    for M in (40, 41, 7):
        x = rn(M, 333, seed=M, dtype=BF).requires_grad_()
        want, got = rms_norm(x, w, out_dtype=F32) * 2, f(x, w)
        assert th.equal(want, got)
        assert all(th.equal(a, b) for a, b in zip(th.autograd.grad(want.sum(), [x, w]), th.autograd.grad(got.sum(), [x, w])))


def test_python_form_gives_the_same():
    """The form that torch.compile traces, called directly, against the eager host path."""
    from wind_rwkv.rwkv7 import dropout, rms_norm
    from wind_rwkv.rwkv7.rwkv7_norm import Dropout, RmsNorm
    for x_t, r_t, p, out in ((BF, BF, 0., BF), (BF, F32, 0.1, F32), (F32, BF, 0.2, BF)):
        x, r, w = rn(70, 200, seed=1, dtype=x_t).requires_grad_(), rn(70, 200, seed=2, dtype=r_t).requires_grad_(), rn(200, seed=3).requires_grad_()
        a = rms_norm(x, w, residual=r, p=p, seed=6, out_dtype=out)
        b = RmsNorm.apply(x, w, r, None, 1e-5, p, 6, out == F32)
        dy, dh = rn(70, 200, seed=4, dtype=out), rn(70, 200, seed=5, dtype=r_t)
        assert all(th.equal(s, t) for s, t in zip([*a, *th.autograd.grad(a, [x, w, r], [dy, dh])], [*b, *th.autograd.grad(b, [x, w, r], [dy, dh])]))
        a, b = dropout(x, 0.3, 8, residual=r), Dropout.apply(x, r, None, 0.3, 8)
        assert all(th.equal(s, t) for s, t in zip([a, *th.autograd.grad(a, [x, r], dh)], [b, *th.autograd.grad(b, [x, r], dh)]))


def test_a_block_in_training():
    """As a program runs them: the stream through two norms with dropout around the channel mixer, forward and backward, against the same in 64 bits on the same masks."""
    from wind_rwkv.rwkv7 import dropout, linear, rms_norm
    M, D, F, p = 300, 256, 1024, 0.1
    x, emb = rn(M, D, seed=1, dtype=BF).requires_grad_(), rn(M, D, seed=2, dtype=BF).requires_grad_()
    w1, w2 = (1 + rn(D, seed=3, std=0.2)).requires_grad_(), (1 + rn(D, seed=4, std=0.2)).requires_grad_()
    wk, wv = rn(F, D, seed=5, dtype=BF, std=D ** -0.5).requires_grad_(), rn(D, F, seed=6, dtype=BF, std=F ** -0.5).requires_grad_()
    leaves = [x, emb, w1, w2, wk, wv]
    dy = rn(M, D, seed=7, dtype=BF)

    def block(x, emb, w1, w2, wk, wv, norm, drop, mix):
        y, h = norm(x, w1, drop(emb, 1), 2)
        y, h = norm(mix(y, wk, wv), w2, h, 3)
        return y + h

    out = block(*leaves, lambda x, w, r, s: rms_norm(x, w, residual=r, p=p, seed=s), lambda e, s: dropout(e, p, s), lambda y, a, b: linear(linear(y, a, act='relu2'), b))
    got = th.autograd.grad(out, leaves, dy)
    ref = [t.detach().double().requires_grad_() for t in leaves]

    def mask(t, s):
        return th.where(mask_of((M, D), p, s), t / (1 - p), 0.)

    def norm(x, w, r, s):
        h = r + mask(x, s)
        return h / (h.square().mean(-1, keepdim=True) + 1e-5).sqrt() * w, h

    want_out = block(*ref, norm, mask, lambda y, a, b: th.relu(y @ a.T).square() @ b.T)
    want = th.autograd.grad(want_out, ref, dy.double())
    # a dozen tensors rounded to bf16 on the way there and back: rms 2^-9 / sqrt(3) of each, relu2 doubles what comes before it
    for g, w in zip([out.detach(), *got], [want_out.detach(), *want]):
        assert float((g.double() - w).norm() / w.norm()) < 24 * 2.0 ** -9 / 3 ** 0.5


@pytest.mark.parametrize('x_t,r_t', [(F32, None), (F32, F32), (F32, BF), (BF, F32)])
@pytest.mark.parametrize('form', ['eager', 'python'])
def test_second_derivatives_of_dropout(x_t, r_t, form):
    """A penalty on the gradient: y = r + k x with k = kept / (1 - p), dx = k dy, and so through dx to dy."""
    from wind_rwkv.rwkv7 import dropout
    from wind_rwkv.rwkv7.rwkv7_norm import Dropout
    shape, p, seed = (50, 77), 0.3, 19
    x = rn(*shape, seed=1, dtype=x_t).requires_grad_()
    r = None if r_t is None else rn(*shape, seed=2, dtype=r_t).requires_grad_()
    leaves = [t for t in (x, r) if t is not None]
    y = dropout(x, p, seed, residual=r) if form == 'eager' else Dropout.apply(x, r, None, p, seed)
    first = th.autograd.grad(y.square().sum(), leaves, create_graph=True)
    assert all(g.requires_grad for g in first) and first[0].dtype == x_t
    u = rn(*shape, seed=3, dtype=x_t)
    second = th.autograd.grad(first[0], leaves, u)
    K = mask_of(shape, p, seed).double() / (1 - p)
    X, R = x.detach().double(), 0. if r is None else r.detach().double()
    Y = R + K * X
    # y: three roundings of its parts and its own; 2 y is exact; dx: two and its type's.  Of the second derivative 2 k k u each product: two and its type's
    parts = (K * X).abs() + (0. if r is None else R.abs())
    e = 2 * K * (3 * E * parts + U[y.dtype] * (Y.abs() + 3 * E * parts))
    check('dx', first[0], 2 * K * Y, e + (2 * E + U[x_t]) * ((2 * K * Y).abs() + e))
    for g, want in zip(second, [2 * K * K * u.double()] + ([] if r is None else [2 * K * u.double()])):
        check('second', g, want, (4 * E + U[y.dtype] + U[g.dtype]) * 1.01 * want.abs())
    if form == 'eager' and x_t == r_t:  # linear in dy, whatever x is
        v = rn(*shape, seed=4).requires_grad_()
        dx, = th.autograd.grad(dropout(x, p, seed, residual=r), x, v, create_graph=True)
        back, = th.autograd.grad(dx, v, u)
        check('dv', back, K * u.double(), 4 * E * (K * u.double()).abs())


@pytest.mark.parametrize('D', [128, 333])
@pytest.mark.parametrize('form', ['eager', 'python'])
def test_second_derivatives_of_the_norm_are_refused(D, form):
    """A backward that is recorded gives the same gradients; what is differentiated through them raises, whichever input or gradient it comes from, and no term is left out."""
    from wind_rwkv.rwkv7 import rms_norm
    from wind_rwkv.rwkv7.rwkv7_norm import RmsNorm
    for p, r_t in ((0., BF), (0.2, F32), (0., None)):
        x, w = rn(9, D, seed=1, dtype=BF).requires_grad_(), (1 + rn(D, seed=3, std=0.2)).requires_grad_()
        r = None if r_t is None else rn(9, D, seed=2, dtype=r_t).requires_grad_()
        dy, dh = rn(9, D, seed=4, dtype=BF).requires_grad_(), rn(9, D, seed=5, dtype=r_t or BF).requires_grad_()
        leaves = [t for t in (x, w, r) if t is not None]

        def call(x, w, r):
            y, h = (rms_norm(x, w, residual=r, p=p, seed=6), None) if r is None else rms_norm(x, w, residual=r, p=p, seed=6)
            if form == 'python':
                y, h = RmsNorm.apply(x, w, r, None, 1e-5, p, 6, False)
            return [y] if h is None else [y, h]

        outs = call(x, w, r)
        want = th.autograd.grad(outs, leaves, [dy, dh][:len(outs)], retain_graph=True)
        assert not any(g.requires_grad for g in want)
        got = th.autograd.grad(outs, leaves, [dy, dh][:len(outs)], create_graph=True)
        assert all(th.equal(a, b) for a, b in zip(got, want))
        for i, g in enumerate(got):
            for of in leaves + [dy]:
                if i == 1 and of is w:   # dw does not depend on w
                    continue
                with pytest.raises(RuntimeError, match='second derivative'):
                    th.autograd.grad(g.float().sum() + outs[0].float().sum() + dy.float().sum(), of, retain_graph=True)
        # a constant of what is asked for: there is nothing to refuse
        outs = call(x.detach(), w, None if r is None else r.detach())
        g, = th.autograd.grad(outs[0], w, dy.detach(), create_graph=True)
        assert th.equal(g, th.autograd.grad(call(x.detach(), w, None if r is None else r.detach())[0], w, dy.detach())[0]) and not g.requires_grad
        # a step that records its backward and differentiates nothing through it
        t = [a.detach().requires_grad_() for a in leaves]
        sum(o.float().sum() for o in call(t[0], t[1], t[2] if len(t) > 2 else None)).backward(create_graph=True)
        assert all(a.grad is not None for a in t)


def test_seeds_are_integers_whether_or_not_they_are_used():
    import numpy as np
    from wind_rwkv.rwkv7 import dropout, rms_norm
    x = rn(4, 64, seed=1, dtype=BF)
    for seed in (-1, -2, 1 << 63, 1.5, th.zeros(2, dtype=th.int64, device='cuda'), th.zeros(1, device='cuda')):
        for p in (0., 0.5):
            with pytest.raises(ValueError, match='rms_norm: a seed'):
                rms_norm(x, residual=x, p=p, seed=seed)
            with pytest.raises(ValueError, match='dropout: a seed'):
                dropout(x, p, seed)
    want = rms_norm(x, residual=x)
    for seed in (0, 7, (1 << 63) - 1, np.int64(7), th.tensor([7], device='cuda')):
        assert all(th.equal(a, b) for a, b in zip(rms_norm(x, residual=x, seed=seed), want))
        rms_norm(x, residual=x, p=0.5, seed=seed)
