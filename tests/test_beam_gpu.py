"""beam_select against its definition in 64 bits, and reorder_states against indexing.

The kernel's normaliser is off by at most tol = 2^-22 (exponential) + 2^-23 E[m - l] (its argument: a difference and a product, rounded) + 70 2^-24 (sums of up
to 64 terms a lane, and across lanes), E over the row's softmax.  Candidates of different beams that are closer than 2 tol may change places; equal ones
may not: the lowest index goes first."""
import pytest
import torch as th

pytestmark = pytest.mark.gpu
INF = float('inf')


def reference(logits, scores, k, finished=None, eos=None):
    """(scores, indices, all candidates' scores, tolerance) in 64 bits."""
    B, W, V = logits.shape
    x = logits.double()
    x = th.where(x < INF, x, -INF)
    s = th.where(scores < INF, scores, -INF).double()
    m = x.amax(-1, keepdim=True)
    m0 = th.where(m > -INF, m, 0.)
    p = th.exp(x - m0)
    # (summed down columns: torch's sum along a row goes in an order that depends on the row's alignment, so that equal rows would get unequal sums)
    z = p.transpose(1, 2).contiguous().sum(1)[..., None]
    lp = th.where(x > -INF, (x - m0) - z.log(), -INF)
    spread = th.where(p > 0, p * (m0 - x), 0.).sum(-1) / z[..., 0].clamp(min=1)
    tol = float(2 ** -22 + 2 ** -23 * spread.max() + 70 * 2 ** -24)
    if finished is not None:
        only = th.full((V,), -INF, dtype=th.float64, device=x.device)
        only[eos] = 0.
        lp = th.where(finished[..., None], only, lp)
    every = (s[..., None] + lp).view(B, W * V)
    best, i = every.sort(dim=1, descending=True, stable=True)
    return best, i, every, tol


def compare(logits, scores, k=None, finished=None, eos=None, call=None):
    from wind_rwkv.rwkv7 import beam_select
    B, W, V = logits.shape
    out = (call or beam_select)(logits, scores, k, finished=finished, eos=eos)
    k = W if k is None else k
    got, parents, tokens = out[:3]
    assert got.dtype == th.float32 and parents.dtype == tokens.dtype == th.int64 and all(t.shape == (B, k) for t in out)
    best, index, every, tol = reference(logits, scores, k, finished, eos)
    want = best[:, :k]
    fin = want > -INF
    assert th.equal(got > -INF, fin)
    assert bool(((got.double() - want).abs()[fin] <= tol + 2.0 ** -24 * (want.abs()[fin] + tol)).all())
    mine = parents * V + tokens
    at = every.gather(1, mine)
    assert th.equal(at > -INF, fin) and bool(((at - want).abs()[fin] <= 2 * tol).all())
    assert all(len(set(r.tolist())) == k for r in mine)
    # where neighbours are equal or further apart than the tolerance, the candidate is the definition's
    near = th.diff(best[:, :min(k + 1, best.shape[1])], dim=1).abs()
    near = th.nan_to_num(near, nan=0.0)
    soft = (near > 0) & (near <= 2 * tol)
    loose = th.zeros(B, k + 1, dtype=th.bool, device=best.device)
    loose[:, :soft.shape[1]] |= soft
    loose[:, 1:1 + soft.shape[1]] |= soft[:, :k]
    same = (mine == index[:, :k]) | loose[:, :k]
    assert bool(same.all()), (mine[~same].tolist(), index[:, :k][~same].tolist())
    if finished is not None:
        assert th.equal(out[3], finished.gather(1, parents) | (tokens == eos))
    return out


def make(B, W, V, dtype=th.bfloat16, seed=0, std=3.0):
    g = th.Generator(device='cuda').manual_seed(seed + B * W * V)
    return (th.randn(B, W, V, generator=g, device='cuda') * std).to(dtype), -10 + 3 * th.rand(B, W, generator=g, device='cuda')


@pytest.mark.parametrize('dtype', [th.bfloat16, th.float32])
@pytest.mark.parametrize('B,W,V,k', [(1, 1, 1, 1), (1, 1, 7, 7), (2, 3, 1, 3), (1, 4, 256, 4), (3, 5, 257, 10), (2, 1, 1000, 32), (4, 6, 5003, 6), (1, 4, 65536, 4),
                                     (2, 8, 50001, 16), (1, 64, 3001, 64), (3, 16, 8192, 64), (2, 32, 131072, 32), (70, 4, 300, 8), (8, 23, 3577, 46)])
def test_sizes(B, W, V, k, dtype):
    logits, scores = make(B, W, V, dtype)
    compare(logits, scores, k)
    finished = th.arange(B * W, device='cuda').view(B, W) % 3 == 1
    compare(logits, scores, k, finished, min(2, V - 1))


@pytest.mark.parametrize('dtype', [th.bfloat16, th.float32])
@pytest.mark.parametrize('V', [4096, 3001])
def test_masks(V, dtype):
    """Rows that a mask leaves empty or nearly so, masks of the type's lowest value, NaN and infinities, beams that are not there."""
    low = th.finfo(dtype).min
    for fill in (-INF, low, float('nan'), INF):
        for left in (0, 1, 3, 40):
            logits, scores = make(2, 4, V, dtype, seed=left)
            keep = logits[..., 5:5 + left].clone()
            logits.fill_(fill)
            logits[..., 5:5 + left] = keep
            for k in (1, 4, 16, 64):
                compare(logits, scores, k)
    logits, scores = make(2, 4, V, dtype)
    logits[:, 1] = -INF
    logits[1] = -INF
    compare(logits, scores, 4)
    scores[:, 1:] = -INF
    compare(logits, scores, 9)
    scores[:] = -INF
    compare(logits, scores, 9)
    logits, scores = make(2, 4, V, dtype)
    scores[0, 0], scores[0, 1], scores[1, 2] = float('nan'), INF, -INF
    compare(logits, scores, 4)
    logits[:, :, ::3], logits[:, :, 1::3] = float('nan'), INF
    compare(logits, scores, 64)


@pytest.mark.parametrize('V', [4096, 3001, 50001])
def test_equal_scores(V):
    """Equal candidates: the lowest index goes first, also among beams whose rows lie on different boundaries."""
    logits, scores = make(2, 6, V)
    compare(logits.zero_(), scores, 12)
    compare(logits, scores.fill_(-3.), 64)
    logits, _ = make(2, 1, V)
    compare(logits.expand(2, 6, V).contiguous(), scores, 12)
    compare(logits.round().expand(2, 6, V).contiguous(), scores, 64)
    logits, scores = make(2, 6, V)
    compare((logits / 4).round(), scores, 64)
    compare(logits.expand(2, 6, V)[:, :1].expand(2, 6, V), scores.fill_(0.), 7)          # one row for all beams


@pytest.mark.parametrize('W,V', [(8, 65536), (5, 20001)])
def test_few_allowed(W, V):
    """A mask of the type's lowest value, or of -inf, that leaves the same few tokens to all beams: more and fewer than are asked for."""
    for dtype in (th.bfloat16, th.float32):
        for fill in (th.finfo(dtype).min, -INF):
            for left in (slice(0, 3), slice(V // 2, V // 2 + 40), slice(V - 1, V)):
                logits, scores = make(2, W, V, dtype)
                keep = logits[..., left].clone()
                logits.fill_(fill)
                logits[..., left] = keep
                for k in (W, 64):
                    compare(logits, scores, k)


FILLS = (-1e4, -65504., -1e6, -1e8, -1e9, -2e9, -1e10, -1e12, 1e6, 1e9)


@pytest.mark.parametrize('dtype', [th.bfloat16, th.float32])
@pytest.mark.parametrize('W,V', [(4, 4096), (5, 3001), (2, 263000)])
def test_masks_of_any_size(W, V, dtype):
    """Masks of the constants that programs write: whole beams, beams that are not there, rows with a few tokens left, everything; a beam that has ended among them."""
    for fill in FILLS:
        for whole in ([1], [0, 1], list(range(W))):
            logits, scores = make(2, W, V, dtype)
            logits[:, whole] = fill
            finished = th.arange(2 * W, device='cuda').view(2, W) % 4 == 2
            for k in (1, W, 64):
                compare(logits, scores, k)
            compare(logits, scores, W, finished, V - 1)
            scores[:, whole] = -INF
            compare(logits, scores, W)
            compare(logits, scores, 2 * W, finished, 0)
        for left in (1, 3, 40):
            logits, scores = make(2, W, V, dtype, seed=left)
            keep = logits[..., 5:5 + left].clone()
            logits.fill_(fill)
            logits[..., 5:5 + left] = keep
            for k in (1, W, 64):
                compare(logits, scores, k)


@pytest.mark.parametrize('dtype', [th.bfloat16, th.float32])
@pytest.mark.parametrize('V', [4096, 3001])
def test_masks_of_any_size_beside_nan(V, dtype):
    """Parts of rows that are worked twice, since a NaN or +inf is among them."""
    for fill in FILLS:
        for odd in (float('nan'), INF):
            logits, scores = make(2, 4, V, dtype)
            logits[:, 1] = fill
            logits[:, 2, ::2] = fill
            logits[:, :, 1::7] = odd
            for k in (4, 64):
                compare(logits, scores, k)


@pytest.mark.parametrize('dtype', [th.bfloat16, th.float32])
def test_large_logits(dtype):
    """Rows that lie far from zero, on either side."""
    for by in (1e2, 1e3, 1e4, 1e5, 1e6, 1e7, 1e8, 1e30):
        for sign in (1, -1):
            logits, scores = make(2, 6, 5003, th.float32)
            for k in (6, 64):
                compare((logits + sign * by).to(dtype), scores, k)
                compare((logits * (sign * by)).to(dtype), scores, k)


@pytest.mark.parametrize('dtype', [th.bfloat16, th.float32])
def test_normalisers_of_long_parts(dtype):
    """The best scores themselves, brought next to zero by the beams' own so that no rounding of theirs hides the normaliser's error.  B W V is large enough for parts of sixteen
    segments."""
    from wind_rwkv.rwkv7 import beam_select
    B, W, V = 74, 8, 65536
    g = th.Generator(device='cuda').manual_seed(3)
    x = th.randn(B * W, V, generator=g, device='cuda') * 3
    for shift in (0., 20., 100., -1000., 10000.):
        logits = (x + shift).to(dtype)
        want, tol = [], 0.
        for rows in logits.split(74):
            d = rows.double()
            m = d.amax(-1, keepdim=True)
            p = th.exp(d - m)
            z = p.transpose(0, 1).contiguous().sum(0)
            want.append(-z.log())
            tol = max(tol, float(((p * (m - d)).sum(-1) / z).max()))
        want = th.cat(want).view(B * W, 1)          # the best candidate's log-probability
        tol = 2 ** -22 + 2 ** -23 * tol + 70 * 2 ** -24
        scores = -want.float()
        got, _, tokens = beam_select(logits.view(B * W, 1, V), scores)
        err = (got.double() - (want + scores.double())).abs() - 2.0 ** -24 * 1e-5
        assert bool((err <= tol).all()), (shift, float(err.max()))
        assert th.equal(logits.gather(1, tokens), logits.amax(-1, keepdim=True))


@pytest.mark.parametrize('dtype', [th.bfloat16, th.float32])
@pytest.mark.parametrize('W,V', [(1, 300), (2, 300), (6, 5000)])
def test_scores_at_the_end_of_the_range(W, V, dtype):
    """Beams whose score is fp32's lowest value: a candidate below it that rounds to it counts, one that rounds to -inf does not."""
    from wind_rwkv.rwkv7 import beam_select
    low = th.finfo(th.float32).min
    for score in (low, low / 2):
        for fill in (-1e30, -3e30, -2e31, low / 2, low):
            for left in (0, 1, 2, 40):
                logits, scores = make(2, W, V, dtype, seed=left)
                keep = logits[..., 5:5 + left].clone()
                logits.fill_(max(fill, th.finfo(dtype).min))
                logits[..., 5:5 + left] = keep
                scores.fill_(score)
                scores[1, :-1] = -INF
                every = reference(logits, scores, 1)[2]
                every = th.where(every.float() > -INF, every, -INF)
                best, index = every.sort(dim=1, descending=True, stable=True)
                for k in (1, 4, 64):
                    got, parents, tokens = beam_select(logits, scores, k)
                    assert th.equal(got, best[:, :k].float()) and th.equal(parents * V + tokens, index[:, :k])


def test_orders():
    """Sorted vocabularies, and candidates that crowd into one segment or one thread's segments."""
    V = 20000
    up = (th.arange(V, device='cuda') / V).expand(1, 3, V).contiguous()
    _, scores = make(1, 3, V)
    for t in (up, up.flip(2), up.bfloat16(), up.flip(2).bfloat16(), up * 1e-6, up * 1e-6 + 100):
        for k in (1, 3, 64):
            compare(t, scores, k)
    logits, scores = make(2, 16, V, th.float32)
    logits[0, 3, 512:768] += 50
    logits[1, :, ::256] += 50
    for k in (16, 64):
        compare(logits, scores, k)


def test_finished():
    for V in (1000, 4097):
        for pattern in ([0, 0, 0, 0], [1, 0, 0, 1], [1, 1, 1, 1]):
            logits, scores = make(2, 4, V)
            finished = th.tensor([pattern, pattern[::-1]], device='cuda').bool()
            logits[:, 3] = float('nan')
            for eos in (0, V // 2, V - 1):
                for k in (1, 4, 8):
                    compare(logits, scores, k, finished, eos)


def test_refusals_with_device_tensors():
    from wind_rwkv.rwkv7 import beam_select, reorder_states
    logits, scores = make(2, 4, 100)
    fin = th.zeros(2, 4, dtype=th.bool, device='cuda')
    for bad in (dict(eos=-1), dict(eos=3), dict(finished=fin), dict(finished=fin, eos=-1), dict(finished=fin, eos=100), dict(k=0), dict(k=-1), dict(k=65)):
        with pytest.raises(ValueError, match='beam_select'):
            beam_select(logits, scores, **bad)
    with pytest.raises(RuntimeError):
        beam_select(logits, scores.cpu())
    t, p = th.zeros(8, 6, device='cuda'), th.zeros(2, 4, dtype=th.int64, device='cuda')
    for states, parents in (([t, t], p), ([t[:, :4], t[:, 3:]], p), ([p.view(8, 1)], p), ([t], p[:, :3]), ([t[:7]], p)):
        with pytest.raises(ValueError, match='reorder_states'):
            reorder_states(states, parents, inplace=True)
    with pytest.raises(RuntimeError):
        reorder_states([t, t.cpu()], p)


def test_layouts():
    base, scores = make(3, 5, 4100)
    for view in (base[:, :, 1:], base[:, :, 3:4000], base.transpose(0, 1)[:3, :3], base[:, ::2], base[..., ::3], base[:, :, 8:4096]):
        B, W, V = view.shape
        compare(view, scores[:1, :1].expand(B, W), 6)
        compare(view.float(), scores.t()[:W, :B].t(), 6)
    wide = th.zeros(3, 10, device='cuda')
    wide[:, ::2] = scores
    compare(base, wide[:, ::2], 5)


def test_first_step():
    """From one beam to many, and to fewer."""
    logits, scores = make(4, 1, 5000)
    compare(logits, scores.zero_(), 8)
    logits, scores = make(4, 8, 5000)
    compare(logits, scores, 2)


def test_same_results_in_a_graph_and_on_two_streams():
    from wind_rwkv.rwkv7 import beam_select
    logits, scores = make(4, 8, 30001)
    other, oscores = make(4, 8, 30001, seed=9)
    want, owant = beam_select(logits, scores), beam_select(other, oscores)
    g = th.cuda.CUDAGraph()
    with th.cuda.graph(g):
        out = beam_select(logits, scores)
    g2 = th.cuda.CUDAGraph()
    with th.cuda.graph(g2, pool=g.pool()):
        out2 = beam_select(other, oscores)
    for _ in range(3):
        g.replay()
        assert all(th.equal(a, b) for a, b in zip(out, want))
        g2.replay()
        assert all(th.equal(a, b) for a, b in zip(out2, owant))
    side = th.cuda.Stream()
    side.wait_stream(th.cuda.current_stream())
    for _ in range(5):
        a = beam_select(logits, scores)
        with th.cuda.stream(side):
            b = beam_select(other, oscores)
        th.cuda.synchronize()
        assert all(th.equal(x, y) for x, y in zip(a, want)) and all(th.equal(x, y) for x, y in zip(b, owant))


def test_python_form_and_compile():
    from wind_rwkv.rwkv7 import _lib, beam_select, reorder_states
    from wind_rwkv.rwkv7.rwkv7_beam import reorder, select
    logits, scores = make(3, 4, 999)
    finished = th.tensor([[0, 1, 0, 0]] * 3, device='cuda').bool()

    def call(logits, scores, k, finished, eos):
        return select(logits, scores, finished, k or scores.shape[1], -1 if eos is None else eos)

    compare(logits, scores, 5, finished, 7, call=call)

    def f(l, s, t, u):
        o = beam_select(l, s, finished=finished, eos=7)
        new = reorder_states([t, t[:, 0]], o[1])
        reorder_states(u, o[1], inplace=True)
        return o[0], o[2], o[3], new[0] * 1, new[1]

    t = th.randn(12, 3, 5, device='cuda')
    us = [t.clone(), t.clone()]
    for a, b in zip(f(logits, scores, t, us[0]), th.compile(f, fullgraph=True)(logits, scores, t, us[1])):
        assert th.equal(a, b)
    assert th.equal(*us)
    p = beam_select(logits, scores)[1]
    assert all(th.equal(a, b) for a, b in zip(reorder([t, t[:, 0]], p), reorder_states([t, t[:, 0]], p)))
    assert _lib.device_status() == 0


# ---- reorder_states ------------------------------------------------------------------------------------
def parents_of(B, W, k, seed, dtype=th.int64):
    return th.randint(0, W, (B, k), generator=th.Generator().manual_seed(seed)).to('cuda', dtype)


def rows_of(parents, W):
    return (th.arange(parents.shape[0], device='cuda')[:, None] * W + parents.long()).view(-1)


def tensors(rows, seed=0):
    g = th.Generator(device='cuda').manual_seed(seed)
    wide = th.randn(rows, 40, generator=g, device='cuda')
    return [th.randn(rows, 2, 64, 64, generator=g, device='cuda'), th.randn(rows, 768, generator=g, device='cuda').bfloat16(),
            th.randint(0, 99, (rows, 37), generator=g, device='cuda'), th.randint(0, 99, (rows, 5), generator=g, device='cuda', dtype=th.int32),
            th.rand(rows, generator=g, device='cuda') < 0.5, th.randn(rows, 3, 7, generator=g, device='cuda').half(), wide[:, 1:20], wide[:, 20:33]]


@pytest.mark.parametrize('B,W,k', [(1, 1, 1), (1, 4, 4), (3, 2, 5), (2, 8, 8), (5, 9, 3), (2, 16, 16), (2, 17, 17), (1, 32, 32), (2, 33, 33), (1, 64, 64), (3, 1, 64), (3, 64, 1)])
@pytest.mark.parametrize('dtype', [th.int64, th.int32])
def test_reorder(B, W, k, dtype):
    from wind_rwkv.rwkv7 import reorder_states
    for seed in range(3):
        p = parents_of(B, W, k, seed, dtype)
        if seed == 1 and W == k:
            p = th.arange(k, device='cuda').roll(1).expand(B, k).contiguous().to(dtype)      # one cycle through all rows
        ts = tensors(B * W, seed)
        want = [t[rows_of(p, W)] for t in ts]
        before = [t.clone() for t in ts]
        out = reorder_states(ts, p)
        assert all(th.equal(a, b) for a, b in zip(out, want)) and all(th.equal(a, b) for a, b in zip(ts, before))
        assert th.equal(reorder_states(ts[0], p), want[0])
        if W == k:
            versions = [t._version for t in ts]
            out = reorder_states(ts, p, inplace=True)
            assert all(a is b for a, b in zip(out, ts)) and all(th.equal(a, b) for a, b in zip(ts, want))
            assert all(t._version > v for t, v in zip(ts, versions))
            assert reorder_states(ts[1], p, inplace=True) is ts[1]


def test_reorder_in_place_leaves_what_is_beside():
    from wind_rwkv.rwkv7 import reorder_states
    for cut in (slice(4, 20), slice(1, 20), slice(0, 40)):
        wide = th.randn(13, 40, device='cuda')
        want = wide.clone()
        p = parents_of(3, 4, 4, 1)
        want[:12, cut] = wide[:12, cut][rows_of(p, 4)]
        reorder_states(wide[:12, cut], p, inplace=True)
        assert th.equal(wide, want)


def test_reorder_many_and_empty():
    from wind_rwkv.rwkv7 import reorder_states
    p = parents_of(2, 4, 4, 0)
    ts = [th.randn(8, 1 + i % 9, device='cuda') for i in range(150)]
    want = [t[rows_of(p, 4)] for t in ts]
    assert all(th.equal(a, b) for a, b in zip(reorder_states(ts, p), want))
    reorder_states(ts, p, inplace=True)
    assert all(th.equal(a, b) for a, b in zip(ts, want))
    assert reorder_states([], p) == []
    e = th.zeros(8, 0, 5, device='cuda')
    assert reorder_states([e, ts[0]], p)[0].shape == (8, 0, 5)
    assert reorder_states(th.zeros(0, 3, device='cuda'), th.zeros(0, 4, dtype=th.int64, device='cuda')).shape == (0, 3)
    assert th.equal(reorder_states(ts[3].t().contiguous().t(), p), ts[3][rows_of(p, 4)])
    stacked = th.randn(8, 6, 3, 4, device='cuda')                       # layers as slices of one tensor
    want = stacked[rows_of(p, 4)]
    reorder_states(list(stacked.unbind(1)), p, inplace=True)
    assert th.equal(stacked, want)


def test_parent_that_does_not_exist():
    from wind_rwkv.rwkv7 import _lib, reorder_states
    t = th.randn(8, 33, device='cuda')
    before = t.clone()
    p = th.tensor([[0, 4, 1, -1], [3, 2, 1 << 40, 0]], device='cuda')
    rows = [0, None, 1, None, 7, 6, None, 4]
    out = reorder_states(t, p)
    th.cuda.synchronize()
    with pytest.raises(RuntimeError, match='parent beam that does not exist'):
        reorder_states(t, th.zeros_like(p))
    assert _lib.device_status() == -11 and _lib.device_status() == 0
    for i, r in enumerate(rows):
        assert th.equal(out[i], th.zeros_like(out[i]) if r is None else t[r])
    reorder_states(t, p, inplace=True)
    assert _lib.device_status() == -11
    for i, r in enumerate(rows):
        assert th.equal(t[i], before[i if r is None else r])


@pytest.mark.parametrize('dynamic', [False, True])
def test_compiled_in_place(dynamic):
    """Traced in place: a parent that does not exist leaves its row as it is, states that share memory are refused, rows that lie in wider tensors, layers of one tensor, and
    states made inside the traced function."""
    from wind_rwkv.rwkv7 import _lib, reorder_states
    th.compiler.reset()

    def f(ts, p):
        made = ts[0] * 2
        reorder_states([made, *ts], p, inplace=True)
        return [made + 1] + [t * 1 for t in ts]

    g = th.compile(f, fullgraph=True, dynamic=dynamic)
    for B, W in ((2, 4), (3, 5), (1, 64)):
        p = parents_of(B, W, W, 1)
        for bad in (False, True):
            if bad:
                p[0, 1], p[-1, -1] = W, -1
            wide = th.randn(B * W, 40, device='cuda')
            both = [[t.clone() for t in tensors(B * W)[:4]] + list((w := wide.clone())[:, :36].unflatten(1, (4, 9)).unbind(1)) + [w] for _ in range(2)]
            outs = []
            for call, (*ts, w) in zip((f, g), both):
                outs.append(call(ts, p))
                th.cuda.synchronize()
                assert _lib.device_status() == (-11 if bad else 0)
                assert all(th.equal(o, t) for o, t in zip(outs[-1][1:], ts))
            assert all(th.equal(a, b) for a, b in zip(*both)) and all(th.equal(a, b) for a, b in zip(*outs))
            assert th.equal(both[1][-1][:, 36:], wide[:, 36:])
    t, p = th.randn(8, 6, device='cuda'), parents_of(2, 4, 4, 0)
    before = t.clone()
    for ts in ([t, t], [t[:, :4], t[:, 3:]], [t[:, :3], t[:, 1:4], t[:, 4:]]):
        th.compiler.reset()
        with pytest.raises(ValueError, match='share memory'):
            th.compile(f, dynamic=dynamic)(ts, p)
        assert th.equal(t, before)
    th.compiler.reset()
    with pytest.raises(ValueError, match='share memory'):
        th.compile(lambda s, p: reorder_states([s], p, inplace=True)[0] * 1, dynamic=dynamic)(p.view(8, 1), p)
    q = th.zeros(8, 2, device='cuda', requires_grad=True)
    with th.no_grad():
        th.compile(lambda s, p: reorder_states(s, p, inplace=True) * 1, dynamic=dynamic)(q, p)


def test_large_offsets():
    """States whose rows lie beyond 2^32 bytes."""
    from wind_rwkv.rwkv7 import reorder_states
    t = th.zeros(6, 1 << 28, device='cuda')
    t[:, -1] = th.arange(6, device='cuda')
    t[:, 5] = th.arange(6, device='cuda') + 10
    p = th.tensor([[2, 2, 0], [1, 0, 2]], device='cuda')
    reorder_states(t, p, inplace=True)
    assert t[:, -1].tolist() == [2, 2, 0, 4, 3, 5] and t[:, 5].tolist() == [12, 12, 10, 14, 13, 15]
    del t
    logits = th.zeros(2, 64, 1 << 24, dtype=th.bfloat16, device='cuda')
    logits[1, 63, -3] = 30.
    logits[1, 40, 7] = 29.
    from wind_rwkv.rwkv7 import beam_select
    s, parents, tokens = beam_select(logits, th.zeros(2, 64, device='cuda'), 3)
    assert parents[1].tolist() == [63, 40, 0] and tokens[1].tolist() == [(1 << 24) - 3, 7, 0] and parents[0].tolist() == [0, 0, 0] and tokens[0].tolist() == [0, 1, 2]


def test_a_search():
    """Decode, head, selection and reordering together, against the same search in 64 bits on the same weights: attn_step on beams, linear as its
    head, states that follow.  The scores agree within the path's own error; that a search that keeps its states right would differ by more is
    seen from one that does not reorder them."""
    from wind_rwkv.rwkv7 import attn_step, beam_select, linear, reorder_states
    B, W, H, V, steps = 2, 4, 2, 500, 6
    C = 64 * H
    g = th.Generator(device='cuda').manual_seed(5)
    emb = th.randn(V, 6, C, generator=g, device='cuda') * 0.5
    emb[:, 1] = emb[:, 1] * 0.3 - 0.6
    kappa = th.nn.functional.normalize(th.randn(V, H, 64, generator=g, device='cuda'), dim=-1).view(V, C)
    emb[:, 4], emb[:, 5] = -kappa, kappa * 0.5
    emb = emb.bfloat16()
    head = (th.randn(V, C, generator=g, device='cuda') / C ** 0.5).bfloat16()

    def search(reorder):
        state = th.zeros(B * W, H, 64, 64, device='cuda')
        last = th.zeros(B, W, dtype=th.int64, device='cuda')
        hist = th.zeros(B * W, steps, dtype=th.int64, device='cuda')
        scores = th.full((B, W), -INF, device='cuda')
        scores[:, 0] = 0
        for i in range(steps):
            r, w, k, v, a, b = emb[last.view(-1)].unbind(1)
            y, _ = attn_step(*[t[:, None] for t in (r, w, k, v, a, b)], 64, state, inplace=True)
            logits = linear(y[:, 0], head, out_dtype=th.float32)
            scores, parents, last = beam_select(logits.view(B, W, V), scores)
            if reorder:
                reorder_states([state, hist], parents, inplace=True)
            hist[:, i] = last.view(-1)
        return scores, hist.view(B, W, steps)

    def replay(hist):
        """The log-probability of a token history in 64 bits."""
        S = th.zeros(H, 64, 64, dtype=th.float64, device='cuda')
        total, tok = 0., 0
        E, hd = emb.double(), head.double()
        for nxt in hist.tolist():
            r, w, k, v, a, b = E[tok].view(6, H, 64).unbind(0)
            S = S * th.exp(-th.exp(w))[:, None, :] + (S @ a[..., None]) * b[:, None, :] + v[..., None] * k[:, None, :]
            y = (S @ r[..., None])[..., 0].reshape(C)
            total += float(th.log_softmax(y @ hd.T, -1)[nxt])
            tok = nxt
        return total

    scores, hist = search(True)
    err = max(abs(replay(hist[b, w]) - float(scores[b, w])) for b in range(B) for w in range(W))
    # y is rounded to bf16 (2^-8 relative) before the head: a logit, a sum of C terms of size |y| / sqrt(C), moves by some 2^-8 |y|, and the score by that each step
    assert err < steps * 2 * 2.0 ** -8 * 8, err
    assert th.equal(search(True)[1], hist)
