"""What beam_select and reorder_states refuse, and what their C entry points check before they touch CUDA (no GPU needed)."""
import ctypes

import pytest
import torch as th

P = 0x1000


@pytest.fixture(scope='module')
def lib():
    import __graft_entry__ as ge
    ge.build()
    from wind_rwkv.rwkv7 import _lib
    return _lib.lib()


def select(lib, B=2, W=4, V=100, k=4, eos=-1, sb=400, sw=100, f32=0, logits=P, scores=P, fin=None, out=P, parents=P, tokens=P, ofin=None, ws=P):
    return lib.wkv7_beam_select(logits, scores, fin, out, parents, tokens, ofin, B, W, V, k, eos, sb, sw, f32, ws, None)


def test_select_checks(lib):
    assert select(lib, B=-1) == select(lib, W=0) == select(lib, V=0) == select(lib, k=0) == select(lib, W=65) == select(lib, k=65) == -1
    assert select(lib, W=1, V=3, k=4) == select(lib, sb=-1) == select(lib, sw=-1) == -1
    assert select(lib, fin=P, ofin=P, eos=-1) == select(lib, fin=P, ofin=P, eos=100) == -1
    assert select(lib, V=(1 << 30) + 1, W=1) == select(lib, V=1 << 27, W=16) == -8
    for name in ('logits', 'scores', 'out', 'parents', 'tokens', 'ws'):
        assert select(lib, **{name: None}) == -6
    assert select(lib, fin=P, eos=1) == -6
    assert select(lib, logits=P + 1) == select(lib, logits=P + 2, f32=1) == select(lib, scores=P + 2) == select(lib, parents=P + 4) == select(lib, ws=P + 8) == -4
    assert select(lib, B=0, logits=None) == 0
    size = lib.wkv7_beam_select_workspace_bytes
    assert size(0, 4, 100) == size(2, 0, 100) == size(2, 65, 100) == 0
    assert size(2, 4, 100) >= 2 * 4 * 4 and size(64, 16, 65536) < 64 * 16 * 65536 // 16


def reorder(lib, B=2, W=4, k=4, src=P, dst=2 * P, row=64, sp=64, dp=64, parents=P, i32=0, count=1):
    vp, i64 = ctypes.c_void_p * 1, ctypes.c_int64 * 1
    return lib.wkv7_reorder(count, vp(src), vp(dst), i64(row), i64(sp), i64(dp), parents, i32, B, W, k, None)


def test_reorder_checks(lib):
    assert reorder(lib, B=-1) == reorder(lib, W=0) == reorder(lib, k=0) == reorder(lib, W=65) == reorder(lib, k=65) == reorder(lib, count=-1) == -1
    assert reorder(lib, row=-1) == reorder(lib, sp=63) == reorder(lib, dp=63) == -1
    assert reorder(lib, dst=P, k=3) == reorder(lib, dst=P, dp=128) == -1                  # in place: as many rows, one pitch
    assert reorder(lib, i32=4) == reorder(lib, i32=-1) == reorder(lib, i32=2, k=3) == reorder(lib, i32=3, W=3) == -1
    assert reorder(lib, src=None) == reorder(lib, dst=None) == reorder(lib, parents=None) == -6
    assert reorder(lib, parents=P + 4) == reorder(lib, parents=P + 2, i32=1) == -4
    assert reorder(lib, B=0, src=None) == reorder(lib, count=0) == 0
    assert lib.wkv7_status_string(-11) not in (b'', b'unknown status') and lib.wkv7_status_string(-10) != b'unknown status'


def test_select_refusals(lib):
    from wind_rwkv.rwkv7 import beam_select
    logits, scores = th.zeros(2, 4, 50), th.zeros(2, 4)
    fin = th.zeros(2, 4, dtype=th.bool)
    for bad in (dict(k=0), dict(k=65), dict(finished=fin), dict(eos=3), dict(finished=fin, eos=50), dict(finished=fin, eos=-2), dict(finished=fin[:1], eos=3),
                dict(finished=fin.int(), eos=3)):
        with pytest.raises(ValueError, match='beam_select'):
            beam_select(logits, scores, **bad)
    for bl, bs in ((logits[0], scores), (logits.half(), scores), (logits, scores[:1]), (logits, scores.double()), (logits[:, :, :0], scores), (th.zeros(1, 65, 5), th.zeros(1, 65))):
        with pytest.raises(ValueError, match='beam_select'):
            beam_select(bl, bs)
    with pytest.raises(RuntimeError, match='CUDA'):
        beam_select(logits, scores)


@pytest.mark.parametrize('dynamic', [False, True])
def test_select_refusals_while_torch_compile_traces(lib, dynamic):
    from wind_rwkv.rwkv7 import beam_select
    logits, scores = th.zeros(2, 4, 50), th.zeros(2, 4)
    fin = th.zeros(2, 4, dtype=th.bool)

    def call(logits, scores, k=None, finished=None, eos=None):
        th.compiler.reset()
        return th.compile(lambda l, s, f: beam_select(l, s, k, finished=f, eos=eos)[0] * 1, backend='eager', dynamic=dynamic)(logits, scores, finished)

    for bad in (dict(k=0), dict(k=65), dict(finished=fin), dict(eos=3), dict(finished=fin, eos=50), dict(finished=fin, eos=-2), dict(finished=fin[:1], eos=3),
                dict(finished=fin.int(), eos=3)):
        with pytest.raises(ValueError, match='beam_select'):
            call(logits, scores, **bad)
    for bl, bs in ((logits[0], scores), (logits.half(), scores), (logits.double(), scores), (logits, scores[:1]), (logits, scores[:, :3]), (logits, scores.double()),
                   (th.zeros(1, 65, 5), th.zeros(1, 65))):
        with pytest.raises(ValueError, match='beam_select'):
            call(bl, bs)
    with pytest.raises(RuntimeError, match='CUDA'):
        call(logits, scores, None, fin, 3)


def test_reorder_refusals(lib):
    from wind_rwkv.rwkv7 import reorder_states
    t, p = th.zeros(8, 6), th.zeros(2, 4, dtype=th.int64)
    for states, parents, inplace in (([t], p.float(), False), ([t], p[0], False), ([t], p[:, :0], False), ([t, t[:4]], p, False), ([t[:7]], p, False), ([th.zeros(())], p, False),
                                     ([t], p[:, :3], True), ([th.zeros(130, 2)], p, False), ([t.t().contiguous().t()], p, True), ([t[:1].expand(8, 6)], p, True),
                                     ([t, t], p, True), ([t[:, :4], t[:, 3:]], p, True), ([t, t.view(th.int32)], p, True)):
        with pytest.raises(ValueError, match='reorder_states'):
            reorder_states(states, parents, inplace=inplace)
    q = th.zeros(8, 4, dtype=th.int64)
    with pytest.raises(ValueError, match='share memory'):
        reorder_states([q], q[:2], inplace=True)
    g = th.zeros(8, 6, requires_grad=True)
    with pytest.raises(RuntimeError, match='autograd'):
        reorder_states([g], p, inplace=True)
    with pytest.raises(RuntimeError, match='CUDA'):
        reorder_states([t[:, :3], t[:, 3:]], p, inplace=True)


@pytest.mark.parametrize('dynamic', [False, True])
def test_reorder_refusals_while_torch_compile_traces(lib, dynamic):
    from wind_rwkv.rwkv7 import reorder_states
    t, p = th.zeros(8, 6), th.zeros(2, 4, dtype=th.int64)

    def call(states, parents, inplace=False):
        th.compiler.reset()
        return th.compile(lambda ts, p: [o * 1 for o in reorder_states(ts, p, inplace=inplace)], backend='eager', dynamic=dynamic)(states, parents)

    for states, parents, inplace in (([t], p.float(), False), ([t], p[0], False), ([t], p[:, :0], False), ([t, t[:4]], p, False), ([t[:4], t], p, False), ([t[:7]], p, False),
                                     ([th.zeros(())], p, False), ([t], p[:, :3], True), ([th.zeros(130, 2)], p, False), ([t.t().contiguous().t()], p, True),
                                     ([t[:1].expand(8, 6)], p, True), ([t], th.zeros(2, 65, dtype=th.int64), False)):
        with pytest.raises(ValueError, match='reorder_states'):
            call(states, parents, inplace)
    with pytest.raises(RuntimeError, match='autograd'):
        call([th.zeros(8, 6, requires_grad=True)], p, True)
    for inplace in (False, True):
        with pytest.raises(RuntimeError, match='CUDA'):
            call([t[:, :3], t[:, 3:]], p, inplace)


def test_rows_that_share_memory():
    from wind_rwkv.rwkv7.rwkv7_beam import _overlap, _row_layout
    t = th.zeros(8, 6, 4)
    assert _row_layout(t) == (96, 96) and _row_layout(t[:, 2]) == (16, 96) and _row_layout(t[:, :, 0]) is None and _row_layout(t[:, 1:3]) == (32, 96)
    assert _row_layout(t[:1, 0]) == (16, 16) and _row_layout(t.transpose(1, 2)) is None and _row_layout(th.zeros(8)) == (4, 4)
    assert not _overlap((0, 8, 16, 96), (16, 8, 16, 96)) and _overlap((0, 8, 17, 96), (16, 8, 16, 96)) and _overlap((0, 8, 16, 96), (88, 8, 16, 96))
    assert not _overlap((0, 8, 96, 96), (768, 8, 96, 96)) and _overlap((0, 8, 16, 96), (16, 8, 16, 80)) and not _overlap((0, 8, 0, 96), (0, 8, 16, 96))
