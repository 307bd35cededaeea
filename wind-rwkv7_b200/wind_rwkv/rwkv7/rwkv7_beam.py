"""Beam search around the decode step: `beam_select` picks each sequence's best continuations, `reorder_states` lets the recurrent
states follow.  The reference has no decoding; the states are those that `attn_step` keeps (fp32 [rows, H, 64, 64]) and whatever else a program
keeps per beam (token-shift rows, token histories).  A step of a search over B sequences with W beams, rows b * W + w:

    y, S = attn_step(r, w, k, v, a, b, 64, S, inplace=True)       # every layer
    scores, parents, tokens = beam_select(logits.view(B, W, V), scores)
    reorder_states([S, shift, history], parents, inplace=True)

Kernels: csrc/beam.cu.  No autograd.
"""
import ctypes

import torch as th

from . import _lib

MAX_BEAMS = 64
I32, KEEP = 1, 2


def select(logits, scores, finished, k, eos):
    """Launcher: (scores fp32, parents, tokens int64, finished bool (empty without `finished`)), each [B, k]."""
    B, W, V = logits.shape
    dev = logits.device
    if V > 1 and logits.stride(2) != 1:
        logits = logits.contiguous()
    scores = scores.contiguous()
    fin = None if finished is None else finished.contiguous()
    out = th.empty(B, k, dtype=th.float32, device=dev)
    parents, tokens = (th.empty(B, k, dtype=th.int64, device=dev) for _ in range(2))
    out_fin = th.empty(B if fin is not None else 0, k, dtype=th.bool, device=dev)
    ws = th.empty(_lib.lib().wkv7_beam_select_workspace_bytes(B, W, V), dtype=th.uint8, device=dev)
    with _lib.on_device(logits, scores, fin):
        rc = _lib.lib().wkv7_beam_select(logits.data_ptr(), scores.data_ptr(), _lib.ptr(fin), out.data_ptr(), parents.data_ptr(), tokens.data_ptr(),
                                         out_fin.data_ptr() if fin is not None else None, B, W, V, k, eos, logits.stride(0), logits.stride(1),
                                         int(logits.dtype == th.float32), ws.data_ptr(), _lib.stream_of(logits))
    _lib.check(rc, 'wkv7_beam_select')
    return out, parents, tokens, out_fin


def _fake_select(logits, scores, finished, k, eos):
    B = logits.shape[0]
    return (logits.new_empty((B, k), dtype=th.float32), logits.new_empty((B, k), dtype=th.int64), logits.new_empty((B, k), dtype=th.int64),
            logits.new_empty((B if finished is not None else 0, k), dtype=th.bool))


_select_op = _lib.opaque_op('beam_select', select, _fake_select,
                            '(Tensor logits, Tensor scores, Tensor? finished, int k, int eos) -> (Tensor, Tensor, Tensor, Tensor)')


def _check_select(logits, scores, k, finished, eos):
    if logits.dim() != 3 or logits.dtype not in (th.bfloat16, th.float32):
        raise ValueError(f'beam_select takes logits [B, W, V] in bfloat16 or float32, got {list(logits.shape)} {logits.dtype}')
    B, W, V = logits.shape
    if scores.dtype != th.float32 or list(scores.shape) != [B, W]:
        raise ValueError(f'beam_select takes scores {[B, W]} in float32, got {list(scores.shape)} {scores.dtype}')
    if not (1 <= W <= MAX_BEAMS and 1 <= k <= MAX_BEAMS and V >= 1 and k <= W * V):
        raise ValueError(f'beam_select takes 1 to {MAX_BEAMS} beams and k of 1 to {MAX_BEAMS}, at most W * V: got W = {W}, k = {k}, V = {V}')
    if (finished is None) != (eos is None):
        raise ValueError('beam_select: finished and eos come together')
    if finished is not None:
        if finished.dtype != th.bool or list(finished.shape) != [B, W]:
            raise ValueError(f'beam_select takes finished {[B, W]} in bool, got {list(finished.shape)} {finished.dtype}')
        if not 0 <= eos < V:
            raise ValueError(f'beam_select: eos {eos} is no token of {V}')


def beam_select(logits, scores, k=None, *, finished=None, eos=None):
    """The k (default: W) best continuations of each sequence: (scores fp32, parents int64, tokens int64), each [B, k], best first.

    logits [B, W, V] bf16 or fp32 (not normalised; any strides of the first two dimensions), scores [B, W] fp32 sums of log-probabilities.  A candidate's
    score is its beam's plus its log-softmax; equal ones are ordered by beam, then token.  Logits of -inf, +inf and NaN are ruled out, and so are beams of
    such a score (-inf: a beam that is not there, as all but the first are at the start); where too few candidates are left the rest have score
    -inf.  finished [B, W] bool with eos: an ended beam goes on with eos alone, its score unchanged, and a fourth output [B, k] says who has
    ended.  Up to 64 beams and 64 results.  No autograd."""
    k = logits.shape[1] if k is None and logits.dim() == 3 else k
    if not th.compiler.is_compiling():
        out = _lib.ext().beam_select(logits, scores, -1 if k is None else k, finished, -1 if eos is None else eos if eos >= 0 else -2)
        if out is not None:
            return out
    _check_select(logits, scores, k, finished, eos)  # (while torch.compile traces, too: the launcher takes what it is given)
    _lib.require_cuda(logits, scores, finished)
    out, parents, tokens, fin = _lib.call(_select_op, select, logits.detach(), scores.detach(), finished, k, -1 if eos is None else eos)
    return (out, parents, tokens) if finished is None else (out, parents, tokens, fin)


def _row_layout(t):
    """(bytes of a row, pitch in bytes) of t [rows, ...], whose rows lie apart and each in one piece; None otherwise."""
    size, n = t.element_size(), 1
    for length, stride in zip(reversed(t.shape[1:]), reversed(t.stride()[1:])):
        if length != 1 and stride != n:
            return None
        n *= length
    pitch = n if t.shape[0] <= 1 else t.stride(0)
    return (n * size, pitch * size) if pitch >= n else None


def _overlap(a, b):
    """Whether rows of a and b, each (start, rows, row bytes, pitch), share memory; strided ones of different pitch count as if they did."""
    (p, m, n, ld), (q, r, o, le) = sorted((a, b))
    if min(m, n, r, o) == 0 or q >= p + (m - 1) * ld + n:
        return False
    d = (q - p) % ld
    return not (ld == le and d >= n and d + o <= ld)


def reorder(states, parents, replaces=False):
    """Launcher: the reordered states, as new tensors.  `replaces`: the states will be overwritten with them, so that what holds in place holds here: a row
    whose parent does not exist stays, and no two states share memory (which only addresses show; they cannot be looked at while a call is traced)."""
    B, k = parents.shape
    if replaces:
        _check_apart(states, parents)
    outs = [th.empty((B * k, *t.shape[1:]), dtype=t.dtype, device=t.device) for t in states]
    states = [t.resolve_conj().resolve_neg() for t in states]
    _launch([t if _row_layout(t) else t.contiguous() for t in states], outs, parents, KEEP if replaces else 0)
    return outs


def _launch(src, dst, parents, flags=0):
    B, k = parents.shape
    if B == 0 or not src:
        return
    ps, pd = [_row_layout(t) for t in src], [_row_layout(t) for t in dst]
    n = len(src)
    ptrs, i64s = ctypes.c_void_p * n, ctypes.c_int64 * n
    parents = parents.contiguous()
    with _lib.on_device(parents, *src, *dst):
        rc = _lib.lib().wkv7_reorder(n, ptrs(*[t.data_ptr() for t in src]), ptrs(*[t.data_ptr() for t in dst]), i64s(*[p[0] for p in ps]), i64s(*[p[1] for p in ps]),
                                     i64s(*[p[1] for p in pd]), parents.data_ptr(), flags | (I32 if parents.dtype == th.int32 else 0), B, src[0].shape[0] // B, k, _lib.stream_of(parents))
    _lib.check(rc, 'wkv7_reorder')


_reorder_op = _lib.opaque_op('reorder_states', reorder, lambda states, parents, replaces: [t.new_empty((parents.numel(), *t.shape[1:])) for t in states],
                             '(Tensor[] states, Tensor parents, bool replaces) -> Tensor[]')


def _check_reorder(states, parents, inplace):
    if parents.dim() != 2 or parents.dtype not in (th.int64, th.int32):
        raise ValueError(f'reorder_states takes parents [B, k] in int64 or int32, got {list(parents.shape)} {parents.dtype}')
    B, k = parents.shape
    if k < 1 or k > MAX_BEAMS:
        raise ValueError(f'reorder_states takes 1 to {MAX_BEAMS} parents a sequence, got {k}')
    if any(t.dim() == 0 or t.shape[0] != states[0].shape[0] for t in states):
        raise ValueError(f'reorder_states: all states have a row per beam, got {[list(t.shape) for t in states]}')
    if states:
        n = states[0].shape[0]
        if (n % B or not 1 <= n // B <= MAX_BEAMS) if B else n:
            raise ValueError(f'reorder_states: {n} rows are not 1 to {MAX_BEAMS} beams for each of {B} sequences')
        if inplace and n != B * k:
            raise ValueError(f'reorder_states in place keeps the number of rows: {n} rows, parents {[B, k]}')
    if inplace:
        if th.is_grad_enabled() and any(t.requires_grad for t in states):
            raise RuntimeError('reorder_states has no autograd: in place it takes states that require no gradient')
        if any(_row_layout(t) is None for t in states):
            raise ValueError('reorder_states in place takes states whose rows are contiguous and apart')


def _check_apart(states, parents):
    at = [(t.data_ptr(), t.shape[0], *lay) for t in states if (lay := _row_layout(t))]
    at = sorted(at + [(parents.data_ptr(), 1, parents.numel() * parents.element_size(), 1)])
    for i, a in enumerate(at):
        for b in at[i + 1:]:
            if b[0] >= a[0] + max(a[1] * a[3], a[2]):
                break
            if _overlap(a, b):
                raise ValueError('reorder_states in place: two of the states, or one and parents, share memory')


def reorder_states(states, parents, *, inplace=False):
    """Row b * k + j of each state := row b * W + parents[b, j], for a tensor or a sequence of tensors [B * W, ...] of any type; parents [B, k].

    Returns a tensor, or a list of them, of B * k rows; with inplace=True (k == W) the states themselves, of which only rows that change are
    touched.  All tensors in one launch (64 at a time).  A parent outside 0 .. W - 1 leaves its row zero (in place: as it is), and the next call that looks
    at the device status raises.  No autograd.  (While torch.compile traces, in place is a reordering out of place and a copy back.)"""
    one = isinstance(states, th.Tensor)
    ts = [states] if one else list(states)
    if not th.compiler.is_compiling():
        out = _lib.ext().reorder_states(ts, parents, inplace)
        if out is None:
            _check_reorder(ts, parents, inplace)
            if inplace:
                _check_apart(ts, parents)
            _lib.require_cuda(parents, *ts)
            if inplace:
                _launch(ts, ts, parents)
                out = ts
                th.autograd.graph.increment_version([t for t in ts if not t.is_inference()])
            else:
                out = reorder([t.detach() for t in ts], parents)
        return out[0] if one else out
    _check_reorder(ts, parents, inplace)  # (the launcher takes what it is given)
    _lib.require_cuda(parents, *ts)
    out = _reorder_op([t.detach() for t in ts], parents, inplace)
    if inplace:
        for t, o in zip(ts, out):
            t.copy_(o)
        out = ts
    return out[0] if one else out
