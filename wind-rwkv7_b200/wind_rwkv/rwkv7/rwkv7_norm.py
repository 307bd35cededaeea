"""The residual stream between the mixers: `rms_norm(x, weight, residual=)`, its addition, dropout and norm in one pass, and `dropout(x, p, seed)`.

The reference leaves both to the model around the mixer.  A block of a model, in training and in serving (there with the norm in 8 bits, see rwkv7_int8.py):

    y, h = rms_norm(mixed, weight, residual=h, p=0.1, seed=seed)          # h += dropout(mixed); y = norm(h)
    q8, h = rms_norm(mixed, weight, residual=h, out_dtype=torch.int8)     # h += mixed; q8 = Int8(q, scale)

Dropout comes from a counter-based generator (Philox4x32-10): which elements are dropped is a function of the seed and of an element's place, no mask is
stored and the backward forms it again.  Kernels: csrc/norm_fwd.cu and norm_bwd.cu (rms_norm), norm.cu (dropout).  The norm is by the root mean square alone: no mean is taken off and no
bias added, so that a model with LayerNorm cannot use it.
"""
import torch as th

from . import _lib
from .rwkv7_int8 import Int8, pitch8
from .rwkv7_linear import rows_of

X_F32, R_F32, W_F32, Y_F32, Y_INT8 = 1, 2, 4, 8, 16
MAX_D = 16384
FLOATS = (th.bfloat16, th.float32)
OUTS = {None: -1, th.bfloat16: 0, th.float32: 1, th.int8: 2}  # of y, -1: x's


def f32(t):
    return t is not None and t.dtype == th.float32


def fw_norm(x, weight, residual, seed_t, eps, p, seed, out, save):
    """Launcher: y (out 0: bf16, 1: fp32, 2: 8 bits, rows pitch8(D) apart), h (empty without residual), rstd (empty unless `save`), scale (empty unless 8 bits)."""
    D = x.shape[-1]
    M = x.numel() // D
    dev, lead = x.device, x.shape[:-1]
    y = th.empty(*lead, pitch8(D) if out == 2 else D, dtype=(th.bfloat16, th.float32, th.int8)[out], device=dev)
    h = th.empty(x.shape if residual is not None else (0,), dtype=x.dtype if residual is None else residual.dtype, device=dev)
    rstd = th.empty(M if save else 0, dtype=th.float32, device=dev)
    scale = th.empty(lead if out == 2 else (0,), dtype=th.float32, device=dev)
    x, ldx = rows_of(x)
    r, ldr = (None, D) if residual is None else rows_of(residual)
    w = None if weight is None else weight.contiguous()
    flags = (X_F32 if f32(x) else 0) | (R_F32 if f32(r) else 0) | (W_F32 if f32(w) else 0) | (0, Y_F32, Y_INT8)[out]
    with _lib.on_device(x, w, r, seed_t):
        rc = _lib.lib().wkv7_rms_norm_fwd(x.data_ptr(), _lib.ptr(r), _lib.ptr(w), y.data_ptr(), h.data_ptr() if r is not None else None, rstd.data_ptr() if save else None,
                                          scale.data_ptr() if out == 2 else None, M, D, ldx, ldr, y.shape[-1], D, eps, p, seed, _lib.ptr(seed_t), flags,
                                          _lib.stream_of(x))
    _lib.check(rc, 'wkv7_rms_norm_fwd')
    return y, h, rstd, scale


def bw_norm(h, rstd, weight, dy, dh, seed_t, p, seed, x_f32, want_dx, want_dr, want_dw):
    """Launcher: dx, dr [..., D], dw [D] fp32, each empty where it is not wanted."""
    D = h.shape[-1]
    M = h.numel() // D
    dev = h.device
    dx = th.empty(h.shape if want_dx else (0,), dtype=th.float32 if x_f32 else th.bfloat16, device=dev)
    dr = th.empty(h.shape if want_dr else (0,), dtype=h.dtype, device=dev)
    dw = th.empty(D if want_dw else 0, dtype=th.float32, device=dev)
    h, ldh = rows_of(h)
    dy, lddy = rows_of(dy)
    dh, lddh = (None, D) if dh is None else rows_of(dh)
    w = None if weight is None else weight.contiguous()
    flags = (X_F32 if x_f32 else 0) | (R_F32 if f32(h) else 0) | (W_F32 if f32(w) else 0) | (Y_F32 if f32(dy) else 0)
    with _lib.on_device(h, w, dy, dh, seed_t):
        ws = th.empty(_lib.lib().wkv7_rms_norm_bwd_workspace_bytes(M, D) if want_dw else 0, dtype=th.uint8, device=dev)
        rc = _lib.lib().wkv7_rms_norm_bwd(h.data_ptr(), rstd.data_ptr(), _lib.ptr(w), dy.data_ptr(), _lib.ptr(dh), dx.data_ptr() if want_dx else None,
                                          dr.data_ptr() if want_dr else None, dw.data_ptr() if want_dw else None, M, D, ldh, lddy, lddh, D, D, p, seed,
                                          _lib.ptr(seed_t), flags, ws.data_ptr() or None, _lib.stream_of(h))
    _lib.check(rc, 'wkv7_rms_norm_bwd')
    return dx, dr, dw


def drop(x, residual, seed_t, p, seed, out_f32):
    """Launcher: residual + dropout(x), contiguous."""
    y = th.empty(x.shape, dtype=th.float32 if out_f32 else th.bfloat16, device=x.device)
    x, r = (t if t is None or (t.is_contiguous() and t.data_ptr() % 16 == 0) else t.clone(memory_format=th.contiguous_format) for t in (x, residual))
    flags = (X_F32 if f32(x) else 0) | (R_F32 if f32(r) else 0) | (Y_F32 if out_f32 else 0)
    with _lib.on_device(x, r, seed_t):
        rc = _lib.lib().wkv7_dropout(x.data_ptr(), _lib.ptr(r), y.data_ptr(), x.numel(), p, seed, _lib.ptr(seed_t), flags, _lib.stream_of(x))
    _lib.check(rc, 'wkv7_dropout')
    return y


def _fake_fw(x, weight, residual, seed_t, eps, p, seed, out, save):
    D = x.shape[-1]
    lead = x.shape[:-1]
    return (x.new_empty((*lead, pitch8(D) if out == 2 else D), dtype=(th.bfloat16, th.float32, th.int8)[out]),
            x.new_empty(x.shape if residual is not None else (0,), dtype=x.dtype if residual is None else residual.dtype),
            x.new_empty((x.numel() // D if save else 0,), dtype=th.float32), x.new_empty(lead if out == 2 else (0,), dtype=th.float32))


def _fake_bw(h, rstd, weight, dy, dh, seed_t, p, seed, x_f32, want_dx, want_dr, want_dw):
    return (h.new_empty(h.shape if want_dx else (0,), dtype=th.float32 if x_f32 else th.bfloat16), h.new_empty(h.shape if want_dr else (0,)),
            h.new_empty((h.shape[-1] if want_dw else 0,), dtype=th.float32))


_fw_op = _lib.opaque_op('rms_norm_fwd', fw_norm, _fake_fw,
                        '(Tensor x, Tensor? weight, Tensor? residual, Tensor? seed_t, float eps, float p, int seed, int out, bool save) -> (Tensor, Tensor, Tensor, Tensor)')
_bw_op = _lib.opaque_op('rms_norm_bwd', bw_norm, _fake_bw,
                        '(Tensor h, Tensor rstd, Tensor? weight, Tensor dy, Tensor? dh, Tensor? seed_t, float p, int seed, bool x_f32, bool want_dx, bool want_dr, '
                        'bool want_dw) -> (Tensor, Tensor, Tensor)')
_drop_op = _lib.opaque_op('dropout', drop, lambda x, residual, seed_t, p, seed, out_f32: x.new_empty(x.shape, dtype=th.float32 if out_f32 else th.bfloat16),
                          '(Tensor x, Tensor? residual, Tensor? seed_t, float p, int seed, bool out_f32) -> Tensor')


class NormGrad(th.autograd.Function):
    """A gradient whose own derivative is not formed.  Where autograd records the backward, the gradient stays joined to what it depends on, and a second backward that comes
    this way raises instead of leaving the term out."""
    @staticmethod
    def forward(ctx, g, *of):
        return g

    @staticmethod
    def backward(ctx, dg):
        raise RuntimeError('rms_norm has no second derivative')


class RmsNorm(th.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, seed_t, eps, p, seed, out_f32):
        grad = any(ctx.needs_input_grad[:3])
        y, h, rstd, _ = _lib.call(_fw_op, fw_norm, x, weight, residual, seed_t, eps, p, seed, int(out_f32), grad)
        if grad:
            ctx.save_for_backward(x if residual is None else h, rstd, weight, seed_t)
        ctx.how = (p, seed, x.dtype, out_f32)
        ctx.set_materialize_grads(False)
        return y, (None if residual is None else h)

    @staticmethod
    def backward(ctx, dy, dh):
        p, seed, x_dtype, out_f32 = ctx.how
        want_x, want_w, want_r = ctx.needs_input_grad[:3]
        if (dy is None and dh is None) or not (want_x or want_w or want_r):
            return (None,) * 8
        h, rstd, weight, seed_t = ctx.saved_tensors
        from_y, from_h = dy, dh
        dy = th.zeros(h.shape, dtype=th.float32 if out_f32 else th.bfloat16, device=h.device) if dy is None else dy.to(th.float32 if out_f32 else th.bfloat16)
        dh = None if dh is None else dh.to(h.dtype)
        one = not p and x_dtype == h.dtype  # x and the stream have the same gradient
        dx, dr, dw = _lib.call(_bw_op, bw_norm, h, rstd, weight, dy, dh, seed_t, p, seed, x_dtype == th.float32, want_x and not one, want_r or (want_x and one), want_w)
        dx, dw, dr = (dr if one else dx) if want_x else None, dw.to(weight.dtype) if want_w else None, dr if want_r else None
        if not th.compiler.is_compiling() and th.is_grad_enabled():
            h = h if want_x or want_r else None  # (as an output it belongs to the graph for the weight's sake alone, too)
            dx, dr = (g if g is None else NormGrad.apply(g, from_y, from_h, h, weight) for g in (dx, dr))
            dw = dw if dw is None else NormGrad.apply(dw, from_y, h)
        return dx, dw, dr, None, None, None, None, None


class Dropout(th.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, seed_t, p, seed, out_f32=None):
        ctx.save_for_backward(seed_t)
        ctx.how = (p, seed, x.dtype)
        return _lib.call(_drop_op, drop, x, residual, seed_t, p, seed, f32(x if residual is None else residual) if out_f32 is None else out_f32)

    @staticmethod
    def backward(ctx, dy):
        p, seed, x_dtype = ctx.how
        dx = None
        if ctx.needs_input_grad[0]:
            how = (ctx.saved_tensors[0], p, seed, x_dtype == th.float32)
            # (where autograd records the backward dx is dropout of dy, and differentiated as such)
            again = not th.compiler.is_compiling() and th.is_grad_enabled() and dy.requires_grad
            dx = Dropout.apply(dy, None, *how) if again else _lib.call(_drop_op, drop, dy, None, *how)
        return dx, dy if ctx.needs_input_grad[1] else None, None, None, None, None


def _check_floats(name, what, t, shape=None):
    if t.dtype not in FLOATS:
        raise TypeError(f'{name} takes {what} in bfloat16 or float32, not {t.dtype}')
    if shape is not None and list(t.shape) != list(shape):
        raise ValueError(f'{name} takes {what} {list(shape)}, got {list(t.shape)}')


def _check_dropout(name, p, seed):
    """(p, seed as a number, seed as a tensor or None)"""
    if not 0 <= p <= 1:
        raise ValueError(f'{name}: p is a probability, got {p}')
    if isinstance(seed, th.Tensor):
        if seed.dtype != th.int64 or seed.numel() != 1:
            raise ValueError(f'{name}: a seed on the device is one int64, got {list(seed.shape)} {seed.dtype}')
        return float(p), 0, seed.detach()
    if seed is None and p > 0:
        raise ValueError(f'{name} needs a seed where p > 0')
    if seed is not None and not (0 <= seed < 1 << 63 and int(seed) == seed):
        raise ValueError(f'{name}: a seed is an integer from 0 to 2^63 - 1, got {seed}')
    return float(p), 0 if seed is None else int(seed), None


def _check_norm(x, weight, residual, eps, p, seed, out_dtype):
    _check_floats('rms_norm', 'x', x)
    if x.dim() < 1 or not 0 < x.shape[-1] <= MAX_D:
        raise ValueError(f'rms_norm takes x [..., D] of 1 to {MAX_D} elements a row, got {list(x.shape)}')
    if weight is not None:
        _check_floats('rms_norm', 'weight', weight, x.shape[-1:])
    if residual is not None:
        _check_floats('rms_norm', 'residual', residual, x.shape)
    if out_dtype not in (None, th.int8, *FLOATS):
        raise TypeError(f'rms_norm gives bfloat16, float32 or int8, not {out_dtype}')
    if not eps >= 0:
        raise ValueError(f'rms_norm: eps is not negative, got {eps}')
    how = _check_dropout('rms_norm', p, seed)
    if p > 0 and residual is None:
        raise ValueError('rms_norm: dropout is of what joins the residual stream; without one use dropout()')
    if out_dtype == th.int8 and th.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, residual)):
        raise RuntimeError('rms_norm in 8 bits has no backward: call it under torch.no_grad()')
    if out_dtype == th.int8:
        _lib.refuse_tangents('rms_norm in 8 bits', x, weight, residual)
    return how


def rms_norm(x, weight=None, *, residual=None, eps=1e-5, p=0.0, seed=None, out_dtype=None):
    """y = h weight / sqrt(mean(h^2) + eps) over the last dimension, h = residual + dropout(x): returns y, or (y, h) with a residual.

    x [..., D] bf16 or fp32, D up to 16384; weight [D] bf16 or fp32, or None; residual [..., D] bf16 or fp32, whose type h has: the stream, rounded to it, is what is normed.
    y has x's type unless out_dtype says bf16, fp32 or int8; int8 gives Int8(q, scale) for linear_int8 (see quantize), without a backward.  p, seed: of dropout(),
    elements counted in row-major order.  Backward for x, weight and residual; a second derivative is refused.  Squares are summed in fp32: a row
    beyond 1e19 leaves its range and gives 0 (with eps = 0, one below 1e-19 infinities).  Rows may lie in a wider tensor; other layouts are copied."""
    if not th.compiler.is_compiling():
        number, seed_t = _seed_of(seed)
        out = _lib.ext().rms_norm(x, weight, residual, eps, p, number, seed_t, OUTS.get(out_dtype, -2))
        if out is not None:
            if out_dtype is not th.int8:
                return out
            return Int8(*out) if residual is None else (Int8(out[0], out[1]), out[2])
    p, number, seed_t = _check_norm(x, weight, residual, eps, p, seed, out_dtype)
    _lib.require_cuda(x, weight, residual, seed_t)
    if out_dtype == th.int8:
        q, h, _, scale = _lib.call(_fw_op, fw_norm, x.detach(), None if weight is None else weight.detach(), None if residual is None else residual.detach(), seed_t,
                                   float(eps), p, number, 2, False)
        q8 = Int8(q[..., :x.shape[-1]], scale)
        return q8 if residual is None else (q8, h)
    y, h = RmsNorm.apply(x, weight, residual, seed_t, float(eps), p, number, f32(x) if out_dtype is None else out_dtype == th.float32)
    return y if residual is None else (y, h)


def _seed_of(seed):
    """(number, tensor or None) for the eager path, which leaves what it does not know to the checks; -1: no number given, -2: not a seed."""
    if seed is None or isinstance(seed, th.Tensor):
        return -1, seed
    return (seed if isinstance(seed, int) and 0 <= seed < 1 << 63 else -2), None


def dropout(x, p, seed, *, residual=None):
    """residual + x / (1 - p) where an element of x is kept, residual (0 without one) where it is dropped; p in [0, 1].

    x [...] bf16 or fp32; residual of x's shape, bf16 or fp32, whose type the result then has.  Which elements are dropped is a function of the seed and of an element's
    place in row-major order: equal seeds drop equal elements, so each layer and step takes its own.  seed: an integer from 0 to 2^63 - 1, or an int64 tensor
    of one element on x's device, which is read when the kernel runs (a captured step draws anew when the tensor was changed before its replay).  A probability
    is met to 2^-33.  Backward for x and residual, to any order; no mask is stored."""
    if not th.compiler.is_compiling():
        number, seed_t = _seed_of(seed)
        out = _lib.ext().dropout(x, p, number, seed_t, residual)
        if out is not None:
            return out
    _check_floats('dropout', 'x', x)
    if residual is not None:
        _check_floats('dropout', 'residual', residual, x.shape)
    if seed is None:
        raise ValueError('dropout needs a seed')
    p, number, seed_t = _check_dropout('dropout', p, seed)
    _lib.require_cuda(x, residual, seed_t)
    return Dropout.apply(x, residual, seed_t, p, number)
