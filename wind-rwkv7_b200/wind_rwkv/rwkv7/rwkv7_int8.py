"""Products in 8 bits for serving: `quantize(x)` gives rows as integers with a scale each, `linear_int8(x, w, ...)` multiplies two such tensors.

The weight's stream, which bounds the generation of a few sequences, is half of bf16's, and so is the tensor cores' time for a prompt.  The rows' own way to 8 bits comes on
top.  With it large prompts through wide weights and a head take 0.6 to 0.7 of `linear`'s time.  A few tokens' calls wait for the host; in a captured graph one token gains (1 x 2048 -> 8192 with its norm 7.1
us, in bf16 11.5), 24 x 8192 -> 2048 does not (12.5, 11.9).  Weights are quantized once, a scale a channel; activations row by row, by `rms_norm(..., out_dtype=torch.int8)` where a norm precedes the product and by `quantize` elsewhere:

    w8 = quantize(w)                                                     # once: w [N, K]
    q8, h = rms_norm(mixed, weight, residual=h, out_dtype=torch.int8)
    k = linear_int8(q8, wk8, act='relu2')                                # channel mixer
    h = linear_int8(quantize(k), wv8, residual=h)

Kernels: csrc/norm.cu (quantize), csrc/linear.cu (products, on the 8-bit integer tensor cores with exact 32-bit sums), csrc/linear_int8.cu (one and two rows).  The
reference has no 8-bit path.
"""
from typing import NamedTuple

import torch as th

from . import _lib
from .rwkv7_linear import ACTS, F32_BIAS, F32_OUT, rows_of

MAX_K = (1 << 17) - 1


class Int8(NamedTuple):
    """Rows in 8 bits: row m stands for q[m] * scale[m].  q [..., K] int8, its rows on 16-byte boundaries; scale [...] fp32."""
    q: th.Tensor
    scale: th.Tensor


def pitch8(n):
    """Bytes from row to row of a tensor in 8 bits: rows on 16-byte boundaries, as the products take them."""
    return (n + 15) // 16 * 16


def rows8(x):
    """Launcher: q [..., pitch8(K)], scale [...]."""
    K = x.shape[-1]
    M = x.numel() // K
    q = th.empty(*x.shape[:-1], pitch8(K), dtype=th.int8, device=x.device)
    scale = th.empty(x.shape[:-1], dtype=th.float32, device=x.device)
    x, ldx = rows_of(x)
    with _lib.on_device(x):
        rc = _lib.lib().wkv7_quantize(x.data_ptr(), q.data_ptr(), scale.data_ptr(), M, K, ldx, q.shape[-1], int(x.dtype == th.float32), _lib.stream_of(x))
    _lib.check(rc, 'wkv7_quantize')
    return q, scale


def operand8(t):
    """(tensor, row pitch) of an operand in 8 bits; a copy where its rows are not on 16-byte boundaries."""
    if t.numel() == 0:
        return t, pitch8(t.shape[-1])
    t, ld = rows_of(t)
    if ld % 16 or t.data_ptr() % 16:
        n, to = t.shape[-1], th.empty(*t.shape[:-1], pitch8(t.shape[-1]), dtype=th.int8, device=t.device)
        to[..., :n] = t
        return to[..., :n], to.shape[-1]
    return t, ld


def fw_int8(xq, xs, wq, ws, bias, residual, act, out_f32):
    """Launcher: y [..., N]."""
    N, K = wq.shape
    M = xq.numel() // K
    y = th.empty(*xq.shape[:-1], N, dtype=th.float32 if out_f32 else th.bfloat16, device=xq.device)
    (xq, ldx), (wq, ldw) = operand8(xq), operand8(wq)
    r, ldr = (None, N) if residual is None else rows_of(residual)
    xs, ws, b = xs.contiguous(), ws.contiguous(), None if bias is None else bias.contiguous()
    flags = (F32_OUT if out_f32 else 0) | (F32_BIAS if b is not None and b.dtype == th.float32 else 0)
    with _lib.on_device(xq, xs, wq, ws, b, r):
        work = th.empty(_lib.lib().wkv7_linear_int8_workspace_bytes(M, N, K), dtype=th.uint8, device=y.device)
        rc = _lib.lib().wkv7_linear_int8(xq.data_ptr(), xs.data_ptr(), wq.data_ptr(), ws.data_ptr(), _lib.ptr(b), _lib.ptr(r), y.data_ptr(), M, N, K, ldx, ldw, ldr, N, act,
                                         flags, work.data_ptr() or None, _lib.stream_of(y))
    _lib.check(rc, 'wkv7_linear_int8')
    return y


_rows_op = _lib.opaque_op('quantize', rows8, lambda x: (x.new_empty((*x.shape[:-1], pitch8(x.shape[-1])), dtype=th.int8), x.new_empty(x.shape[:-1], dtype=th.float32)),
                          '(Tensor x) -> (Tensor, Tensor)')
_fw_op = _lib.opaque_op('linear_int8', fw_int8,
                        lambda xq, xs, wq, ws, bias, residual, act, out_f32: xs.new_empty((*xq.shape[:-1], wq.shape[0]), dtype=th.float32 if out_f32 else th.bfloat16),
                        '(Tensor xq, Tensor xs, Tensor wq, Tensor ws, Tensor? bias, Tensor? residual, int act, bool out_f32) -> Tensor')


def quantize(x):
    """Rows of x [..., K] in 8 bits: Int8(q, scale) with scale = max |row| / 127 and q = row / scale, rounded to the nearest, ties to even:
    exactly for bf16 rows, while an element of an fp32 row may be one off where row / scale is within a few of fp32's roundings of a half.

    x bf16 or fp32, K up to 2^30.  A row without a magnitude above 2^-100 becomes zeros with scale 0; one that holds a NaN or an infinity becomes zeros with a NaN for
    its scale, so that its products are NaN.  q's rows lie on 16-byte boundaries (K rounded up to 16 apart).  No autograd: the results are constants for a
    backward; a forward-mode tangent is refused."""
    if not th.compiler.is_compiling():
        out = _lib.ext().quantize(x)
        if out is not None:
            return Int8(*out)
    if x.dtype not in (th.bfloat16, th.float32):
        raise TypeError(f'quantize takes bfloat16 or float32, not {x.dtype}')
    if x.dim() < 1 or not 0 < x.shape[-1] <= 1 << 30:
        raise ValueError(f'quantize takes x [..., K] with K from 1 to 2^30, got {list(x.shape)}')
    _lib.refuse_tangents('quantize', x)
    _lib.require_cuda(x)
    q, scale = _lib.call(_rows_op, rows8, x.detach())
    return Int8(q[..., :x.shape[-1]], scale)


def _check(x, w, bias, residual, act, out_dtype):
    if act not in ACTS:
        raise ValueError(f'linear_int8: act must be one of {sorted(a for a in ACTS if a)} or None, got {act!r}')
    if out_dtype not in (None, th.bfloat16, th.float32):
        raise TypeError(f'linear_int8 gives bfloat16 or float32, not {out_dtype}')
    for name, pair in (('x', x), ('w', w)):
        if not isinstance(pair, tuple) or len(pair) != 2:
            raise TypeError(f'linear_int8: {name} is a pair (q, scale), as quantize gives it, got {type(pair).__name__}')
        q, scale = pair
        if q.dtype != th.int8 or scale.dtype != th.float32:
            raise TypeError(f'linear_int8: {name} is int8 with float32 scales, got {q.dtype} and {scale.dtype}')
        if q.dim() < 1 or scale.shape != q.shape[:-1]:
            raise ValueError(f'linear_int8: {name} has a scale a row, got {list(q.shape)} and {list(scale.shape)}')
    (xq, xs), (wq, ws) = x, w
    if wq.dim() != 2 or wq.shape[1] != xq.shape[-1]:
        raise ValueError(f'linear_int8: x [..., K] and w [N, K], got {list(xq.shape)} and {list(wq.shape)}')
    N, K = wq.shape
    if N == 0 or not 0 < K <= MAX_K:
        raise ValueError(f'linear_int8 needs N > 0 and K from 1 to {MAX_K}, whose sums fit 32 bits, got w {[N, K]}')
    if bias is not None and (list(bias.shape) != [N] or bias.dtype not in (th.bfloat16, th.float32)):
        raise ValueError(f'linear_int8: bias [{N}] bfloat16 or float32, got {list(bias.shape)} {bias.dtype}')
    out = out_dtype or th.bfloat16
    if residual is not None and (list(residual.shape) != [*xq.shape[:-1], N] or residual.dtype != out):
        raise ValueError(f'linear_int8: residual {[*xq.shape[:-1], N]} of the output\'s type {out}, got {list(residual.shape)} {residual.dtype}')
    if th.is_grad_enabled() and any(t is not None and t.requires_grad for t in (xs, ws, bias, residual)):
        raise RuntimeError('linear_int8 has no backward: call it under torch.no_grad()')
    _lib.refuse_tangents('linear_int8', xs, ws, bias, residual)


def linear_int8(x, w, bias=None, *, act=None, residual=None, out_dtype=None):
    """y = act((xq @ wq^T) xs ws + bias) + residual: x = (xq [..., K] int8, xs [...] fp32), w = (wq [N, K] int8, ws [N] fp32), as quantize and rms_norm give them.

    bias [N] bf16 or fp32, act and residual as linear's; y bf16, or fp32 with out_dtype=torch.float32.  K from 1 to 131071, any N.  The sum is exact (32-bit integers); behind it
    ws, xs, the bias, the activation and the residual are applied in fp32, in this order, and the result is rounded once.  What must stay within fp32's range is sum ws, not sum xs.  Rows may lie in a wider tensor, on 16-byte boundaries; other
    layouts are copied.  No backward."""
    if not th.compiler.is_compiling():
        if act in ACTS and out_dtype in (None, th.bfloat16, th.float32) and isinstance(x, tuple) and isinstance(w, tuple) and len(x) == len(w) == 2:
            out = _lib.ext().linear_int8(*x, *w, bias, residual, ACTS[act], out_dtype == th.float32)
            if out is not None:
                return out
    _check(x, w, bias, residual, act, out_dtype)  # (while torch.compile traces, too: the launchers take what they are given)
    (xq, xs), (wq, ws) = x, w
    _lib.require_cuda(xq, xs, wq, ws, bias, residual)
    plain = (t if t is None else t.detach() for t in (xq, xs, wq, ws, bias, residual))
    return _lib.call(_fw_op, fw_int8, *plain, ACTS[act], out_dtype == th.float32)
