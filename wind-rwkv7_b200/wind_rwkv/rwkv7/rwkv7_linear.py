"""Dense products with their epilogue: `linear(x, w, bias, act=, residual=)` = act(x @ w^T + bias) + residual.

What a model computes around the time mixer: both halves of the channel mixer (relu^2 in the first, the residual stream added in the
second) and the head.  The reference leaves them to torch (`x @ W.bfloat16().mT`, time_mixer.py:120-131, 167).  Here the product and its
epilogue are one tcgen05 kernel (csrc/linear.cu), and so are the two products of the backward; a few rows (decoding) take a form
that streams the weight with all SMs.  `proj` is the narrow product of the LoRAs, tanh on a range of columns.
"""
import torch as th

from . import _lib

ACTS = {None: 0, 'relu': 1, 'relu2': 2, 'tanh': 3, 'sigmoid': 4, 'silu': 5, 'gelu': 6}
F32_OUT, F32_BIAS, FROM_Y, F32_Z = 1, 2, 4, 8


def rows_of(t):
    """(tensor, row pitch) of t [..., n] as rows of n adjacent elements one pitch apart; a copy where it does not lie so."""
    n = t.shape[-1]
    if t.numel() == 0:
        return t, n
    pitch, rows, lies = None, 1, n == 1 or t.stride(-1) == 1
    for size, stride in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        if size == 1:
            continue
        if pitch is None:
            pitch = stride
        lies = lies and stride == pitch * rows and pitch >= n
        rows *= size
    return (t, n if pitch is None else pitch) if lies else (t.contiguous(), n)


def operand_of(t):
    """The same for an operand of the products: rows on 16-byte boundaries."""
    t, ld = rows_of(t)
    if ld % 8 or t.data_ptr() % 16:
        t, ld = t.clone(memory_format=th.contiguous_format), t.shape[-1]
    return t, ld


def saves(act, out_f32, residual, bias_f32):
    """What the backward needs of the forward: None, 'y', 'z' or 'z32'.  relu and relu^2 have their derivative in their value (2 sqrt(y), a bf16 y's
    rounding halved by the root); of the others it is formed from the argument, kept in bf16: no worse than the rounding of dz for the products.  With
    a bias in fp32, whose gradient goes out in fp32, what is summed for it is formed from an argument in fp32."""
    if act == 0:
        return None
    if bias_f32 and act != ACTS['relu']:
        return 'z32'
    return 'y' if act in (ACTS['relu'], ACTS['relu2']) and not out_f32 and not residual else 'z'


def fw_linear(x, w, bias, residual, act, out_f32, save):
    """Launcher: y [..., N], z [rows, N rounded up to 8] (empty unless save is 'z' or 'z32')."""
    save_z = save in ('z', 'z32')
    K, N = x.shape[-1], w.shape[0]
    M = x.numel() // K
    n8 = (N + 7) // 8 * 8
    y = th.empty(*x.shape[:-1], N, dtype=th.float32 if out_f32 else th.bfloat16, device=x.device)
    z = th.empty(M if save_z else 0, n8, dtype=th.float32 if save == 'z32' else th.bfloat16, device=x.device)
    x, ldx = operand_of(x)
    w, ldw = operand_of(w)
    r, ldr = (None, N) if residual is None else rows_of(residual)
    b = None if bias is None else bias.contiguous()
    flags = (F32_OUT if out_f32 else 0) | (F32_BIAS if b is not None and b.dtype == th.float32 else 0) | (F32_Z if save == 'z32' else 0)
    with _lib.on_device(x, w, b, r):
        ws = th.empty(_lib.lib().wkv7_linear_fwd_workspace_bytes(M, N, K), dtype=th.uint8, device=x.device)
        rc = _lib.lib().wkv7_linear_fwd(x.data_ptr(), w.data_ptr(), _lib.ptr(b), _lib.ptr(r), y.data_ptr(), z.data_ptr() if save_z else None,
                                        M, N, K, ldx, ldw, ldr, N, n8, act, flags, ws.data_ptr() or None, _lib.stream_of(x))
    _lib.check(rc, 'wkv7_linear_fwd')
    return y, z


def bw_linear(x, w, saved, dy, act, out_f32, from_y, want_dx, want_dw, want_db):
    """Launcher: dx like x, dw like w, dbias [N] fp32, each empty where it is not wanted."""
    K, N = x.shape[-1], w.shape[0]
    M = x.numel() // K
    dev = x.device
    dx = th.empty(x.shape if want_dx else (0,), dtype=th.bfloat16, device=dev)
    dw = th.empty(w.shape if want_dw else (0,), dtype=th.bfloat16, device=dev)
    db = th.empty(N if want_db else 0, dtype=th.float32, device=dev)
    x, ldx = operand_of(x)
    w, ldw = operand_of(w)
    dy, lddy = rows_of(dy)
    saved, lds = rows_of(saved) if act else (None, N)
    flags = (F32_OUT if out_f32 else 0) | (FROM_Y if from_y else 0) | (F32_Z if act and saved.dtype == th.float32 else 0)
    with _lib.on_device(x, w, dy, saved):
        ws = th.empty(_lib.lib().wkv7_linear_bwd_workspace_bytes(M, N, K), dtype=th.uint8, device=dev)
        rc = _lib.lib().wkv7_linear_bwd(x.data_ptr(), w.data_ptr(), _lib.ptr(saved), dy.data_ptr(), dx.data_ptr() if want_dx else None,
                                        dw.data_ptr() if want_dw else None, db.data_ptr() if want_db else None, M, N, K, ldx, ldw, lds, lddy, act, flags,
                                        ws.data_ptr(), _lib.stream_of(x))
    _lib.check(rc, 'wkv7_linear_bwd')
    return dx, dw, db


def _fake_fw(x, w, bias, residual, act, out_f32, save):
    N = w.shape[0]
    rows = x.numel() // x.shape[-1]
    return (x.new_empty((*x.shape[:-1], N), dtype=th.float32 if out_f32 else th.bfloat16),
            x.new_empty((rows if save in ('z', 'z32') else 0, (N + 7) // 8 * 8), dtype=th.float32 if save == 'z32' else th.bfloat16))


def _fake_bw(x, w, saved, dy, act, out_f32, from_y, want_dx, want_dw, want_db):
    return (x.new_empty(x.shape if want_dx else (0,)), w.new_empty(w.shape if want_dw else (0,)),
            x.new_empty((w.shape[0] if want_db else 0,), dtype=th.float32))


_fw_op = _lib.opaque_op('linear_fwd', fw_linear, _fake_fw,
                        '(Tensor x, Tensor w, Tensor? bias, Tensor? residual, int act, bool out_f32, str save) -> (Tensor, Tensor)')
_bw_op = _lib.opaque_op('linear_bwd', bw_linear, _fake_bw,
                        '(Tensor x, Tensor w, Tensor saved, Tensor dy, int act, bool out_f32, bool from_y, bool want_dx, bool want_dw, bool want_db) -> '
                        '(Tensor, Tensor, Tensor)')


class Linear(th.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, bias, residual, act, out_f32):
        grad = any(ctx.needs_input_grad[:3])
        save = saves(act, out_f32, residual is not None, bias is not None and bias.dtype == th.float32) if grad else None
        y, z = _lib.call(_fw_op, fw_linear, x, w, bias, residual, act, out_f32, save or '')
        if grad:
            ctx.save_for_backward(x, w, y if save == 'y' else z)
        ctx.how = (act, out_f32, save == 'y', None if bias is None else bias.dtype)
        return y

    @staticmethod
    def backward(ctx, dy):
        act, out_f32, from_y, bias_dtype = ctx.how
        want = ctx.needs_input_grad
        dx = dw = db = None
        if any(want[:3]):
            x, w, saved = ctx.saved_tensors
            dx, dw, db = _lib.call(_bw_op, bw_linear, x, w, saved, dy.to(th.float32 if out_f32 else th.bfloat16), act, out_f32, from_y, want[0], want[1], want[2])
            dx, dw, db = dx if want[0] else None, dw if want[1] else None, db.to(bias_dtype) if want[2] else None
        return dx, dw, db, dy if want[3] else None, None, None


def _check(x, w, bias, residual, act, out_dtype):
    if act not in ACTS:
        raise ValueError(f'linear: act must be one of {sorted(a for a in ACTS if a)} or None, got {act!r}')
    if out_dtype not in (None, th.bfloat16, th.float32):
        raise TypeError(f'linear gives bfloat16 or float32, not {out_dtype}')
    if x.dtype != th.bfloat16 or w.dtype != th.bfloat16:
        raise TypeError(f'linear takes bfloat16 x and w, got {x.dtype} and {w.dtype}')
    if x.dim() < 1 or w.dim() != 2 or w.shape[1] != x.shape[-1]:
        raise ValueError(f'linear: x [..., K] and w [N, K], got {list(x.shape)} and {list(w.shape)}')
    N, K = w.shape
    if N == 0 or K == 0 or K % 8:
        raise ValueError(f'linear needs N > 0 and K a positive multiple of 8, got w {[N, K]}')
    if bias is not None and (list(bias.shape) != [N] or bias.dtype not in (th.bfloat16, th.float32)):
        raise ValueError(f'linear: bias [{N}] bfloat16 or float32, got {list(bias.shape)} {bias.dtype}')
    out = out_dtype or th.bfloat16
    if residual is not None and (list(residual.shape) != [*x.shape[:-1], N] or residual.dtype != out):
        raise ValueError(f'linear: residual {[*x.shape[:-1], N]} of the output\'s type {out}, got {list(residual.shape)} {residual.dtype}')


def linear(x, w, bias=None, *, act=None, residual=None, out_dtype=None):
    """y = act(x @ w^T + bias) + residual: x [..., K], w [N, K] bf16, K a multiple of 8, any N; bias [N] bf16 or fp32; residual [..., N] of y's type.

    act: None, 'relu', 'relu2' (relu(z)^2, the channel mixer's), 'tanh', 'sigmoid', 'silu', 'gelu' (its tanh form).  y is bf16, or fp32 with
    out_dtype=torch.float32 (logits).  Sums are formed in the tensor cores' fp32 accumulators, whose additions cut, and rounded once: results in fp32 are off by some 1e-9 K
    (as the library's are; less for few rows).  Backward for x, w, bias and residual; the gradient that enters the products, dy act'(z), is rounded to bf16, and
    z is kept in bf16 (in fp32 beside an fp32 bias; of relu and relu2 y is kept instead).  Rows may lie in a wider tensor; other layouts are copied.

    What it saves is the passes over y that an activation, bias or residual would take, and in few rows the weight's time.  A product alone of a few hundred to a few
    thousand rows is quicker by x @ w.mT: 512 x 2048 x 2048 11 against 6 us, 2048^3 15 against 13.5, 1283 x 2560 x 10240 52 against 48; from 8192 rows on they are equal."""
    if not th.compiler.is_compiling():
        if act in ACTS and out_dtype in (None, th.bfloat16, th.float32):
            out = _lib.ext().linear(x, w, bias, residual, ACTS[act], out_dtype == th.float32)
            if out is not None:
                return out
    _check(x, w, bias, residual, act, out_dtype)  # (while torch.compile traces, too: the launchers take what they are given)
    _lib.require_cuda(x, w, bias, residual)
    return Linear.apply(x, w, bias, residual, ACTS[act], out_dtype == th.float32)
