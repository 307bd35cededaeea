"""Operators between the mixers of a model: the residual stream's norm and dropout in training, products in 8 bits in serving.

  int8     rows of activations to 8 bits, by themselves (front 'quantize') or as the norm of the residual stream (front 'norm'), and the product with
           weights in 8 bits behind them: linear_int8(quantize(x), w8), linear_int8(rms_norm(..., out_dtype=int8), w8)
  norm     y, h = rms_norm(x, weight, residual=...): h = residual + dropout(x), y = its root-mean-square norm.  `train`: with the gradients of all that goes in
  dropout  residual + dropout(x) from a counter-based generator.  `train`: with the gradients

With `own` false the operators are computed in elementary torch operations in fp32, otherwise by this package.
"""
import math
import os
import sys

import torch as th

own = False

_PKG = os.path.join(os.getcwd(), 'wind-rwkv7_b200')
DTYPES = {'bf16': th.bfloat16, 'f32': th.float32}
EPS = 1e-5
TINY = 2.0 ** -100  # rows without a larger magnitude are zeros in 8 bits


def _package():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import wind_rwkv.rwkv7 as pkg
    return pkg


def listed():
    return [
        # generation, one sequence of the 1.5B shape: the residual stream's norm and the first half of the channel mixer
        dict(name='norm_mix_token', op='int8', front='norm', M=1, K=2048, N=8192, act='relu2', bias=False, residual=False, out='bf16'),
        # batched generation: second half, with the residual stream, on 24 sequences
        dict(name='mix_out_tokens', op='int8', front='quantize', M=24, K=8192, N=2048, act='none', bias=False, residual=True, out='bf16'),
        # logits of 16 sequences over a vocabulary of odd size
        dict(name='head_tokens', op='int8', front='quantize', M=16, K=2048, N=50001, act='none', bias=False, residual=False, out='f32'),
        # a prompt of odd length: norm and first half at the 2.9B shape
        dict(name='norm_mix_prompt', op='int8', front='norm', M=1283, K=2560, N=10240, act='relu2', bias=False, residual=False, out='bf16'),
        # prompts of a batch, first half at the 1.5B shape
        dict(name='mix_prompts', op='int8', front='quantize', M=8192, K=2048, N=8192, act='relu2', bias=False, residual=False, out='bf16'),
        # everything on it, odd sizes
        dict(name='small_odd', op='int8', front='quantize', M=333, K=203, N=77, act='gelu', bias=True, residual=True, out='bf16'),
        # generation, one token's residual stream
        dict(name='norm_token', op='norm', M=1, D=2048, x='bf16', r='bf16', w='f32', p=0.0, train=False),
        # a small model of odd width in fp32
        dict(name='norm_odd', op='norm', M=1003, D=333, x='f32', r='f32', w='f32', p=0.2, train=True),
        # training at the 1.5B shape with the residual stream's dropout
        dict(name='norm_train', op='norm', M=8192, D=2048, x='bf16', r='bf16', w='bf16', p=0.1, train=True),
        # a wide model with the stream in fp32
        dict(name='norm_wide', op='norm', M=16384, D=4096, x='bf16', r='f32', w='f32', p=0.0, train=True),
        # a small layer's dropout
        dict(name='dropout_small', op='dropout', M=512, D=768, x='bf16', r='bf16', p=0.1, train=True),
        # a batch's embeddings and mixer outputs, without a stream to be added to
        dict(name='dropout_large', op='dropout', M=65536, D=1024, x='bf16', r='none', p=0.1, train=True),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(['int8', 'int8', 'norm', 'norm', 'dropout'])
    if op == 'int8':
        front = rng.choice(['quantize', 'norm'])
        K = rng.choice([_log_int(rng, 8, 8192), 16 * _log_int(rng, 1, 512)])
        N = _log_int(rng, 1, 50001)
        M = _log_int(rng, 1, max(1, min(16384, 8192 * 2048 * 8192 // (N * K), (1 << 27) // max(N, K))))
        act = rng.choice(['none', 'none', 'relu2', 'relu2', 'relu', 'tanh', 'sigmoid', 'silu', 'gelu'])
        return dict(op=op, front=front, M=M, K=K, N=N, act=act, bias=rng.random() < 0.5, residual=rng.random() < 0.5,
                    out='f32' if front == 'quantize' and act == 'none' and rng.random() < 0.3 else 'bf16')
    D = rng.choice([_log_int(rng, 16, 8192), 64 * _log_int(rng, 1, 128)])
    M = _log_int(rng, 1, (1 << 26) // D)
    r = rng.choice(['none', 'bf16', 'bf16', 'f32'])
    x = rng.choice(['bf16', 'bf16', 'f32'])
    p = rng.choice([0.05, 0.1, 0.2, 0.5])
    if x == 'f32' or r == 'f32':
        M = max(1, M // 2)
    if op == 'dropout':
        return dict(op=op, M=M, D=D, x=x, r=r, p=p, train=rng.random() < 0.7)
    train = rng.random() < 0.7
    p = p if train and r != 'none' and rng.random() < 0.6 else 0.0
    # a stream in bf16 whose sums hold more than it does is rounded, a few elements in a million another way in 64 bits than in 32: a gain in fp32, whose
    # gradient would show that, is for other streams
    w = 'bf16' if r == 'bf16' and (p or x == 'f32') else rng.choice(['f32', 'f32', 'bf16'])
    return dict(op=op, M=M, D=D, x=x, r=r, w=w, p=p, train=train)


# ---- inputs -------------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = th.Generator(device='cuda')
    gen.manual_seed(seed * 1000003 + 29)

    def rn(*shape, std=1.0, dtype=th.float32):
        return (th.randn(*shape, generator=gen, device='cuda') * std).to(dtype)

    st = dict(case=case, seed=seed * 7919 + (1 << 33) + 5)
    if case['op'] == 'int8':
        M, K, N = case['M'], case['K'], case['N']
        st['x'] = rn(M, K, dtype=th.bfloat16)
        if case['front'] == 'norm':
            st['stream'] = rn(M, K, std=2.0, dtype=th.bfloat16)
            st['gain'] = 1.0 + rn(K, std=0.2)
        # weights as they are kept for serving: 8 bits, a scale a channel, rows on 16-byte boundaries
        w = rn(N, K, std=K ** -0.5)
        st['ws'] = w.abs().amax(1).clamp_(min=1e-6) / 127.0
        rows = th.zeros(N, (K + 15) // 16 * 16, dtype=th.int8, device='cuda')
        rows[:, :K] = th.round(w / st['ws'][:, None]).to(th.int8)
        st['wq'] = rows[:, :K]
        del w
        st['bias'] = rn(N, std=0.5) if case['bias'] else None
        st['residual'] = rn(M, N, dtype=DTYPES[case['out']]) if case['residual'] else None
        return st
    M, D = case['M'], case['D']
    st['x'] = rn(M, D, dtype=DTYPES[case['x']])
    st['residual'] = rn(M, D, std=2.0, dtype=DTYPES[case['r']]) if case['r'] != 'none' else None
    if case['op'] == 'norm':
        st['weight'] = (1.0 + rn(D, std=0.2)).to(DTYPES[case['w']])
    if case['train']:
        h_type = DTYPES[case['r'] if case['r'] != 'none' else case['x']]
        if case['op'] == 'norm':
            st['dy'] = rn(M, D, dtype=DTYPES[case['x']])
            st['dh'] = rn(M, D, dtype=h_type) if case['r'] != 'none' else None
        else:
            st['dy'] = rn(M, D, dtype=h_type)
        for n in ('x', 'residual', 'weight'):
            if st.get(n) is not None:
                st[n].requires_grad_()
    return st


# ---- plain forms --------------------------------------------------------------------------------------
_GELU = math.sqrt(2 / math.pi)


def _act(z, act):
    if act == 'none':
        return z
    if act == 'relu':
        return z.clamp(min=0)
    if act == 'relu2':
        return z.clamp(min=0) * z.clamp(min=0)
    if act == 'tanh':
        return (1 - th.exp(-2 * z.abs())) / (1 + th.exp(-2 * z.abs())) * th.sign(z)
    if act == 'sigmoid':
        return 1 / (1 + th.exp(-z))
    if act == 'silu':
        return z / (1 + th.exp(-z))
    return z / (1 + th.exp(-2 * _GELU * (z + 0.044715 * z * z * z)))


def _keep(numel, p, seed):
    """1 / (1 - p) where an element is kept, else 0.  Words of Philox4x32-10 (Salmon et al. 2011): counter = index / 4, key = seed."""
    block = th.arange((numel + 3) // 4, device='cuda')
    low = 0xFFFFFFFF
    c0, c1, c2, c3 = block & low, block >> 32, th.zeros_like(block), th.zeros_like(block)
    k0, k1 = seed & low, seed >> 32
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # (modulo 2^64: both halves are right)
        c0, c1, c2, c3 = (b >> 32 & low) ^ c1 ^ k0, b & low, (a >> 32 & low) ^ c3 ^ k1, a & low
        k0, k1 = k0 + 0x9E3779B9 & low, k1 + 0xBB67AE85 & low
    words = th.stack([c0, c1, c2, c3], 1).view(-1)[:numel]
    return (words >= round(p * 2 ** 32)).float() * (1 / (1 - p))


def _to_int8(y):
    a = y.abs().amax(-1, keepdim=True)
    live = a > TINY
    return th.where(live, th.round(y * 127.0 / a), th.zeros_like(y)), th.where(live, a / 127.0, th.zeros_like(a))


def _int8_plain(st):
    case = st['case']
    if case['front'] == 'norm':
        h = (st['x'].float() + st['stream'].float()).to(th.bfloat16)
        f = h.float()
        q, s = _to_int8(f / th.sqrt((f * f).mean(-1, keepdim=True) + EPS) * st['gain'])
    else:
        h = None
        q, s = _to_int8(st['x'].float())
    z = (q @ st['wq'].float().T) * s * st['ws']
    if st['bias'] is not None:
        z = z + st['bias']
    y = _act(z, case['act'])
    if st['residual'] is not None:
        y = y + st['residual'].float()
    y = y.to(DTYPES[case['out']])
    return [y] if h is None else [y, h]


def _norm_plain(st):
    case = st['case']
    x, w = st['x'].detach(), st['weight'].detach().float()
    f = x.float()
    keep = _keep(x.numel(), case['p'], st['seed']).view_as(x) if case['p'] else None
    if keep is not None:
        f = f * keep
    h = None
    if st['residual'] is not None:
        r = st['residual'].detach()
        h = (r.float() + f).to(r.dtype)
        f = h.float()
    rms = 1 / th.sqrt((f * f).mean(-1, keepdim=True) + EPS)
    out = [(f * rms * w).to(x.dtype)]
    if h is not None:
        out.append(h)
    if case['train']:
        dy = st['dy'].float()
        g = dy * w
        dh = rms * (g - f * rms * rms * (g * f).mean(-1, keepdim=True))
        if h is not None:
            dh = dh + st['dh'].float()
        out.append((dh if keep is None else dh * keep).to(x.dtype))
        out.append((dy * f * rms).sum(0).to(st['weight'].dtype))
        if h is not None:
            out.append(dh.to(h.dtype))
    return out


def _dropout_plain(st):
    case = st['case']
    x = st['x'].detach()
    keep = _keep(x.numel(), case['p'], st['seed']).view_as(x)
    y = x.float() * keep
    out_type = x.dtype
    if st['residual'] is not None:
        r = st['residual'].detach()
        y, out_type = r.float() + y, r.dtype
    out = [y.to(out_type)]
    if case['train']:
        out.append((st['dy'].float() * keep).to(x.dtype))
        if st['residual'] is not None:
            out.append(st['dy'].clone())
    return out


def run(st):
    case = st['case']
    if not own:
        return {'int8': _int8_plain, 'norm': _norm_plain, 'dropout': _dropout_plain}[case['op']](st)
    pkg = _package()
    if case['op'] == 'int8':
        how = dict(act=None if case['act'] == 'none' else case['act'], residual=st['residual'], out_dtype=DTYPES[case['out']])
        if case['front'] == 'quantize':
            return [pkg.linear_int8(pkg.quantize(st['x']), (st['wq'], st['ws']), st['bias'], **how)]
        x8, h = pkg.rms_norm(st['x'], st['gain'], residual=st['stream'], eps=EPS, out_dtype=th.int8)
        return [pkg.linear_int8(x8, (st['wq'], st['ws']), st['bias'], **how), h]
    if case['op'] == 'norm':
        out = pkg.rms_norm(st['x'], st['weight'], residual=st['residual'], eps=EPS, p=case['p'], seed=st['seed'] if case['p'] else None)
        out = list(out) if st['residual'] is not None else [out]
        grads = [st['dy']] + ([st['dh']] if st['residual'] is not None else []) if case['train'] else []
        leaves = [st['x'], st['weight']]
    else:
        out = [pkg.dropout(st['x'], case['p'], st['seed'], residual=st['residual'])]
        grads = [st['dy']] if case['train'] else []
        leaves = [st['x']]
    if not case['train']:
        return out
    if st['residual'] is not None:
        leaves.append(st['residual'])
    return [t.detach() for t in out] + list(th.autograd.grad(out, leaves, grads))


# ---- what the operators cannot do without -----------------------------------------------------------------
def work(case):
    size = {'bf16': 2, 'f32': 4, 'none': 0}
    if case['op'] == 'int8':
        M, K, N, o = case['M'], case['K'], case['N'], size[case['out']]
        b = 2 * M * K + N * K + 4 * N + o * M * N * (2 if case['residual'] else 1) + (4 * N if case['bias'] else 0)
        if case['front'] == 'norm':
            b += 4 * M * K + 4 * K  # the stream goes in and out, and the gain
        return dict(bytes=b, flops=2 * M * N * K)
    n, x, r = case['M'] * case['D'], size[case['x']], size[case['r']]
    if case['op'] == 'dropout':
        b = x + r + (r or x)
        if case['train']:
            b += (r or x) + x
        return dict(bytes=n * b, flops=n * (4 if case['train'] else 2))
    b = x + r + x + r  # x and the stream in, y and the stream out
    if case['train']:
        # the gradients of both come in; those of x and of the stream go out, one and the same where nothing is dropped and the types are equal
        b += x + r + x + (r if case['p'] or x != r else 0)
    weight = size[case['w']] * case['D']
    return dict(bytes=n * b + weight * (2 if case['train'] else 1), flops=n * (16 if case['train'] else 4))


# ---- the definitions in 64 bits -------------------------------------------------------------------------------
def _mulhilo(x, m):
    """Both halves of 32 x 32-bit products from 16-bit parts, which stay within a signed 64-bit word."""
    lo, hi = x % 65536, x // 65536
    p0, p1, p2, p3 = lo * (m % 65536), lo * (m // 65536), hi * (m % 65536), hi * (m // 65536)
    mid = p1 + p2 + p0 // 65536
    return p3 + mid // 65536, (mid % 65536) * 65536 + p0 % 65536


def _kept(shape, p, seed):
    n = math.prod(shape)
    idx = th.arange(-(-n // 4), device='cuda')
    ctr = [idx % 2 ** 32, idx // 2 ** 32, idx * 0, idx * 0]
    for i in range(10):
        key = [(seed % 2 ** 32 + i * 0x9E3779B9) % 2 ** 32, (seed // 2 ** 32 + i * 0xBB67AE85) % 2 ** 32]
        (h0, l0), (h1, l1) = _mulhilo(ctr[0], 0xD2511F53), _mulhilo(ctr[2], 0xCD9E8D57)
        ctr = [th.bitwise_xor(th.bitwise_xor(h1, ctr[1]), key[0]), l1, th.bitwise_xor(th.bitwise_xor(h0, ctr[3]), key[1]), l0]
    return th.stack(ctr, -1).flatten()[:n].ge(round(p * 2.0 ** 32)).reshape(shape)


def _rows8(v):
    top = v.abs().max(-1, keepdim=True).values
    return th.where(top > TINY, (v * 127 / top).round(), 0.0), th.where(top > TINY, top / 127, 0.0)


def exact(case, seed):
    st = prepare(case, seed)
    if case['op'] == 'int8':
        v, tail = st['x'].double(), []
        if case['front'] == 'norm':
            v = v + st['stream'].double()
            tail = [v]
            v = v.bfloat16().double()  # (the stream as it is kept)
            v = v * th.rsqrt(v.square().mean(-1, keepdim=True) + EPS) * st['gain'].double()
        q, s = _rows8(v)
        y = th.einsum('mk,nk->mn', q, st['wq'].double()) * s * st['ws'].double()
        if st['bias'] is not None:
            y = y + st['bias'].double()
        y = {'none': lambda t: t, 'relu': th.relu, 'relu2': lambda t: th.relu(t).square(), 'tanh': th.tanh, 'sigmoid': th.sigmoid,
             'silu': th.nn.functional.silu, 'gelu': lambda t: th.nn.functional.gelu(t, approximate='tanh')}[case['act']](y)
        if st['residual'] is not None:
            y = y + st['residual'].double()
        return [y] + tail
    x = st['x'].detach().double()
    r = None if st['residual'] is None else st['residual'].detach()
    mask = _kept(x.shape, case['p'], st['seed']) if case['p'] else None
    drop = (lambda t: t) if mask is None else (lambda t: th.where(mask, t / (1 - case['p']), 0.0))
    h = drop(x) if r is None else r.double() + drop(x)
    if case['op'] == 'dropout':
        if not case['train']:
            return [h]
        dy = st['dy'].double()
        return [h, drop(dy)] + ([] if r is None else [dy])
    kept = (h if r is None else h.to(r.dtype).double()).requires_grad_(case['train'])  # (the stream as it is kept)
    w = st['weight'].detach().double().requires_grad_(case['train'])
    y = kept * th.rsqrt(kept.square().mean(-1, keepdim=True) + EPS) * w
    out = [y.detach()] + ([] if r is None else [h.detach()])
    if not case['train']:
        return out
    dh, dw = th.autograd.grad(y, [kept, w], st['dy'].double())
    if r is not None:
        dh = dh + st['dh'].double()
    return out + [drop(dh), dw] + ([] if r is None else [dh])
