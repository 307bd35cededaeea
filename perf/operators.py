"""Operators that stand next to the time mixer in a training or generating program: dense products with their epilogue, beam
search's selection, and the reordering of recurrent states that follows it.

  linear    y = act(x w^T + bias) + residual.  `train`: with the gradients of everything that goes in
  beam      beam_select: the best continuations of each sequence's beams over the vocabulary
  reorder   reorder_states: the beams' recurrent states follow their parents

With `own` false the operators are computed in elementary torch operations, in fp32 (selection: fp64, since an order hangs on the last
bits), otherwise by this package.
"""
import math
import os
import sys

import torch as th

own = False

_PKG = os.path.join(os.getcwd(), 'wind-rwkv7_b200')
DTYPES = {'bf16': th.bfloat16, 'f32': th.float32}


def _package():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import wind_rwkv.rwkv7 as pkg
    return pkg


def listed():
    return [
        # generation, one sequence of the 1.5B shape: first half of the channel mixer on one token, once per layer and token
        dict(name='mix_token', op='linear', M=1, K=2048, N=8192, act='relu2', bias=False, residual=False, out='bf16', train=False),
        # batched generation: second half, with the residual stream, on 24 sequences
        dict(name='mix_out_tokens', op='linear', M=24, K=8192, N=2048, act='none', bias=False, residual=True, out='bf16', train=False),
        # logits of two sequences with eight beams, over a vocabulary of odd size
        dict(name='head_beams', op='linear', M=16, K=2048, N=50001, act='none', bias=False, residual=False, out='f32', train=False),
        # a prompt of odd length through the channel mixer of the 2.9B shape
        dict(name='mix_prompt', op='linear', M=1283, K=2560, N=10240, act='relu2', bias=False, residual=False, out='bf16', train=False),
        # a small head with everything on it, odd sizes
        dict(name='small_train', op='linear', M=333, K=200, N=77, act='gelu', bias=True, residual=True, out='bf16', train=True),
        # training, both halves of the channel mixer at the 1.5B shape
        dict(name='mix_train', op='linear', M=8192, K=2048, N=8192, act='relu2', bias=False, residual=False, out='bf16', train=True),
        dict(name='mix_out_train', op='linear', M=8192, K=8192, N=2048, act='none', bias=True, residual=True, out='bf16', train=True),
        # one sequence with four beams
        dict(name='beam_one', op='beam', B=1, W=4, k=4, V=65536, dtype='bf16', ends=False),
        # a batch with ended beams, fp32 logits, odd vocabulary
        dict(name='beam_batch', op='beam', B=16, W=6, k=6, V=50001, dtype='f32', ends=True),
        # batched service with wide beams
        dict(name='beam_wide', op='beam', B=64, W=16, k=16, V=65536, dtype='bf16', ends=True),
        # states of one sequence's four beams, 12 layers of 12 heads (a WKV state and two token-shift rows a layer)
        dict(name='reorder_one', op='reorder', B=1, W=4, k=4, H=12, layers=12, inplace=True),
        # 16 sequences with eight beams, 12 layers at the 1.5B shape
        dict(name='reorder_batch', op='reorder', B=16, W=8, k=8, H=32, layers=12, inplace=True),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(['linear', 'linear', 'linear', 'beam', 'beam', 'reorder'])
    if op == 'linear':
        train = rng.random() < 0.5
        act = rng.choice(['none', 'none', 'relu2', 'relu2', 'relu', 'tanh', 'sigmoid', 'silu', 'gelu'])
        K, N = 8 * _log_int(rng, 1, 1024), _log_int(rng, 1, 50001 if not train else 10240)
        most = 8192 * 2048 * 8192  # M N K of the largest training case
        M = _log_int(rng, 1, max(1, min(65536 if train else 16384, most // (N * K), (1 << 28) // max(N, K))))
        return dict(op=op, M=M, K=K, N=N, act=act, bias=rng.random() < 0.5, residual=rng.random() < 0.5,
                    out='f32' if act == 'none' and rng.random() < 0.3 else 'bf16', train=train)
    if op == 'beam':
        W = _log_int(rng, 1, 32)
        dtype = rng.choice(['bf16', 'bf16', 'f32'])
        V = _log_int(rng, 1000, 131072)
        B = _log_int(rng, 1, max(1, min(64, (64 * 16 * 65536 // (2 if dtype == 'f32' else 1)) // (W * V))))
        return dict(op=op, B=B, W=W, k=rng.choice([W, W, min(64, 2 * W), _log_int(rng, 1, 32)]), V=V, dtype=dtype, ends=rng.random() < 0.5)
    W, H = _log_int(rng, 1, 32), rng.choice([8, 12, 16, 32, 40])
    inplace = rng.random() < 0.6
    B = _log_int(rng, 1, max(1, min(32, 128 // W)))
    layers = _log_int(rng, 1, max(1, min(24, 12 * 32 * 128 // (B * W * H))))
    return dict(op='reorder', B=B, W=W, k=W if inplace else rng.choice([W, max(1, W // 2), W]), H=H, layers=layers, inplace=inplace)


# ---- inputs -------------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = th.Generator(device='cuda')
    gen.manual_seed(seed * 1000003 + 17)

    def rn(*shape, std=1.0, dtype=th.float32):
        return (th.randn(*shape, generator=gen, device='cuda') * std).to(dtype)

    st = dict(case=case)
    if case['op'] == 'linear':
        M, K, N = case['M'], case['K'], case['N']
        st['x'] = rn(M, K, dtype=th.bfloat16)
        st['w'] = rn(N, K, std=K ** -0.5, dtype=th.bfloat16)
        st['bias'] = rn(N, std=0.5) if case['bias'] else None
        st['residual'] = rn(M, N, dtype=DTYPES[case['out']]) if case['residual'] else None
        if case['train']:
            st['dy'] = rn(M, N, dtype=DTYPES[case['out']])
            for n in ('x', 'w', 'bias', 'residual'):
                if st[n] is not None:
                    st[n].requires_grad_()
        return st
    if case['op'] == 'beam':
        B, W, V = case['B'], case['W'], case['V']
        # a vocabulary's logits: a broad floor, a few tokens well above it, tokens that are ruled out
        logits = rn(B, W, V, std=2.0)
        logits += 6.0 * th.rand(B, W, V, generator=gen, device='cuda').pow(40.0 * math.log10(V))
        logits[:, :, 1::97] = float('-inf')
        st['logits'] = logits.to(DTYPES[case['dtype']])
        st['scores'] = -(th.rand(B, W, generator=gen, device='cuda') * 6.0 + 10.0)
        st['finished'] = th.rand(B, W, generator=gen, device='cuda') < 0.25 if case['ends'] else None
        st['eos'] = 2 if case['ends'] else None
        return st
    B, W, k, H = case['B'], case['W'], case['k'], case['H']
    st['states'] = []
    for _ in range(case['layers']):
        st['states'] += [rn(B * W, H, 64, 64), rn(B * W, H * 64, dtype=th.bfloat16), rn(B * W, H * 64, dtype=th.bfloat16)]
    # beams that do well have several children, many go on in their place
    stay = th.arange(k, device='cuda').remainder(W).expand(B, k)
    jump = (th.rand(B, k, generator=gen, device='cuda') ** 2 * W).long().clamp_(max=W - 1)
    st['parents'] = th.where(th.rand(B, k, generator=gen, device='cuda') < 0.3, stay, jump)
    return st


# ---- plain forms --------------------------------------------------------------------------------------
_GELU = math.sqrt(2 / math.pi)


def _act(z, act):
    """act(z) and its derivative."""
    if act == 'none':
        return z, th.ones_like(z)
    if act == 'relu':
        return z.clamp(min=0), (z > 0).to(z.dtype)
    if act == 'relu2':
        p = z.clamp(min=0)
        return p * p, 2 * p
    if act == 'tanh':
        t = (1 - th.exp(-2 * z.abs())) / (1 + th.exp(-2 * z.abs())) * th.sign(z)
        return t, 1 - t * t
    if act == 'sigmoid':
        s = 1 / (1 + th.exp(-z))
        return s, s * (1 - s)
    if act == 'silu':
        s = 1 / (1 + th.exp(-z))
        return z * s, s * (1 + z * (1 - s))
    u = 2 * _GELU * (z + 0.044715 * z * z * z)
    s = 1 / (1 + th.exp(-u))
    return z * s, s + z * s * (1 - s) * 2 * _GELU * (1 + 3 * 0.044715 * z * z)


def _linear_plain(st):
    case = st['case']
    x, w = st['x'].detach().float(), st['w'].detach().float()
    z = x @ w.T
    if st['bias'] is not None:
        z = z + st['bias'].detach().float()
    a, d = _act(z, case['act'])
    y = a
    if st['residual'] is not None:
        y = a + st['residual'].detach().float()
    out = [y.to(DTYPES[case['out']])]
    if case['train']:
        dz = st['dy'].float() * d
        out += [(dz @ w).to(th.bfloat16), (dz.T @ x).to(th.bfloat16)]
        if st['bias'] is not None:
            out.append(dz.sum(0))
        if st['residual'] is not None:
            out.append(st['dy'].clone())
    return out


def _beam_plain(st):
    case = st['case']
    B, W, V, k = case['B'], case['W'], case['V'], case['k']
    x = st['logits'].double()
    m = x.amax(-1, keepdim=True)
    lp = (x - m) - th.exp(x - m).sum(-1, keepdim=True).log()
    del x
    if st['finished'] is not None:
        lp.masked_fill_(st['finished'][:, :, None], float('-inf'))
        lp[:, :, st['eos']] = th.where(st['finished'], th.zeros_like(lp[:, :, 0]), lp[:, :, st['eos']])
    lp += st['scores'].double()[:, :, None]
    flat = lp.view(B, W * V)
    at = th.arange(W * V, device=flat.device)
    # the best that is left, the lowest index among equals, k times
    taken = th.zeros_like(flat, dtype=th.bool)
    scores, index = [], []
    for _ in range(k):
        best = flat.masked_fill(taken, float('-inf')).amax(1, keepdim=True)
        i = th.where((flat == best) & ~taken, at, W * V).amin(1, keepdim=True)
        taken.scatter_(1, i, True)
        scores.append(best)
        index.append(i)
    index, scores = th.cat(index, 1), th.cat(scores, 1).float()
    parents, tokens = index // V, index % V
    if st['finished'] is None:
        return [scores, parents, tokens]
    return [scores, parents, tokens, st['finished'].gather(1, parents) | (tokens == st['eos'])]


def _rows(st):
    case = st['case']
    return (th.arange(case['B'], device='cuda')[:, None] * case['W'] + st['parents']).view(-1)


def _reorder_plain(st):
    rows = _rows(st)
    if not st['case']['inplace']:
        return [t[rows] for t in st['states']]
    for t in st['states']:
        t.copy_(t[rows])
    return st['states']


def run(st):
    case = st['case']
    if not own:
        return {'linear': _linear_plain, 'beam': _beam_plain, 'reorder': _reorder_plain}[case['op']](st)
    pkg = _package()
    if case['op'] == 'linear':
        y = pkg.linear(st['x'], st['w'], st['bias'], act=None if case['act'] == 'none' else case['act'], residual=st['residual'],
                       out_dtype=DTYPES[case['out']])
        if not case['train']:
            return [y]
        return [y.detach(), *th.autograd.grad(y, [st[n] for n in ('x', 'w', 'bias', 'residual') if st[n] is not None], st['dy'])]
    if case['op'] == 'beam':
        return list(pkg.beam_select(st['logits'], st['scores'], case['k'], finished=st['finished'], eos=st['eos']))
    return list(pkg.reorder_states(st['states'], st['parents'], inplace=case['inplace']))


# ---- what the operators cannot do without -----------------------------------------------------------------
def work(case):
    if case['op'] == 'linear':
        M, K, N, o = case['M'], case['K'], case['N'], 2 if case['out'] == 'bf16' else 4
        b = 2 * (M * K + N * K) + o * M * N * (2 if case['residual'] else 1) + (4 * N if case['bias'] else 0)
        if not case['train']:
            return dict(bytes=b, flops=2 * M * N * K)
        # the gradient of y comes in; those of x, w, bias and residual go out
        b += o * M * N + 2 * (M * K + N * K) + (4 * N if case['bias'] else 0) + (o * M * N if case['residual'] else 0)
        return dict(bytes=b, flops=6 * M * N * K)
    if case['op'] == 'beam':
        rows = case['B'] * case['W']
        size = 2 if case['dtype'] == 'bf16' else 4
        return dict(bytes=rows * case['V'] * size + 4 * rows + 20 * case['B'] * case['k'], flops=4 * rows * case['V'])
    row = case['layers'] * case['H'] * (64 * 64 * 4 + 2 * 64 * 2)
    return dict(bytes=2 * case['B'] * case['k'] * row, flops=0)


# ---- the definitions in 64 bits -------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    if case['op'] == 'linear':
        ins = [st[n] for n in ('x', 'w', 'bias', 'residual')]
        leaves = [None if t is None else t.detach().double().requires_grad_(case['train']) for t in ins]
        x, w, bias, residual = leaves
        y = th.einsum('mk,nk->mn', x, w)
        if bias is not None:
            y = y + bias
        y = {'none': lambda t: t, 'relu': th.relu, 'relu2': lambda t: th.relu(t).square(), 'tanh': th.tanh, 'sigmoid': th.sigmoid,
             'silu': th.nn.functional.silu, 'gelu': lambda t: th.nn.functional.gelu(t, approximate='tanh')}[case['act']](y)
        if residual is not None:
            y = y + residual
        if not case['train']:
            return [y]
        return [y.detach(), *th.autograd.grad(y, [t for t in leaves if t is not None], st['dy'].double())]
    if case['op'] == 'beam':
        B, W, V, k = case['B'], case['W'], case['V'], case['k']
        scores, parents, tokens = [], [], []
        for b in range(B):
            lp = th.log_softmax(st['logits'][b].double(), -1)
            if st['finished'] is not None:
                only = th.full((V,), float('-inf'), dtype=th.float64, device='cuda')
                only[st['eos']] = 0.0
                lp = th.where(st['finished'][b][:, None], only, lp)
            s, i = (st['scores'][b].double()[:, None] + lp).flatten().sort(descending=True, stable=True)
            scores.append(s[:k])
            parents.append(i[:k] // V)
            tokens.append(i[:k] % V)
        out = [th.stack(scores), th.stack(parents), th.stack(tokens)]
        if st['finished'] is not None:
            out.append((out[2] == st['eos']) | th.stack([f[p] for f, p in zip(st['finished'], out[1])]))
        return out
    kids = st['parents'].tolist()
    return [th.stack([t[b * case['W'] + p] for b, ps in enumerate(kids) for p in ps]) for t in st['states']]
