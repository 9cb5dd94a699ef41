"""Operators beside the curvature of a training step, as measurable cases: layer norm with its gradients and Fisher blocks, draws
from filtered predictive distributions, and the global norm of gradients with clipping.

Keys of a case:
  op        'norm' (layer norm), 'sample' (one class per row of logits), 'clip' (norm of all gradients, clipped copies)
norm:
  rows, width; x, w      types of the rows (and of y, g) and of the weights;  y   type of the result
  train     False: y alone; True: y, then dx, dw, db from a gradient of y
  bias      False: no bias
  blocks    True: the backward pass gives the unit-wise Fisher blocks of weight and bias, too
sample:
  rows, classes, pad     row stride classes + pad;  x  type of the logits
  temperature, top_k, top_p, min_p     0: not used;  mixed: every row has parameters of its own (a batch of requests)
clip:
  model     'mlp' | 'resnet50' | 'decoder', with widths or d and layers;  x  'f32' | 'bf16' | 'mixed' (norms and biases f32)
  norm      'two' | 'max';  copies   False: the norm alone
"""
import math

import numpy as np
import torch

own = False

TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
EPS = 1e-5
MOST_LOGITS = 4096 * 50257
EXACT_LOGITS = 1 << 21


def listed():
    norm = dict(op='norm', x='f32', y='f32', w='f32', train=True, bias=True, blocks=False)
    sample = dict(op='sample', x='f32', pad=0, temperature=1.0, top_k=0, top_p=0.0, min_p=0.0, mixed=False)
    clip = dict(op='clip', x='f32', norm='two', copies=True)
    return [
        # four sequences that are decoded token by token: latency alone
        dict(norm, name='norm_decode', rows=4, width=768, x='bf16', y='bf16', train=False),
        # a layer of the decoder of GPT-2-small shape under bf16 autocast (its residual stream is fp32), with its Fisher blocks
        dict(norm, name='norm_decoder_blocks', rows=8 * 1024, width=768, blocks=True),
        # rows and columns that are no multiple of anything
        dict(norm, name='norm_ragged', rows=1000, width=1021, bias=False),
        # a wide model kept in bf16
        dict(norm, name='norm_wide_bf16', rows=16384, width=4096, x='bf16', y='bf16', w='bf16'),
        # a batch of requests that are answered: the usual filters, logits of the last token
        dict(sample, name='sample_decode', rows=8, classes=50257, x='bf16', temperature=0.8, top_k=50, top_p=0.95),
        # requests with parameters of their own, logits padded to whole blocks
        dict(sample, name='sample_requests', rows=256, classes=50257, x='bf16', pad=47, mixed=True),
        # sampled targets of an image classifier without its unlikely classes
        dict(sample, name='sample_classes', rows=1024, classes=1000, min_p=0.02),
        # sampled targets of a decoder's whole batch, from the nucleus of its distribution
        dict(sample, name='sample_decoder', rows=4096, classes=50257, top_p=0.9),
        # the MLP of the benchmark: six small tensors
        dict(clip, name='clip_mlp', model='mlp', widths='784-512-512-10'),
        # the headline network: 161 tensors, most of them tiny
        dict(clip, name='clip_resnet50', model='resnet50'),
        # a decoder in bf16 whose norms and biases are fp32: the norm for a log
        dict(clip, name='norm_of_gradients_mixed', model='decoder', d=512, layers=12, x='mixed', copies=False),
        # the largest set of gradients
        dict(clip, name='clip_decoder', model='decoder', d=1280, layers=16),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, round(low * (high / low) ** rng.random())))


def draw(rng):
    op = rng.choice(['norm', 'norm', 'sample', 'sample', 'clip'])
    if op == 'norm':
        width = _log_int(rng, 16, 8192)
        x = rng.choice(['f32', 'bf16', 'f16'])
        return dict(op=op, rows=_log_int(rng, 1, min(65536, 16384 * 4096 // width)), width=width, x=x, y=rng.choice([x, 'f32']), w=rng.choice([x, 'f32']),
                    train=rng.random() < 0.75, bias=rng.random() < 0.75, blocks=rng.random() < 0.4)
    if op == 'sample':
        classes = _log_int(rng, 10, 131072)
        return dict(op=op, rows=_log_int(rng, 1, min(8192, MOST_LOGITS // classes)), classes=classes, x=rng.choice(['f32', 'bf16', 'f16']),
                    pad=rng.choice([0, 0, rng.randint(1, 64)]), temperature=rng.choice([1.0, 0.0, round(rng.uniform(0.3, 2.0), 2)]),
                    top_k=rng.choice([0, 1, rng.randint(2, 100), _log_int(rng, 2, 20000)]), top_p=rng.choice([0.0, round(rng.uniform(0.05, 0.99), 3)]),
                    min_p=rng.choice([0.0, 0.0, round(rng.uniform(0.001, 0.3), 4)]), mixed=rng.random() < 0.25)
    case = dict(op=op, model=rng.choice(['mlp', 'decoder']), x=rng.choice(['f32', 'bf16', 'mixed']), norm=rng.choice(['two', 'two', 'max']), copies=rng.random() < 0.75)
    if case['model'] == 'mlp':
        case.update(widths='-'.join(str(_log_int(rng, 5, 4096)) for _ in range(rng.randint(2, 12))))
    else:
        case.update(d=_log_int(rng, 33, 1024), layers=rng.randint(1, 20))
    return case


# ------------------------------------------------------------------------------------------------ a user's program
def _shapes(case):
    """Shapes of a model's gradients."""
    if case['model'] == 'mlp':
        widths = [int(w) for w in case['widths'].split('-')]
        return [s for a, b in zip(widths, widths[1:]) for s in ((b, a), (b,))]
    if case['model'] == 'decoder':
        d = case['d']
        return [s for _ in range(case['layers']) for s in ((d,), (d,), (3 * d, d), (3 * d,), (d, d), (d,), (d,), (d,), (4 * d, d), (4 * d,), (d, 4 * d), (d,))]
    blocks = [(64 << i, (64 << max(i - 1, 0)) * (4 if i else 1) if j == 0 else 256 << i, j == 0) for i, depth in enumerate((3, 4, 6, 3)) for j in range(depth)]
    convs = [(64, 3, 7, 7)] + [s for w, cin, first in blocks for s in [(w, cin, 1, 1), (w, w, 3, 3), (4 * w, w, 1, 1)] + ([(4 * w, cin, 1, 1)] if first else [])]
    return [s for c in convs for s in (c, (c[0],), (c[0],))] + [(1000, 2048), (1000,)]


def _requests(rows, rng):
    """Parameters of a batch of requests: some greedy, some without a filter, most with one or two."""
    def pick(values):
        return torch.tensor(values, device='cuda')[torch.randint(0, len(values), (rows,), device='cuda', generator=rng)]
    return dict(temperature=pick([0.0, 0.7, 1.0, 1.3]), top_k=pick([0, 1, 40, 1000]), top_p=pick([1.0, 0.5, 0.9, 0.99]), min_p=pick([0.0, 0.0, 0.05, 0.2]))


def prepare(case, seed):
    rng = torch.Generator('cuda').manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, device='cuda', generator=rng)
    if case['op'] == 'norm':
        rows, width, xt, yt, wt = case['rows'], case['width'], TYPES[case['x']], TYPES[case['y']], TYPES[case['w']]
        # a residual stream: features with means of their own and a few of a larger scale; gradients of a mean loss
        scale = 1 + 9 * (torch.rand(width, device='cuda', generator=rng) < 0.01)
        state = dict(case=case, x=(normal(rows, width) * scale + 0.5 * normal(width)).to(xt), w=(1 + 0.2 * normal(width)).to(wt),
                     b=(0.1 * normal(width)).to(wt) if case['bias'] else None)
        if case['train']:
            state['g'] = (normal(rows, width) * 1e-2).to(yt)
        if case['train'] and case['blocks']:
            state['blocks'] = torch.zeros(width, 2, 2, device='cuda')
        return state
    if case['op'] == 'sample':
        rows, classes = case['rows'], case['classes']
        # a Zipf-like predictive distribution in an order of its own: a few likely classes, a long tail
        tail = -torch.log1p(torch.arange(classes, device='cuda').float())[torch.randperm(classes, device='cuda', generator=rng)]
        logits = torch.empty(rows, classes + case['pad'], device='cuda', dtype=TYPES[case['x']])[:, :classes]
        logits.copy_(1.3 * tail + 1.5 * normal(rows, classes))
        state = dict(case=case, logits=logits, u=torch.rand(rows, device='cuda', dtype=torch.float64, generator=rng))
        state['filters'] = _requests(rows, rng) if case['mixed'] else dict(
            temperature=case['temperature'], top_k=case['top_k'] or None, top_p=case['top_p'] or None, min_p=case['min_p'] or None)
        return state
    grads = []
    for shape in _shapes(case):
        kind = TYPES['f32' if case['x'] == 'mixed' and len(shape) == 1 else 'bf16' if case['x'] == 'mixed' else case['x']]
        g = (normal(*shape) * 10 ** (-4 + 3 * torch.rand((), device='cuda', generator=rng))).to(kind)
        grads.append(g.contiguous(memory_format=torch.channels_last) if len(shape) == 4 else g)      # (as a channels-last model has them)
    state = dict(case=case, grads=grads, max_norm=1.0)
    if case['copies']:      # one bucket for all clipped gradients, each with the strides of its own
        state['bucket'] = torch.zeros(sum(g.numel() for g in grads), device='cuda', dtype=TYPES['bf16' if case['x'] == 'bf16' else 'f32'])
        parts = state['bucket'].split([g.numel() for g in grads])
        state['outs'] = [part.as_strided(g.shape, g.stride(), part.storage_offset()) for part, g in zip(parts, grads)]
    return state


# ------------------------------------------------------------------------------------------------ one pass
def _plain_norm(x, w, b, g, case, blocks):
    xf, wf = x.float(), w.float()
    centred = xf - xf.mean(-1, keepdim=True)
    rstd = (centred.square().mean(-1, keepdim=True) + EPS).rsqrt()
    h = centred * rstd
    y = h * wf if b is None else h * wf + b.float()
    out = [y.to(TYPES[case['y']])]
    if not case['train']:
        return out
    gf = g.float()
    gw, gh = gf * wf, gf * h
    dx = rstd * (gw - gw.mean(-1, keepdim=True) - h * (gw * h).mean(-1, keepdim=True))
    out += [dx.to(x.dtype), gh.sum(0).to(w.dtype)]
    if b is not None:
        out.append(gf.sum(0).to(w.dtype))
    if blocks is not None:
        cross = (gh * gf).sum(0)
        out.append(blocks.copy_(torch.stack([gh.square().sum(0), cross, cross, gf.square().sum(0)], -1).view(-1, 2, 2) / x.shape[0]))
    return out


def _plain_sample(logits, u, temperature, top_k, top_p, min_p):
    """Borders of sums over all classes decide: 64 bits."""
    rows, classes = logits.shape

    def column(v, off):
        return torch.full((rows, 1), off if v is None else v, device='cuda', dtype=torch.float64) if not torch.is_tensor(v) else v.double().view(-1, 1)
    t, k, p, m = column(temperature, 1.0), column(top_k, 0), column(top_p, 1.0), column(min_p, 0.0)
    ordered, index = torch.sort(logits, dim=1, descending=True, stable=True)
    rank = torch.arange(classes, device='cuda')
    ordered = ordered.double()
    weight = torch.exp((ordered - ordered[:, :1]) / torch.where(t > 0, t, 1.0))
    weight = weight * ((rank < torch.where(k > 0, k, classes)) & ((t > 0) | (rank == 0)))
    mass = weight.cumsum(1)
    before = torch.cat([torch.zeros_like(mass[:, :1]), mass[:, :-1]], 1)
    weight = weight * (((before < p * mass[:, -1:]) | (p >= 1)) & (weight >= m))
    del ordered, mass, before
    mass = torch.empty_like(weight).scatter_(1, index, weight).cumsum(1)
    return (mass <= u.view(-1, 1) * mass[:, -1:]).sum(1).clamp(max=classes - 1)


def _plain_clip(grads, case, max_norm, outs):
    if case['norm'] == 'two':
        norm = torch.stack([g.double().square().sum() for g in grads]).sum().sqrt()
    else:
        norm = torch.stack([g.float().abs().max() for g in grads]).max().double()
    if outs is not None:
        factor = (max_norm / (norm + 1e-6)).clamp(max=1.0).float()
        [o.copy_(g.float() * factor) for o, g in zip(outs, grads)]
    return norm.float()


def run(state):
    case = state['case']
    if own:
        from asdl_amd import kernels as K
    if case['op'] == 'norm':
        x, w, b, g, blocks = state['x'], state['w'], state['b'], state.get('g'), state.get('blocks')
        if not own:
            return _plain_norm(x, w, b, g, case, blocks)
        y, mean, rstd = K.layer_norm(x, w, b, EPS, out_dtype=TYPES[case['y']])
        if not case['train']:
            return [y]
        grads = K.layer_norm_backward(g, x, mean, rstd, w, blocks=blocks, alpha=1.0 / x.shape[0], need_bias=b is not None)
        return [y] + [t for t in grads if t is not None] + ([blocks] if blocks is not None else [])
    if case['op'] == 'sample':
        if own:
            return K.sample_filtered(state['logits'], state['u'], check=False, **state['filters'])
        return _plain_sample(state['logits'], state['u'], **state['filters'])
    outs = state.get('outs')
    if not own:
        norm = _plain_clip(state['grads'], case, state['max_norm'], outs)
    elif outs is None:
        norm = K.grad_norm(state['grads'], math.inf if case['norm'] == 'max' else 2.0)
    else:
        norm = K.clip_grad_norm(state['grads'], state['max_norm'], math.inf if case['norm'] == 'max' else 2.0, outs=outs)
    return [norm] if outs is None else [norm, state['bucket']]


# ------------------------------------------------------------------------------------------------ what a pass needs
def work(case):
    size = {'f32': 4, 'bf16': 2, 'f16': 2}
    if case['op'] == 'norm':
        rows, width, xs, ys, ws = case['rows'], case['width'], size[case['x']], size[case['y']], size[case['w']]
        vectors = width * ws * (2 if case['bias'] else 1)
        nbytes, flops = rows * width * (xs + ys) + vectors, 8 * rows * width
        if case['train']:      # x is read once for both passes where that can be done; here it is once a pass
            nbytes += rows * width * (2 * xs + ys) + vectors + (16 * width if case['blocks'] else 0)
            flops += rows * width * (14 + (6 if case['blocks'] else 0))
        return {'bytes': nbytes, 'flops': flops}
    if case['op'] == 'sample':
        logits = case['rows'] * case['classes']
        return {'bytes': logits * size[case['x']] + 16 * case['rows'], 'flops': 6 * logits}
    numbers = [(math.prod(s), 4 if case['x'] == 'f32' or (case['x'] == 'mixed' and len(s) == 1) else 2) for s in _shapes(case)]
    to = 2 if case['x'] == 'bf16' else 4
    return {'bytes': sum(n * (s + (to if case['copies'] else 0)) for n, s in numbers) + 4, 'flops': sum(n for n, _ in numbers) * (3 if case['copies'] else 2)}


# ------------------------------------------------------------------------------------------------ the definitions, in 64 bits
def _exact_norm(state, case):
    x, w = state['x'].double(), state['w'].double()
    n = x.shape[1]
    mean = x.sum(1) / n
    var = ((x * x).sum(1) - n * mean * mean) / n
    sigma = torch.sqrt(var + EPS)
    h = (x - mean[:, None]) / sigma[:, None]
    out = [h * w + (0 if state['b'] is None else state['b'].double())]
    if not case['train']:
        return out
    g = state['g'].double()
    # y = w h(x): the Jacobian of h is (1 - 1/n - h h^T / n) / sigma
    d = g * w
    out += [(d - (d.sum(1) / n)[:, None] - h * ((d * h).sum(1) / n)[:, None]) / sigma[:, None], torch.einsum('rf,rf->f', g, h)]
    if state['b'] is not None:
        out.append(g.sum(0))
    if 'blocks' in state:
        per_row = torch.stack([g * h, g], -1)
        out.append(torch.einsum('rfi,rfj->fij', per_row, per_row) / case['rows'])
    return out


def _exact_sample(state):
    """Row by row: the classes are taken from the likeliest on until a filter says stop."""
    logits, u = state['logits'].double().cpu().numpy(), state['u'].cpu().numpy()
    rows, classes = logits.shape

    def each(name, off):
        v = state['filters'][name]
        return v.double().cpu().numpy() if torch.is_tensor(v) else np.full(rows, off if v is None else v)
    t, k, p, m = each('temperature', 1.0), each('top_k', 0), each('top_p', 1.0), each('min_p', 0.0)
    out = []
    for r in range(rows):
        order = np.lexsort((np.arange(classes), -logits[r]))
        if t[r] == 0:
            out.append(int(order[0]))
            continue
        order = order[:int(k[r])] if k[r] > 0 else order
        odds = np.exp((logits[r][order].astype(np.longdouble) - logits[r][order[0]]) / t[r])
        share = odds / odds.sum()
        kept = share[0] * m[r] <= share
        if p[r] < 1:
            kept &= np.concatenate([[0], np.cumsum(share)[:-1]]) < p[r]
        places = np.sort(order[kept])
        share_at = np.zeros(classes, np.longdouble)
        share_at[order] = share
        steps = np.cumsum(share_at[places])
        out.append(int(places[min(np.searchsorted(steps, u[r] * steps[-1], side='right'), len(places) - 1)]))
    return torch.tensor(out)


def exact(case, seed):
    state = prepare(case, seed)
    if case['op'] == 'norm':
        return _exact_norm(state, case)
    if case['op'] == 'sample':
        return _exact_sample(state) if case['rows'] * case['classes'] <= EXACT_LOGITS else None
    grads = [g.double() for g in state['grads']]
    norm = math.sqrt(math.fsum(float(torch.dot(g.flatten(), g.flatten())) for g in grads)) if case['norm'] == 'two' else max(float(g.abs().max()) for g in grads)
    if not case['copies']:
        return [torch.tensor(norm, dtype=torch.float64)]
    factor = min(1.0, state['max_norm'] / (norm + 1e-6))
    bucket = torch.empty(state['bucket'].numel(), dtype=torch.float64, device='cuda')
    for part, g in zip(bucket.split([g.numel() for g in grads]), grads):
        part.as_strided(g.shape, g.stride(), part.storage_offset()).copy_(g * factor)
    return [torch.tensor(norm, dtype=torch.float64), bucket]
