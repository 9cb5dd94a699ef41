"""What a training step of a decoder keeps and touches around its blocks, as measurable cases: the loss at the vocabulary's end without
the logits, the embedding at its other end with its gradient, and activations kept in 8 bits for the backward pass.

Keys of a case:
  op        'loss' (linear layer and softmax cross entropy), 'embed' (rows of a table), 'kept' (activations in 8 bits)
loss:
  rows, classes, width; x   type of the activations and of the weight;  bias   False: no bias (it has the weight's type)
  reduction 'mean' | 'sum' | 'none';  ignored   share of the rows without a target
  train     False: the loss alone; True: the gradients of activations, weight and bias, too
embed:
  tokens, rows, width; x    type of the table (rows of it) and of the gradients;  scale   factor of the rows that are looked up
  padding   a row of the table takes no gradient (a tenth of the tokens are it);  train     False: the lookup alone
kept:
  kind      'values' (kept and read back), 'gelu' (both ways, the way back from the kept input), 'linear' (gradients of weight and
            bias from the kept input)
  rows, width; x   type of activations and gradients;  out   linear: features of the result;  tanh   gelu: its approximation
"""
import math

import torch

own = False

TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
SIZES = {'f32': 4, 'bf16': 2, 'f16': 2}
IGNORE = -100
MOST_LOGITS, MOST_LOSS = 4096 * 128000, 4096 * 128000 * 2048
MOST_TABLE, MOST_LOOKED_UP = 131072 * 1024, 131072 * 1024
MOST_KEPT, MOST_KEPT_LINEAR = 16384 * 4096, 16384 * 4096 * 4096
BLOCK = 128           # features that share a scale
LARGEST = 448.        # of the 8-bit type (4 bits of exponent, 3 of fraction)


def listed():
    loss = dict(op='loss', bias=False, reduction='mean', ignored=0.03, train=True)
    embed = dict(op='embed', scale=1.0, padding=False, train=True)
    kept = dict(op='kept', x='bf16')
    return [
        # four answers that are scored token by token: the weight is read for a few rows
        dict(loss, name='loss_scoring', rows=4, classes=50257, width=768, x='bf16', reduction='none', ignored=0.0, train=False),
        # rows, classes and features that are no multiple of anything, in fp32
        dict(loss, name='loss_ragged', rows=1000, classes=10007, width=513, x='f32', bias=True, reduction='sum'),
        # the benchmark's decoder of GPT-2-small shape, 8 sequences of 1024 tokens under bf16 autocast, its head trained, too
        dict(loss, name='loss_decoder', rows=8 * 1024, classes=50257, width=768, x='bf16'),
        # a wide model with a larger vocabulary, in fp16
        dict(loss, name='loss_wide', rows=4096, classes=128000, width=2048, x='f16'),
        # four sequences that are decoded token by token: latency alone
        dict(embed, name='embed_decode', tokens=4, rows=50257, width=768, x='bf16', train=False),
        # the benchmark's decoder with its token embedding trained
        dict(embed, name='embed_decoder', tokens=8 * 1024, rows=50257, width=768, x='f32'),
        # a small table, odd sizes, padded sequences, rows times the square root of the width
        dict(embed, name='embed_ragged', tokens=5000, rows=1021, width=257, x='f16', scale=16.03, padding=True),
        # long sequences of a wider model in bf16
        dict(embed, name='embed_long', tokens=128 * 1024, rows=131072, width=1024, x='bf16', scale=32.0),
        # activations of odd sizes, kept and read back
        dict(kept, name='kept_values', kind='values', rows=1000, width=1021, x='f32'),
        # the activation function of a block of a wider decoder
        dict(kept, name='kept_gelu', kind='gelu', rows=8 * 1024, width=4096, tanh=False),
        # the layer in front of the attention of the benchmark's decoder
        dict(kept, name='kept_linear', kind='linear', rows=8 * 1024, width=768, out=2304),
        # a layer of a wide model with long sequences
        dict(kept, name='kept_linear_wide', kind='linear', rows=16384, width=4096, out=4096),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, round(low * (high / low) ** rng.random())))


def draw(rng):
    op = rng.choice(['loss', 'embed', 'kept'])
    x = rng.choice(['f32', 'bf16', 'f16', 'bf16'])
    if op == 'loss':
        width, classes = _log_int(rng, 48, 4096), _log_int(rng, 500, 131072)
        if rng.random() < 0.5:      # (as models have them)
            width, classes = max(64, width // 64 * 64), max(512, classes // 8 * 8)
        most = min(8192, MOST_LOGITS // classes, (MOST_LOSS // 4 if x == 'f32' else MOST_LOSS) // (classes * width))
        return dict(op=op, rows=_log_int(rng, 1, most), classes=classes, width=width, x=x, bias=rng.random() < 0.4,
                    reduction=rng.choice(['mean', 'sum', 'none']), ignored=rng.choice([0.0, 0.03, 0.5]), train=rng.random() < 0.75)
    if op == 'embed':
        width = _log_int(rng, 16, 4096)
        return dict(op=op, tokens=_log_int(rng, 1, min(131072, MOST_LOOKED_UP // width)), rows=_log_int(rng, 50, min(131072, MOST_TABLE // width)), width=width, x=x,
                    scale=rng.choice([1.0, round(math.sqrt(width), 3)]), padding=rng.random() < 0.4, train=rng.random() < 0.75)
    kind, width = rng.choice(['values', 'gelu', 'linear', 'linear']), _log_int(rng, 16, 8192)
    case = dict(op=op, kind=kind, width=width, x=x)
    if kind == 'linear':
        out = _log_int(rng, 16, 8192)
        most = (MOST_KEPT_LINEAR // 2 if x == 'f32' else MOST_KEPT_LINEAR) // (width * out)
        return dict(case, rows=_log_int(rng, 1, min(32768, MOST_KEPT // width, MOST_KEPT // out, most)), out=out)
    case['rows'] = _log_int(rng, 1, min(65536, MOST_KEPT // width))
    return dict(case, tanh=rng.random() < 0.5) if kind == 'gelu' else case


# ------------------------------------------------------------------------------------------------ a user's program
def _tokens(count, rows, rng):
    """Tokens of a text, distributed as 1 / rank in an order of their own."""
    rank = torch.exp(torch.rand(count, device='cuda', dtype=torch.float64, generator=rng) * math.log(rows + 1)).long() - 1
    return torch.randperm(rows, device='cuda', generator=rng)[rank.clamp_(0, rows - 1)]


def prepare(case, seed):
    rng = torch.Generator('cuda').manual_seed(seed)
    kind = TYPES[case['x']]

    def normal(*shape):
        return torch.randn(*shape, device='cuda', generator=rng)
    if case['op'] == 'loss':
        rows, classes, width = case['rows'], case['classes'], case['width']
        targets = _tokens(rows, classes, rng)
        weight = (normal(classes, width) * 0.02 * math.sqrt(768 / width)).to(kind)
        # normed activations; half of the rows point towards their class, some of them are sure of it
        sure = 14 * torch.rand(rows, 1, device='cuda', generator=rng) - 6
        h = normal(rows, width) + sure.clamp(min=0) * weight[targets].float() / (0.02 ** 2 * 768)
        targets[torch.rand(rows, device='cuda', generator=rng) < case['ignored']] = IGNORE
        state = dict(case=case, h=h.to(kind), weight=weight, targets=targets, bias=(0.5 * normal(classes)).to(kind) if case['bias'] else None)
        if case['train']:      # the gradient of the loss: a weight of each row, or a factor that keeps fp16 in its range
            state['g'] = torch.rand(rows, device='cuda', generator=rng) if case['reduction'] == 'none' else 64 * torch.rand((), device='cuda', generator=rng) + 1
        return state
    if case['op'] == 'embed':
        tokens, rows, width = case['tokens'], case['rows'], case['width']
        state = dict(case=case, tokens=_tokens(tokens, rows, rng), table=(0.02 * normal(rows, width)).to(kind), padding=None)
        if case['padding']:
            state['padding'] = rows // 3
            state['tokens'][torch.rand(tokens, device='cuda', generator=rng) < 0.1] = rows // 3
        if case['train']:
            state['g'] = (1e-2 * normal(tokens, width)).to(kind)
        return state
    rows, width = case['rows'], case['width']
    # features with means of their own and a few of a larger scale
    scale = 1 + 9 * (torch.rand(width, device='cuda', generator=rng) < 0.01)
    state = dict(case=case, x=(normal(rows, width) * scale + 0.5 * normal(width)).to(kind))
    if case['kind'] != 'values':
        state['g'] = (1e-2 * normal(rows, case['out'] if case['kind'] == 'linear' else width)).to(kind)
    return state


# ------------------------------------------------------------------------------------------------ one pass
def _plain_loss(state, case):
    h, weight, targets = state['h'].float(), state['weight'].float(), state['targets']
    bias = state['bias']
    logits = h @ weight.t()
    if bias is not None:
        logits += bias.float()
    valid = targets != IGNORE
    at = torch.where(valid, targets, 0).view(-1, 1)
    top = logits.max(1, keepdim=True).values
    lse = top + (logits - top).exp().sum(1, keepdim=True).log()
    losses = torch.where(valid, (lse - logits.gather(1, at)).view(-1), 0.)
    mean = case['reduction'] == 'mean'
    loss = losses if case['reduction'] == 'none' else losses.double().sum().float() / (valid.sum() if mean else 1)
    if not case['train']:
        return [loss]
    g = state['g'] / (valid.sum() if mean else 1)
    d = logits.sub_(lse).exp_()
    d.scatter_add_(1, at, torch.full_like(at, -1, dtype=torch.float32))
    d *= torch.where(valid, g, 0.).view(-1, 1)
    out = [loss, (d @ weight).to(state['h'].dtype), (d.t() @ h).to(state['weight'].dtype)]
    return out if bias is None else out + [d.sum(0).to(bias.dtype)]


def _plain_embed(state, case):
    tokens, table, scale = state['tokens'], state['table'], case['scale']
    out = [(table[tokens].float() * scale).to(table.dtype)]
    if case['train']:
        grad = torch.zeros(table.shape, device='cuda').index_add_(0, tokens, state['g'].float())
        if state['padding'] is not None:
            grad[state['padding']] = 0
        out.append((grad * scale).to(table.dtype))
    return out


def _plain_kept(x):
    """The values that ``x`` is kept as: 8 bits times a power of two of each block of a row, the smallest that the block fits."""
    rows, width = x.shape
    blocks = torch.nn.functional.pad(x.float(), (0, -width % BLOCK)).view(rows, -1, BLOCK)
    fraction, exponent = torch.frexp(blocks.abs().amax(2))
    exponent = torch.where(fraction == 0, -127, exponent - 9 + (2 * fraction * 256 > LARGEST).int()).clamp_(-127, 127)
    codes = torch.ldexp(blocks, -exponent[..., None]).to(torch.float8_e4m3fn)
    return torch.ldexp(codes.float(), exponent[..., None]).view(rows, -1)[:, :width]


def _plain_gelu(x, tanh):
    """(GELU, its derivative)"""
    if tanh:
        t = torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3))
        return 0.5 * x * (1 + t), 0.5 * (1 + t) + 0.5 * x * (1 - t * t) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * x * x)
    below = 0.5 * torch.erfc(x * -math.sqrt(0.5))
    return x * below, below + x * torch.exp(-0.5 * x * x) / math.sqrt(2 * math.pi)


def run(state):
    case = state['case']
    if own:
        from asdl_amd import kernels as K
    if case['op'] == 'loss':
        if not own:
            return _plain_loss(state, case)
        h, weight, targets, bias = state['h'], state['weight'], state['targets'], state['bias']
        loss, lse = K.linear_cross_entropy(h, weight, targets, bias, ignore_index=IGNORE, reduction=case['reduction'])
        if not case['train']:
            return [loss]
        grads = K.linear_cross_entropy_backward(state['g'], h, weight, targets, lse, bias, ignore_index=IGNORE, reduction=case['reduction'])
        return [loss] + [t for t in grads if t is not None]
    if case['op'] == 'embed':
        if not own:
            return _plain_embed(state, case)
        out = [K.embedding(state['tokens'], state['table'], case['scale'])]
        if case['train']:
            out.append(K.embedding_backward(state['g'], state['tokens'], case['rows'], case['scale'], padding_idx=state['padding']))
        return out
    x = state['x']
    if case['kind'] == 'values':
        return [K.dequantize_8bit(K.quantize_8bit(x), x.dtype) if own else _plain_kept(x).to(x.dtype)]
    if case['kind'] == 'gelu':
        if own:
            way = 'tanh' if case['tanh'] else 'none'
            y, kept = K.gelu_8bit(x, way)
            return [y, K.gelu_8bit_backward(state['g'], kept, way)]
        return [_plain_gelu(x.float(), case['tanh'])[0].to(x.dtype), (_plain_gelu(_plain_kept(x), case['tanh'])[1] * state['g'].float()).to(x.dtype)]
    if own:
        return list(K.weight_grad_8bit(state['g'], K.quantize_8bit(x)))
    g = state['g'].float()
    return [(g.t() @ _plain_kept(x)).to(x.dtype), g.sum(0).to(x.dtype)]


# ------------------------------------------------------------------------------------------------ what a pass needs
def work(case):
    size = SIZES[case['x']]
    if case['op'] == 'loss':
        rows, classes, width = case['rows'], case['classes'], case['width']
        operands = (rows + classes) * width * size + (classes * size if case['bias'] else 0)
        return {'bytes': operands * (2 if case['train'] else 1) + 12 * rows, 'flops': rows * classes * (2 * width + 4) * (3 if case['train'] else 1)}
    if case['op'] == 'embed':
        looked_up, touched = case['tokens'] * case['width'], min(case['tokens'], case['rows']) * case['width']
        nbytes, flops = (touched + looked_up) * size + 8 * case['tokens'], looked_up
        if case['train']:
            nbytes, flops = nbytes + (looked_up + case['rows'] * case['width']) * size, 2 * flops + case['rows'] * case['width']
        return {'bytes': nbytes, 'flops': flops}
    values = case['rows'] * case['width']
    if case['kind'] == 'linear':
        gradients, out = case['rows'] * case['out'], (case['width'] + 1) * case['out']
        return {'bytes': (values + gradients + out) * size, 'flops': 2 * values * case['out']}
    return {'bytes': values * size * (2 if case['kind'] == 'values' else 4), 'flops': values * (4 if case['kind'] == 'values' else 30)}


# ------------------------------------------------------------------------------------------------ the definitions, in 64 bits
def _exact_loss(state, case):
    """Rows in pieces; a row's loss is the log of a sum of differences, its gradient the shares of the classes less its own."""
    weight, targets = state['weight'].double(), state['targets']
    rows, classes = case['rows'], case['classes']
    valid = (targets != IGNORE).double()
    shares = valid / valid.sum() if case['reduction'] == 'mean' else valid
    losses, dh = torch.zeros(rows, dtype=torch.float64, device='cuda'), torch.zeros(rows, case['width'], dtype=torch.float64, device='cuda')
    dw, db = torch.zeros_like(weight), torch.zeros(classes, dtype=torch.float64, device='cuda')
    for i in range(0, rows, 1024):
        part = slice(i, min(i + 1024, rows))
        h = state['h'][part].double()
        scores = torch.mm(h, weight.t())
        if state['bias'] is not None:
            scores = scores + state['bias'].double()[None]
        own_class = targets[part].clamp(min=0)
        losses[part] = torch.logsumexp(scores, 1) - scores[torch.arange(len(h), device='cuda'), own_class]
        if case['train']:
            d = torch.softmax(scores, 1)
            d[torch.arange(len(h), device='cuda'), own_class] -= 1
            d *= (state['g'].double() * shares)[part, None]
            dh[part] = torch.mm(d, weight)
            dw += torch.mm(d.t(), h)
            db += d.sum(0)
    losses *= valid
    out = [losses if case['reduction'] == 'none' else (losses * shares).sum()]
    if case['train']:
        out += [dh, dw] + ([db] if state['bias'] is not None else [])
    return out


def _exact_embed(state, case):
    table, tokens, scale = state['table'].double(), state['tokens'], case['scale']
    out = [torch.index_select(table, 0, tokens) * scale]
    if case['train']:
        order = torch.argsort(tokens, stable=True)
        grad = torch.zeros_like(table)
        at, g = tokens[order], state['g'][order]
        pieces = max(1, (1 << 27) // case['width'])
        for i in range(0, len(at), pieces):
            grad.index_put_((at[i:i + pieces],), g[i:i + pieces].double() * scale, accumulate=True)
        if state['padding'] is not None:
            grad[state['padding']].zero_()
        out.append(grad)
    return out


def _exact_kept(x):
    """Nearest of the 8-bit values (even fractions on ties), whose step is 2^-3 of the value's power of two and 2^-9 at least."""
    x = x.double()
    out = torch.empty_like(x)
    for i in range(0, x.shape[1], BLOCK):
        block = x[:, i:i + BLOCK]
        largest = block.abs().max(1, keepdim=True).values
        power = torch.floor(torch.log2(largest.clamp(min=2.0 ** -200)))
        power = power - torch.where(torch.exp2(power) > largest, 1.0, 0.0)
        scale = torch.exp2((power - 8 + torch.where(largest * torch.exp2(8 - power) > LARGEST, 1.0, 0.0)).clamp(-127, 127))
        v = block / scale
        own_power = torch.frexp(v)[1].double() - 1
        step = torch.exp2(torch.where(v == 0, -6.0, own_power).clamp(min=-6) - 3)
        out[:, i:i + BLOCK] = torch.round(v / step) * step * scale
    return out


def _exact_normal(x, tanh):
    """(share of the normal distribution below x or its approximation, its derivative)"""
    if not tanh:
        return 0.5 * torch.special.erfc(-x / math.sqrt(2)), torch.exp(-x * x / 2) / math.sqrt(2 * math.pi)
    inner = math.sqrt(8 / math.pi) * (x + 0.044715 * x * x * x)
    below = torch.sigmoid(inner)
    return below, below * torch.sigmoid(-inner) * math.sqrt(8 / math.pi) * (1 + 0.134145 * x * x)


def exact(case, seed):
    state = prepare(case, seed)
    if case['op'] == 'loss':
        return _exact_loss(state, case)
    if case['op'] == 'embed':
        return _exact_embed(state, case)
    kept = _exact_kept(state['x'])
    if case['kind'] == 'values':
        return [kept]
    g = state['g'].double()
    if case['kind'] == 'linear':
        return [torch.mm(g.t(), kept), g.sum(0)]
    x = state['x'].double()
    below, slope = _exact_normal(kept, case['tanh'])
    return [x * _exact_normal(x, case['tanh'])[0], g * (below + kept * slope)]
