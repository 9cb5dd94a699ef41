"""The cross entropy of a linear layer, embeddings and activations in 8 bits against their definitions in 64 bits.

Tolerances.  u = 2^-24 is half a step of float32, e half a step of the type that is stored (relative to the value).  fp16 numbers below 2^-14 are
multiples of 2^-24: half a step of them is 2^-25 whatever their size (a gradient of 4e-6 is off by up to 3e-8): that much more for every fp16 result.
Scores s = h w + b: products of 16-bit numbers are exact in float32, those of float32 numbers are off by 2^-22 at most (three pieces);
a sum of D terms in any order is off by at most D u of the sum of magnitudes a = |h||w| + |b|, twice that where the matrix cores cut
instead of rounding: es = (2 D u + 2^-21) a.  lse: the error of the scores, and of exp, sums and log, 2^-20 (1 + its magnitude) with room: el.
Loss: es of the target's score + el.  A mean or sum of losses: the sum of those.
d = c (p - [target]): off by |c| (p (es + el + 2^-20 (1 + |s - lse|)) + 2^-22), which is systematic and summed up as it is; and by a rounding to
the operands' type, e |d|, half a step each, independent of each other: a sum of w d is off by t times the root of the sum of (w e d)^2 with
probability 2 exp(-t^2 / 2) (Hoeffding): t = 7.  fp16 values of d below 2^-28 of the largest c are rounded to a step of 2^-38 of it.
Sums of d over n terms: 2 n u of the magnitudes.
Embedding: rows are exact products rounded once; a sum of c gradients in fp32, in any order: c u of the magnitudes.
8 bits: codes and exponents are whole numbers and equal.  gelu: P and P' within 2^-21 (1 + |x|)^2 exp(-x^2 / 2 cut at 2^-21 of itself), one half
step stored: written as 2^-20 |x| here.  Weight gradients: exact products, sums of n terms: 2 n u of the magnitudes."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = 2.0 ** -24
NAN, INF = float('nan'), float('inf')


@pytest.fixture(scope='module')
def K():
    from asdl_amd import kernels
    return kernels


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rand(*shape, seed, dtype=F32, scale=1.0, shift=0.0):
    gen = torch.Generator('cuda').manual_seed(seed)
    return (torch.randn(shape, device='cuda', generator=gen) * scale + shift).to(dtype)


def ints(high, *shape, seed):
    return torch.randint(0, high, shape, device='cuda', generator=torch.Generator('cuda').manual_seed(seed))


def within(got, want, bound, what):
    got = got.double()
    bad = ~((got - want).abs() <= bound) & ~((got == want) | (got.isnan() & want.isnan()))
    worst = ((got - want).abs() / bound.clamp_min(1e-300)).nan_to_num(posinf=1e9).max()
    assert not bool(bad.any()), f'{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(worst):.3g} of the bound'


# ------------------------------------------------------------------------------------------------ cross entropy of a linear layer
def loss64(h, w, t, b=None, ignore=-100, reduction='mean', g=None):
    """Values and bounds: dict of name -> (value, bound)."""
    e = half_step(h.dtype)
    dtype, rows = h.dtype, t.numel()
    h, w, t = h.reshape(rows, -1).double(), w.double(), t.reshape(-1)
    D = h.shape[1]
    s, a = h @ w.t(), h.abs() @ w.abs().t()
    if b is not None:
        s, a = s + b.double(), a + b.double().abs().nan_to_num(posinf=0.0)
    es = (2 * D * U + 2.0 ** -21) * a
    lse = torch.logsumexp(s, 1)
    p = torch.exp(s - lse[:, None])
    el = (p * es).sum(1) + 2.0 ** -20 * (1 + lse.abs())
    valid = t != ignore
    at = torch.where(valid, t, 0)[:, None]
    losses = torch.where(valid, lse - s.gather(1, at)[:, 0], 0.0)
    bounds = torch.where(valid, es.gather(1, at)[:, 0] + el + 2 * U * losses.abs(), 0.0)
    count = int(valid.sum())
    share = valid.double() / (count if reduction == 'mean' else 1)
    out = dict(lse=(lse, el + U * lse.abs()))
    if reduction == 'none':
        out['loss'] = (losses, bounds)
    else:
        total = (losses * share).sum()
        out['loss'] = (total, (bounds * share).sum() + 2 * U * total.abs())
    if g is None:
        return out
    c = torch.where(valid, g.reshape(-1).double() * share, 0.0)[:, None]
    d = p.scatter_add(1, at, torch.full_like(at, -1, dtype=torch.float64)) * c
    fixed = c.abs() * (p * (es + el[:, None] + 2.0 ** -20 * (1 + (s - lse[:, None]).abs().nan_to_num(posinf=0.0))) + 2.0 ** -22)
    loose = e * d.abs() if dtype != F32 else 0 * d
    if dtype == F16:
        loose = loose + 2.0 ** -38 * c.abs().max()

    def product(d_left, x, n):
        """d_left(d) @ x with the errors above."""
        value, magnitude = d_left(d) @ x, d_left(d.abs()) @ x.abs()
        return value, d_left(fixed) @ x.abs() + 7 * (d_left(loose * loose) @ (x * x)).sqrt() + 2 * n * U * magnitude + e * value.abs() + (2.0 ** -25 if dtype == F16 else 1e-30)
    out['dh'] = product(lambda m: m, w, w.shape[0])
    out['dw'] = product(lambda m: m.t(), h, rows)
    ones = torch.ones(rows, 1, dtype=torch.float64, device='cuda')
    value, bound = product(lambda m: m.t(), ones, rows)
    out['db'] = (value[:, 0], bound[:, 0])
    return out


def check_loss(K, h, w, t, b=None, ignore=-100, reduction='mean', g=None, **need):
    want = loss64(h, w, t, b, ignore, reduction, g)
    loss, lse = K.linear_cross_entropy(h, w, t, b, ignore, reduction)
    assert loss.dtype == lse.dtype == F32 and lse.shape == t.shape and loss.shape == (t.shape if reduction == 'none' else ())
    within(lse.reshape(-1), *want['lse'], 'lse')
    within(loss.reshape(want['loss'][0].shape), *want['loss'], 'loss')
    if g is None:
        return
    grads = K.linear_cross_entropy_backward(g, h, w, t, lse, b, ignore, reduction, **need)
    for name, got, like in zip(('dh', 'dw', 'db'), grads, (h, w, b)):
        if like is None:
            assert got is None
            continue
        assert got.dtype == like.dtype and got.shape == like.shape
        bound = want[name][1]
        if like.dtype != h.dtype:
            bound = bound + half_step(like.dtype) * want[name][0].abs()
        within(got.reshape(want[name][0].shape), want[name][0], bound, name)


def gradient_of(reduction, t, seed):
    gen = torch.Generator('cuda').manual_seed(seed)
    return torch.rand(t.shape if reduction == 'none' else (), device='cuda', generator=gen) * 3 - 1


LOSSES = [(1, 1, 1), (1, 2, 8), (3, 17, 33), (5, 130, 64), (16, 1000, 100), (17, 257, 128), (33, 129, 257), (64, 5003, 72), (65, 300, 40), (130, 1000, 136),
          (300, 257, 520), (257, 1030, 64), (1, 5003, 768), (700, 50, 31)]


@pytest.mark.parametrize('dtype', [F32, BF16, F16])
@pytest.mark.parametrize('rows,classes,width', LOSSES)
def test_linear_cross_entropy_matches_its_definition(K, rows, classes, width, dtype):
    print(f'linear_cross_entropy {rows}x{classes}x{width} {dtype}', flush=True)
    h, w = rand(rows, width, seed=rows, dtype=dtype), rand(classes, width, seed=classes, dtype=dtype, scale=2 / math.sqrt(width))
    t = ints(classes, rows, seed=width)
    if rows > 4:
        t[::5] = -100
    reduction = ('mean', 'sum', 'none')[(rows + classes) % 3]
    b = None if rows % 2 else rand(classes, seed=7, dtype=(dtype, F32)[classes % 2])
    check_loss(K, h, w, t, b, reduction=reduction, g=gradient_of(reduction, t, rows))


@pytest.mark.parametrize('dtype', [F32, BF16, F16])
@pytest.mark.parametrize('reduction', ['mean', 'sum', 'none'])
def test_linear_cross_entropy_of_sure_rows(K, dtype, reduction):
    """Rows whose class has almost all of the probability, and rows whose class has almost none."""
    rows, classes, width = 200, 700, 64
    w = rand(classes, width, seed=1, dtype=dtype)
    t = ints(classes, rows, seed=2)
    h = (rand(rows, width, seed=3) * 0.1 + w[t].float() * torch.linspace(-0.3, 0.5, rows, device='cuda')[:, None]).to(dtype)
    check_loss(K, h, w, t, reduction=reduction, g=gradient_of(reduction, t, 4) * (1000 if reduction == 'none' else 1))


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('rows', [3, 150])
def test_linear_cross_entropy_of_masked_classes(K, dtype, rows):
    """A bias of -inf, or of the type's lowest value, takes classes out; a row of nothing else is NaN, as softmax of it is."""
    classes, width = 400, 48
    h, w = rand(rows, width, seed=1, dtype=dtype), rand(classes, width, seed=2, dtype=dtype, scale=0.2)
    t = ints(100, rows, seed=3) * 4 + 1
    for mask in (-INF, torch.finfo(dtype).min):
        b = rand(classes, seed=4, dtype=dtype)
        b[::2] = mask
        check_loss(K, h, w, t, b, reduction='none')
        loss, lse = K.linear_cross_entropy(h, w, t, b, reduction='none')
        dh, dw, db = K.linear_cross_entropy_backward(torch.ones_like(loss), h, w, t, lse, b, reduction='none')
        assert not bool(dh.isnan().any()) and bool((dw[::2] == 0).all()) and bool((db[::2] == 0).all()) and bool((db[1::2] != 0).any())
    assert bool((K.linear_cross_entropy(h, w, t - 1, torch.where(torch.arange(classes, device='cuda') % 2 == 0, -INF, 0.0).to(dtype), reduction='none')[0] == INF).all())
    loss, lse = K.linear_cross_entropy(h, w, t, torch.full((classes,), -INF, device='cuda', dtype=dtype), reduction='none')
    assert bool(loss.isnan().all()) and bool((lse == -INF).all())


@pytest.mark.parametrize('dtype', [F32, BF16, F16])
@pytest.mark.parametrize('rows', [4, 100])
def test_linear_cross_entropy_keeps_rows_apart(K, dtype, rows):
    """NaN and infinity in a row, targets that are no class: that row's loss is NaN, the others' are what they are; an ignored row
    of NaN gives no gradient."""
    classes, width = 300, 40
    h, w = rand(rows, width, seed=1, dtype=dtype), rand(classes, width, seed=2, dtype=dtype)
    t = ints(classes, rows, seed=3)
    want, _ = K.linear_cross_entropy(h, w, t, reduction='none')
    h[0, 3], h[1, 5] = NAN, INF
    bad = t.clone()
    bad[2] = classes
    bad[3] = -1
    loss, lse = K.linear_cross_entropy(h, w, bad, reduction='none')
    assert bool(loss[:4].isnan().all()) and torch.equal(loss[4:], want[4:])
    ignored = t.clone()
    ignored[:2] = -100
    loss, lse = K.linear_cross_entropy(h, w, ignored)
    assert not bool(loss.isnan())
    dh, dw, _ = K.linear_cross_entropy_backward(torch.ones_like(loss), h, w, ignored, lse)
    assert bool((dh[:2] == 0).all()) and not bool(dh.isnan().any())
    if rows == 4:
        return
    h[:2] = 0
    dh2, dw2, _ = K.linear_cross_entropy_backward(torch.ones_like(loss), h, w, ignored, lse)
    assert torch.equal(dh[2:], dh2[2:])


def test_linear_cross_entropy_without_targets(K):
    h, w = rand(20, 16, seed=1), rand(30, 16, seed=2)
    t = torch.full((20,), 7, device='cuda')
    loss, lse = K.linear_cross_entropy(h, w, t, ignore_index=7)
    assert bool(loss.isnan())
    for x, like in zip(K.linear_cross_entropy_backward(torch.ones_like(loss), h, w, t, lse, ignore_index=7), (h, w)):
        assert torch.equal(x, torch.zeros_like(like))
    assert float(K.linear_cross_entropy(h, w, t, ignore_index=7, reduction='sum')[0]) == 0
    none, none_lse = K.linear_cross_entropy(h[:0], w, t[:0])
    assert bool(none.isnan()) and none_lse.shape == (0,)
    dh, dw, db = K.linear_cross_entropy_backward(none, h[:0], w, t[:0], none_lse, torch.zeros(30, device='cuda'))
    assert dh.shape == (0, 16) and torch.equal(dw, torch.zeros_like(w)) and torch.equal(db, torch.zeros(30, device='cuda'))


@pytest.mark.parametrize('dtype', [F32, BF16, F16])
@pytest.mark.parametrize('rows', [6, 120])
def test_linear_cross_entropy_reads_strided_operands_of_any_alignment(K, dtype, rows):
    classes, width = 260, 72
    big, wide = rand(rows, 3, width + 5, seed=1, dtype=dtype), rand(classes, width + 3, seed=2, dtype=dtype, scale=0.3)
    t = ints(classes, 2 * rows, seed=3)[::2]
    b = rand(2 * classes, seed=4, dtype=dtype)[1::2]
    for off in (0, 1, 3):
        h, w = big[:, 1, off:off + width], wide[:, min(off, 3):min(off, 3) + width]
        check_loss(K, h, w, t, b, g=gradient_of('mean', t, 5))
        assert all(torch.equal(p, q) for p, q in zip(K.linear_cross_entropy(h, w, t, b), K.linear_cross_entropy(h.contiguous(), w.contiguous(), t, b)))
    h3 = big[:, :, :width]
    t3 = ints(classes, rows, 3, seed=6)
    check_loss(K, h3, w, t3, b, reduction='none', g=gradient_of('none', t3, 7))


@pytest.mark.parametrize('dtype', [F32, BF16, F16])
@pytest.mark.parametrize('rows', [8, 9, 16, 17, 40, 64])
def test_linear_cross_entropy_of_few_rows_of_any_alignment(K, rows, dtype):
    """Either operand where vectors do not begin; rows that end with the tensors' memory."""
    for off_h, off_w, width in ((0, 0, 64), (1, 0, 64), (0, 1, 64), (3, 1, 151), (0, 0, 151)):
        h = rand(rows * (width + off_h), seed=1, dtype=dtype).view(rows, -1)[:, off_h:]
        w = rand(300 * (width + off_w), seed=2, dtype=dtype, scale=0.2).view(300, -1)[:, off_w:]
        t = ints(300, rows, seed=3)
        check_loss(K, h, w, t, reduction='sum', g=gradient_of('sum', t, 4))


@pytest.mark.parametrize('dtype', [F32, BF16, F16])
def test_linear_cross_entropy_gives_what_is_asked_for(K, dtype):
    h, w, t, b = rand(90, 64, seed=1, dtype=dtype), rand(500, 64, seed=2, dtype=dtype), ints(500, 90, seed=3), rand(500, seed=4)
    loss, lse = K.linear_cross_entropy(h, w, t, b)
    g = torch.ones_like(loss)
    whole = K.linear_cross_entropy_backward(g, h, w, t, lse, b)
    for bits in range(8):
        need = dict(need_h=bool(bits & 1), need_weight=bool(bits & 2), need_bias=bool(bits & 4))
        got = K.linear_cross_entropy_backward(g, h, w, t, lse, b, **need)
        for wanted, x, y in zip(need.values(), got, whole):
            assert torch.equal(x, y) if wanted else x is None
    assert all(torch.equal(x, y) for x, y in zip(whole, K.linear_cross_entropy_backward(g, h, w, t, lse, b)))       # the same bits every time


@pytest.mark.parametrize('dtype,rows,classes,width', [(BF16, 2100, 70001, 64), (F16, 4200, 33000, 40), (F32, 1030, 66000, 36), (BF16, 9000, 16500, 72),
                                                      (BF16, 4200, 70001, 64), (F16, 9000, 33000, 40), (F32, 1030, 90001, 36), (BF16, 1100000, 600, 8), (BF16, 3, (1 << 24) + 300, 8)])
def test_linear_cross_entropy_in_pieces(K, dtype, rows, classes, width):
    """Up to 512 MB of the logits' gradient, as float32 in three pieces of 16 bits, and more: several pieces of the classes, the last one shorter;
    with very many rows pieces of 256 classes, with very many classes pieces of 2^24."""
    print(f'linear_cross_entropy {rows}x{classes}x{width} {dtype}', flush=True)
    h, w = rand(rows, width, seed=1, dtype=dtype), rand(classes, width, seed=2, dtype=dtype, scale=0.2)
    t = ints(classes, rows, seed=3)
    t[7::9] = -100
    check_loss(K, h, w, t, rand(classes, seed=4), g=torch.tensor(2.5, device='cuda'))


@pytest.mark.parametrize('dtype', [BF16, F16])
@pytest.mark.parametrize('scale', [2.0 ** -60, 1e-4, 1.0, 2.0 ** 20])
def test_linear_cross_entropy_of_scaled_gradients(K, dtype, scale):
    """Gradients of the loss of any size lose nothing in the 16-bit gradient of the logits (results are checked before they leave fp16's
    range: as float32 sums of float32 weights would be)."""
    h, w, t = rand(150, 64, seed=1, dtype=dtype), rand(3000, 64, seed=2, dtype=dtype, scale=0.1), ints(3000, 150, seed=3)
    loss, lse = K.linear_cross_entropy(h, w, t, reduction='none')
    g = gradient_of('none', t, 4)
    one = K.linear_cross_entropy_backward(g, h, w, t, lse, reduction='none')
    scaled = K.linear_cross_entropy_backward(g * scale, h, w, t, lse, reduction='none')
    if dtype == BF16 and math.log2(scale) % 1 == 0:
        assert all(torch.equal(x.float() * scale, y.float()) for x, y in zip(one[:2], scaled[:2]))
    elif scale in (1e-4, 1.0):
        check_loss(K, h, w, t, reduction='none', g=g)
    assert all(bool(y.isfinite().all()) for y in scaled[:2]) or (dtype == F16 and scale > 1)


@pytest.mark.parametrize('dtype', [F32, BF16, F16])
def test_linear_cross_entropy_of_gradients_that_are_no_numbers(K, dtype):
    """An infinite or NaN gradient of one row leaves the other rows' alone."""
    h, w, t = rand(70, 64, seed=1, dtype=dtype), rand(300, 64, seed=2, dtype=dtype, scale=0.1), ints(300, 70, seed=3)
    loss, lse = K.linear_cross_entropy(h, w, t, reduction='none')
    g = gradient_of('none', t, 4) * 50
    g[5] = g[9] = 0
    want = loss64(h, w, t, reduction='none', g=g)['dh']
    g[5], g[9] = INF, NAN
    dh = K.linear_cross_entropy_backward(g, h, w, t, lse, reduction='none')[0]
    rest = torch.ones(70, dtype=torch.bool, device='cuda')
    rest[[5, 9]] = False
    within(dh[rest], want[0][rest], want[1][rest], 'dh')
    assert not bool(dh[~rest].isfinite().any())


def test_linear_cross_entropy_refuses(K):
    h, w, t, b = rand(6, 8, seed=1), rand(10, 8, seed=2), ints(10, 6, seed=3), rand(10, seed=4)
    loss, lse = K.linear_cross_entropy(h, w, t, b)
    for call in (lambda: K.linear_cross_entropy(h, w[:, :7], t), lambda: K.linear_cross_entropy(h, w, t[:5]), lambda: K.linear_cross_entropy(h, w, t.int()),
                 lambda: K.linear_cross_entropy(h, w, t, b[:9]), lambda: K.linear_cross_entropy(h, w, t, reduction='max'),
                 lambda: K.linear_cross_entropy(h[:, :0], w[:, :0], t), lambda: K.linear_cross_entropy(h, w[:0], t),
                 lambda: K.linear_cross_entropy_backward(loss.double(), h, w, t, lse), lambda: K.linear_cross_entropy_backward(lse, h, w, t, lse),
                 lambda: K.linear_cross_entropy_backward(loss, h, w, t, lse[:3])):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: K.linear_cross_entropy(h.double(), w.double(), t), lambda: K.linear_cross_entropy(h, w.bfloat16(), t),
                 lambda: K.linear_cross_entropy(h, w, t, b.half())):
        with pytest.raises(TypeError):
            call()
    for call in (lambda: K.linear_cross_entropy(h.cpu(), w, t), lambda: K.linear_cross_entropy(h, w.cpu(), t), lambda: K.linear_cross_entropy(h, w, t.cpu())):
        with pytest.raises(RuntimeError, match='ROCm device'):
            call()


# ------------------------------------------------------------------------------------------------ embedding
def check_embedding(K, tokens, table, scale=1.0, padding=None, g=None, out_dtype=None, dtype=None):
    y = K.embedding(tokens, table, scale, out_dtype)
    assert y.dtype == (out_dtype or table.dtype) and y.shape == (*tokens.shape, table.shape[1])
    exact = table.double()[tokens.long()] * scale
    # (the factor is a float32 number, its product is rounded twice where the result has fewer bits)
    within(y, exact, exact.abs() * (half_step(y.dtype) + 2 * U) + 2.0 ** -25, 'rows')
    if g is None:
        return
    V, D = table.shape
    got = K.embedding_backward(g, tokens, V, scale, padding, dtype=dtype)
    assert got.dtype == (dtype or g.dtype) and got.shape == (V, D)
    flat, gd = tokens.reshape(-1).long(), g.reshape(-1, D).double()
    want = torch.zeros(V, D, dtype=torch.float64, device='cuda').index_add_(0, flat, gd) * scale
    size = torch.zeros(V, D, dtype=torch.float64, device='cuda').index_add_(0, flat, gd.abs()) * abs(scale)
    count = torch.bincount(flat, minlength=V).double()[:, None]
    if padding is not None:
        want[padding], size[padding] = 0, 0
    within(got, want, (count + 4) * U * size + half_step(got.dtype) * want.abs() + (2.0 ** -25 if got.dtype == F16 else 0), 'gradient')
    assert torch.equal(got, K.embedding_backward(g, tokens, V, scale, padding, dtype=dtype))
    absent = count[:, 0] == 0
    assert bool((got[absent] == 0).all())


EMBEDDINGS = [(1, 1, 1), (1, 50, 8), (3, 7, 33), (64, 5, 100), (65, 1000, 257), (500, 513, 64), (1000, 3, 520), (4099, 1021, 36), (3000, 50257, 48), (9000, 131, 768),
              (20011, 600, 17)]


@pytest.mark.parametrize('dtype', [F32, BF16, F16])
@pytest.mark.parametrize('tokens,rows,width', EMBEDDINGS)
def test_embedding_matches_its_definition(K, tokens, rows, width, dtype):
    print(f'embedding {tokens} of {rows}x{width} {dtype}', flush=True)
    table, g = rand(rows, width, seed=rows, dtype=dtype), rand(tokens, width, seed=tokens, dtype=dtype)
    rank = torch.rand(tokens, device='cuda', generator=torch.Generator('cuda').manual_seed(width))
    skewed = (rows ** rank.double()).long().clamp_(max=rows) - 1
    even = ints(rows, tokens, seed=5)
    check_embedding(K, skewed, table, 1.0, None, g)
    check_embedding(K, even.int(), table, 3.7, rows // 2, g, out_dtype=F32, dtype=F32)
    check_embedding(K, torch.full_like(even, rows - 1), table, -0.5, None, g, dtype=dtype)


@pytest.mark.parametrize('gt', [F32, BF16, F16])
@pytest.mark.parametrize('wt', [F32, BF16, F16])
def test_embedding_gradient_is_added_to(K, gt, wt):
    """out <- beta*out + gradient, of any two types, rows of any stride: of a weight that the head has written to before."""
    V, D = 300, 72
    tokens = ints(200, 900, seed=1)
    g = rand(900, D, seed=2, dtype=gt)
    grad = K.embedding_backward(g, tokens, V, 2.0, dtype=F32).double()
    size = K.embedding_backward(g.abs(), tokens, V, 2.0, dtype=F32).double()
    for beta in (1.0, 0.5):
        room = torch.full((V, D + 11), 7.0, device='cuda', dtype=wt)
        out = room[:, 3:3 + D]
        old = rand(V, D, seed=3, dtype=wt)
        out.copy_(old)
        assert K.embedding_backward(g, tokens, V, 2.0, out=out, beta=beta) is out
        want = beta * old.double() + grad
        within(out, want, half_step(wt) * want.abs() + 40 * U * (size + old.double().abs()) + (2.0 ** -25 if wt == F16 else 0), 'sum')
        assert bool((room[:, :3] == 7).all()) and bool((room[:, 3 + D:] == 7).all())
        if beta == 1.0:
            assert torch.equal(out[200:], old[200:])
    room = torch.full((V, D), NAN, device='cuda', dtype=wt)
    K.embedding_backward(g, tokens, V, out=room)
    assert not bool(room.isnan().any())


@pytest.mark.parametrize('dtype', [F32, BF16, F16])
def test_embedding_of_tokens_that_name_no_row(K, dtype):
    table = rand(40, 24, seed=1, dtype=dtype)
    tokens = ints(40, 300, seed=2)
    odd = tokens.clone()
    odd[3], odd[77], odd[200] = -1, 40, 2 ** 40
    y = K.embedding(odd, table)
    bad = torch.zeros(300, dtype=torch.bool, device='cuda')
    bad[[3, 77, 200]] = True
    assert bool(y[bad].isnan().all()) and torch.equal(y[~bad], table[tokens[~bad]])
    g = rand(300, 24, seed=3, dtype=dtype)
    assert torch.equal(K.embedding_backward(g, odd, 40), K.embedding_backward(g[~bad], tokens[~bad], 40))


def test_embedding_of_nothing(K):
    table = rand(10, 8, seed=1)
    none = torch.zeros(0, 5, dtype=torch.int64, device='cuda')
    assert K.embedding(none, table).shape == (0, 5, 8)
    assert torch.equal(K.embedding_backward(torch.zeros(0, 5, 8, device='cuda'), none, 10), torch.zeros(10, 8, device='cuda'))
    one = torch.tensor(3, device='cuda')
    assert torch.equal(K.embedding(one, table), table[3])
    assert K.embedding_backward(torch.ones(2, 8, device='cuda'), torch.zeros(2, dtype=torch.int64, device='cuda'), 0).shape == (0, 8)


def test_embedding_reads_strided_rows(K):
    wide, grads = rand(60, 50, seed=1, dtype=BF16), rand(4, 30, 2, 41, seed=2, dtype=BF16)
    tokens = ints(60, 30, 4, seed=3).t()
    for off in (0, 1, 7):
        table, g = wide[:, off:off + 41], grads[:, :, 1, :]
        assert torch.equal(K.embedding(tokens, table), table[tokens])
        assert torch.equal(K.embedding_backward(g, tokens, 60), K.embedding_backward(g.contiguous(), tokens.contiguous(), 60))


def test_embedding_refuses(K):
    table, tokens, g = rand(10, 8, seed=1), ints(10, 6, seed=2), rand(6, 8, seed=3)
    for call in (lambda: K.embedding(tokens, table[0]), lambda: K.embedding(tokens, table[:, :0]), lambda: K.embedding_backward(g[:5], tokens, 10),
                 lambda: K.embedding_backward(g, tokens, -1), lambda: K.embedding_backward(g, tokens, 10, padding_idx=10), lambda: K.embedding_backward(g, tokens, 10, padding_idx=-11),
                 lambda: K.embedding_backward(g, tokens, 10, out=table[:9]), lambda: K.embedding_backward(g, tokens, 10, out=rand(8, 10, seed=4).t())):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: K.embedding(tokens.float(), table), lambda: K.embedding(tokens.short(), table), lambda: K.embedding(tokens, table.double()),
                 lambda: K.embedding(tokens, table, out_dtype=BF16), lambda: K.embedding_backward(g, tokens, 10, dtype=torch.float64),
                 lambda: K.embedding_backward(g, tokens, 10, out=table, dtype=BF16), lambda: K.embedding_backward(g.double(), tokens, 10)):
        with pytest.raises(TypeError):
            call()
    for call in (lambda: K.embedding(tokens.cpu(), table), lambda: K.embedding(tokens, table.cpu()), lambda: K.embedding_backward(g.cpu(), tokens, 10)):
        with pytest.raises(RuntimeError, match='ROCm device'):
            call()
    assert torch.equal(K.embedding_backward(g, tokens, 10, padding_idx=-1), K.embedding_backward(g, tokens, 10, padding_idx=9))


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('rows', [300001, 1048577])
def test_embedding_of_many_rows(K, rows, dtype):
    """With and without many tokens being brought into ranges of rows first."""
    width = 8
    for tokens in (20000, 70001):
        print(f'embedding {tokens} of {rows}x{width} {dtype}', flush=True)
        at = ints(rows, tokens, seed=tokens)
        at[::1000] = rows - 1
        check_embedding(K, at, rand(rows, width, seed=1, dtype=dtype), 1.5, None, rand(tokens, width, seed=2, dtype=dtype))


# ------------------------------------------------------------------------------------------------ offsets beyond 32 bits
def ends(n, k):
    """Positions at both ends of n, in order."""
    return torch.cat([torch.arange(k, device='cuda'), n - k + torch.arange(k, device='cuda')])


def test_linear_cross_entropy_of_very_many_rows(K):
    """h of more than 2^32 bytes: only rows at both ends have a gradient."""
    rows, width, classes = 2200001, 1000, 70
    print(f'linear_cross_entropy {rows}x{classes}x{width}', flush=True)
    h = rand(rows, width, seed=1, dtype=BF16)
    w, b = rand(classes, width, seed=2, dtype=BF16, scale=0.05), rand(classes, seed=3, dtype=BF16)
    t, at = ints(classes, rows, seed=4), ends(rows, 300)
    g = torch.zeros(rows, device='cuda')
    g[at] = gradient_of('none', t[at], 6)
    loss, lse = K.linear_cross_entropy(h, w, t, b, reduction='none')
    dh, dw, db = K.linear_cross_entropy_backward(g, h, w, t, lse, b, reduction='none')
    want = loss64(h[at], w, t[at], b, reduction='none', g=g[at])
    for name, got in (('lse', lse[at]), ('loss', loss[at]), ('dh', dh[at]), ('dw', dw), ('db', db)):
        within(got, *want[name], name)
    assert bool((dh[300:-300].view(-1) == 0).all())


def test_embedding_of_very_large_tables(K):
    """A table, and gradients, of more than 2^32 elements."""
    rows, width = 4300001, 1000
    print(f'embedding of {rows}x{width}', flush=True)
    table = torch.zeros(rows, width, device='cuda', dtype=BF16)
    at = ends(rows, 500)
    table[at] = rand(len(at), width, seed=2, dtype=BF16)
    tokens = at[ints(len(at), 20000, seed=3)]
    assert torch.equal(K.embedding(tokens, table), table[tokens])
    g = rand(20000, width, seed=4, dtype=BF16)
    got = K.embedding_backward(g, tokens, rows)
    few = torch.searchsorted(at, tokens)
    assert torch.equal(got[at], K.embedding_backward(g, few, len(at)))
    got[at] = 0
    assert bool((got == 0).all())
    del got, table
    print(f'embedding of {rows} tokens', flush=True)
    small = rand(700, width, seed=5, dtype=BF16)
    tokens = ints(700, rows, seed=6)
    assert torch.equal(K.embedding(tokens, small)[-500:], small[tokens[-500:]])
    g = torch.zeros(rows, width, device='cuda', dtype=BF16)
    g[at] = rand(len(at), width, seed=7, dtype=BF16)
    want = torch.zeros(700, width, dtype=torch.float64, device='cuda').index_add_(0, tokens[at], g[at].double())
    size = torch.zeros(700, width, dtype=torch.float64, device='cuda').index_add_(0, tokens[at], g[at].double().abs())
    within(K.embedding_backward(g, tokens, 700), want, 20 * U * size + half_step(BF16) * want.abs(), 'gradient')     # (at most 16 of a row's are not zero)
    assert int(torch.bincount(tokens[at]).max()) <= 16


def test_activations_of_very_many_rows_are_kept(K):
    """Codes of more than 2^32 bytes."""
    rows, width, out = 4300001, 1000, 24
    print(f'quantize_8bit {rows}x{width}', flush=True)
    x = torch.zeros(rows, width, device='cuda', dtype=BF16)
    at = ends(rows, 500)
    x[at] = rand(len(at), width, seed=1, dtype=BF16)
    kept, few = K.quantize_8bit(x), K.quantize_8bit(x[at])
    assert torch.equal(kept.codes.view(torch.uint8)[at], few.codes.view(torch.uint8)) and torch.equal(kept.exponents[at], few.exponents)
    assert torch.equal(K.dequantize_8bit(kept, BF16)[at], K.dequantize_8bit(few, BF16))
    y, also = K.gelu_8bit(x)
    assert torch.equal(y[at], K.gelu_8bit(x[at])[0]) and torch.equal(also.codes.view(torch.uint8)[at], few.codes.view(torch.uint8))
    del also
    assert torch.equal(K.gelu_8bit_backward(y, kept)[at], K.gelu_8bit_backward(y[at], few))
    del y, x
    g = torch.zeros(rows, out, device='cuda', dtype=BF16)
    g[at] = rand(len(at), out, seed=2, dtype=BF16)
    dw, db = K.weight_grad_8bit(g, kept, dtype=F32)
    values, gd = K.dequantize_8bit(few).double(), g[at].double()
    within(dw, gd.t() @ values, 2 * (len(at) + 8) * U * (gd.abs().t() @ values.abs()), 'dw')
    within(db, gd.sum(0), (len(at) + 8) * U * gd.abs().sum(0), 'db')


# ------------------------------------------------------------------------------------------------ activations in 8 bits
def e4m3_values():
    """The non-negative e4m3 numbers in ascending order, from their definition."""
    tiny = [m * 2.0 ** -9 for m in range(8)]
    return torch.tensor(tiny + [(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8) if (e, m) != (8, 7)], dtype=torch.float64, device='cuda')


def kept64(x):
    """(values, exponents) by search in the list of numbers."""
    shape, F = x.shape, x.shape[-1]
    x = x.double().reshape(-1, F)
    values = e4m3_values()
    out, exps = torch.full_like(x, NAN), []
    for c in range(0, F, 128):
        part = x[:, c:c + 128]
        most = torch.where(part.isfinite(), part.abs(), 0.0).amax(1)
        e = torch.full_like(most, -127)
        for k in range(-127, 128):                 # the least that fits
            fits = most * 2.0 ** -k <= 448
            e = torch.where(fits & (e == -127) & (most * 2.0 ** 127 > 448) & (most * 2.0 ** -(k - 1) > 448), float(k), e)
        v = part.abs() * torch.exp2(-e)[:, None]
        above = torch.searchsorted(values, v.nan_to_num(posinf=0.0).contiguous()).clamp(max=len(values) - 1)
        low, high = values[(above - 1).clamp(min=0)], values[above]
        odd = ((above - 1) % 2 == 1)
        near = torch.where((v - low < high - v) | ((v - low == high - v) & ~odd), low, high)
        near = torch.where((e == 120)[:, None], near.clamp(max=240), near)       # (256 * 2^120 is no float32)
        out[:, c:c + 128] = torch.where(part.isfinite(), torch.copysign(near * torch.exp2(e)[:, None], part), NAN)
        exps.append(e)
    return out.reshape(shape), torch.stack(exps, 1).reshape(*shape[:-1], -1)


def check_kept(K, x):
    kept = K.quantize_8bit(x)
    values, exps = kept64(x)
    assert kept.codes.shape == x.shape and kept.codes.dtype == torch.float8_e4m3fn
    assert torch.equal(kept.exponents.double(), exps)
    got = K.dequantize_8bit(kept).double()
    assert bool(((got == values) | (got.isnan() & values.isnan())).all())
    for dtype in (BF16, F16):
        low = K.dequantize_8bit(kept, dtype)
        want = K.dequantize_8bit(kept).to(dtype)
        assert bool(((low == want) | (low.isnan() & want.isnan())).all())
    return kept, values


KEPT = [(1, 1), (1, 7), (3, 8), (5, 100), (17, 128), (9, 129), (64, 257), (33, 768), (1000, 1021), (2, 8192), (130, 2050)]


@pytest.mark.parametrize('dtype', [F32, BF16, F16])
@pytest.mark.parametrize('rows,width', KEPT)
def test_activations_are_kept_as_defined(K, rows, width, dtype):
    print(f'quantize_8bit {rows}x{width} {dtype}', flush=True)
    x = rand(rows, width, seed=rows + width, scale=3.0) * torch.exp2(ints(20, 1, width, seed=4) - 10)
    check_kept(K, x.to(dtype))


@pytest.mark.parametrize('dtype', [F32, BF16, F16])
def test_activations_of_every_size_are_kept(K, dtype):
    """Ties, powers of two, the largest and the smallest numbers of the type, zeros, infinities and NaN."""
    least, most = (-24, 16) if dtype == F16 else (-149, 128) if dtype == F32 else (-133, 128)
    powers = torch.exp2(torch.arange(least, most, device='cuda', dtype=torch.float64)).to(dtype)
    for x in (powers.view(-1, 1), torch.cat([powers, -powers]).view(2, -1), powers.view(-1, 1) * torch.tensor([1.0, 1.75, -1.8, 0.0], device='cuda').to(dtype),
              torch.full((2, 300), torch.finfo(dtype).max, device='cuda', dtype=dtype), torch.zeros(3, 130, device='cuda', dtype=dtype)):
        check_kept(K, x)
    values = e4m3_values()
    between = torch.cat([values, (values[1:] + values[:-1]) / 2, -(values[1:] + values[:-1]) / 2])
    x = torch.zeros(len(between), 128, device='cuda', dtype=torch.float64)
    x[:, 0], x[:, 1] = 448, between
    check_kept(K, (x * 2.0 ** -3).to(dtype))
    x = rand(8, 200, seed=1, dtype=dtype)
    x[1, 5], x[2, 7], x[3, 130], x[4] = INF, NAN, -INF, NAN
    kept, _ = check_kept(K, x)
    assert torch.equal(K.dequantize_8bit(kept)[5:], K.dequantize_8bit(K.quantize_8bit(x[5:])))


def gelu64(x, way):
    """(y, dy/dx)"""
    x = x.double()
    if way == 'none':
        below = 0.5 * torch.special.erfc(-x / math.sqrt(2))
        return x * below, below + x * torch.exp(-x * x / 2) / math.sqrt(2 * math.pi)
    k = math.sqrt(2 / math.pi)
    u = k * (x + 0.044715 * x ** 3)
    t = torch.tanh(u)
    return torch.nn.functional.gelu(x, approximate='tanh'), 0.5 * (1 + t) + 0.5 * x / torch.cosh(u) ** 2 * k * (1 + 3 * 0.044715 * x * x)


@pytest.mark.parametrize('way', ['none', 'tanh'])
@pytest.mark.parametrize('dtype', [F32, BF16, F16])
@pytest.mark.parametrize('rows,width', [(1, 1), (5, 100), (64, 257), (33, 768), (300, 4096)])
def test_gelu_with_its_input_in_8_bits(K, rows, width, dtype, way):
    print(f'gelu_8bit {rows}x{width} {dtype} {way}', flush=True)
    x, g = rand(rows, width, seed=rows, scale=2.5, dtype=dtype), rand(rows, width, seed=width, dtype=dtype)
    y, kept = K.gelu_8bit(x, way)
    want = gelu64(x, way)[0]
    tiny = 2.0 ** -25 if dtype == F16 else 0
    within(y, want, half_step(dtype) * want.abs() + 2.0 ** -20 * x.double().abs() + tiny, 'gelu')
    alone = K.quantize_8bit(x)
    assert torch.equal(kept.codes.view(torch.uint8), alone.codes.view(torch.uint8)) and torch.equal(kept.exponents, alone.exponents)
    values = K.dequantize_8bit(kept).double()
    dx = K.gelu_8bit_backward(g, kept, way)
    want = g.double() * gelu64(values, way)[1]
    within(dx, want, half_step(dtype) * want.abs() + 2.0 ** -20 * g.double().abs() * (1 + values.abs()) + tiny, 'its gradient')


def test_gelu_far_from_zero(K):
    """Large numbers of either sign, infinities and NaN."""
    x = torch.tensor([[100.0, -100.0, 1e30, -1e30, 13.0, -13.0, 0.0, -0.0]], device='cuda').t().contiguous()
    for way in ('none', 'tanh'):
        y, kept = K.gelu_8bit(x, way)
        want = torch.tensor([100.0, 0, 1e30, 0, 13.0, 0, 0, 0], device='cuda')[:, None]
        assert torch.allclose(y, want, rtol=1e-6, atol=1e-30), (way, y)
        dx = K.gelu_8bit_backward(torch.ones_like(x), kept, way)
        assert torch.allclose(dx, torch.tensor([1.0, 0, 1, 0, 1, 0, 0.5, 0.5], device='cuda')[:, None], atol=1e-6), (way, dx)
        y, kept = K.gelu_8bit(torch.tensor([[NAN]], device='cuda'), way)
        assert bool(y.isnan()) and bool(K.gelu_8bit_backward(torch.ones(1, 1, device='cuda'), kept, way).isnan())


WEIGHTS = [(1, 1, 1), (3, 8, 5), (40, 33, 70), (64, 128, 128), (100, 257, 136), (1000, 72, 300), (33, 1000, 520), (3000, 40, 24), (700, 768, 1030)]


@pytest.mark.parametrize('dtype', [F32, BF16, F16])
@pytest.mark.parametrize('rows,width,out', WEIGHTS)
def test_weight_gradients_from_kept_inputs(K, rows, width, out, dtype):
    print(f'weight_grad_8bit {rows}x{width}->{out} {dtype}', flush=True)
    x, g = rand(rows, width, seed=rows, dtype=dtype), rand(rows, out, seed=out, dtype=dtype)
    kept = K.quantize_8bit(x)
    values, gd = K.dequantize_8bit(kept).double(), g.double()
    for made in (dtype, F32):
        dw, db = K.weight_grad_8bit(g, kept, dtype=made)
        assert dw.dtype == db.dtype == made
        want = gd.t() @ values
        tiny = 2.0 ** -25 if made == F16 else 0
        within(dw, want, half_step(made) * want.abs() + 2 * (rows + 8) * U * (gd.abs().t() @ values.abs()) + tiny, 'dw')
        within(db, gd.sum(0), half_step(made) * gd.sum(0).abs() + (rows + 8) * U * gd.abs().sum(0) + tiny, 'db')
        again = K.weight_grad_8bit(g, kept, dtype=made)
        assert torch.equal(dw, again[0]) and torch.equal(db, again[1])
    none, alone = K.weight_grad_8bit(g, None, need_weight=False)
    assert none is None and torch.equal(alone, K.weight_grad_8bit(g, kept)[1])
    assert K.weight_grad_8bit(g, kept, need_bias=False)[1] is None and K.weight_grad_8bit(g, kept, need_weight=False)[0] is None


@pytest.mark.parametrize('dtype', [F32, BF16, F16])
def test_weight_gradients_of_strided_tensors(K, dtype):
    big, wide = rand(50, 4, 140, seed=1, dtype=dtype), rand(50, 4, 100, seed=2, dtype=dtype)
    x, g = big[:, 1:3, 5:133], wide[:, 2:, 3:75]
    kept = K.quantize_8bit(x)
    same = K.quantize_8bit(x.contiguous())
    assert torch.equal(kept.codes.view(torch.uint8), same.codes.view(torch.uint8)) and torch.equal(kept.exponents, same.exponents)
    assert all(torch.equal(a, b) for a, b in zip(K.weight_grad_8bit(g, kept), K.weight_grad_8bit(g.contiguous(), same)))


def test_weight_gradients_pass_nan_and_infinity_on(K):
    """In the columns they belong to."""
    for dtype in (F32, BF16, F16):
        x, g = rand(60, 40, seed=1, dtype=dtype), rand(60, 24, seed=2, dtype=dtype)
        x[3, 7], g[5, 2], g[6, 4] = NAN, NAN, INF
        dw, db = K.weight_grad_8bit(g, K.quantize_8bit(x))
        assert bool(dw[:, 7].isnan().all()) and bool(dw[2].isnan().all()) and not bool(dw[4, :7].isfinite().any())
        clean = torch.ones_like(dw, dtype=torch.bool)
        clean[:, 7], clean[2], clean[4] = False, False, False
        assert bool(dw[clean].isfinite().all())
        assert bool(db[2].isnan()) and float(db[4]) == INF


def test_8_bit_activations_of_nothing_and_refusals(K):
    kept = K.quantize_8bit(rand(0, 40, seed=1))
    assert kept.codes.shape == (0, 40) and K.dequantize_8bit(kept).shape == (0, 40)
    dw, db = K.weight_grad_8bit(rand(0, 6, seed=2), kept)
    assert torch.equal(dw, torch.zeros(6, 40, device='cuda')) and torch.equal(db, torch.zeros(6, device='cuda'))
    x, g = rand(5, 40, seed=3), rand(5, 6, seed=4)
    kept = K.quantize_8bit(x)
    for call in (lambda: K.gelu_8bit(x, 'fast'), lambda: K.gelu_8bit_backward(g, kept), lambda: K.weight_grad_8bit(g[:4], kept), lambda: K.quantize_8bit(x[:, :0]),
                 lambda: K.dequantize_8bit((kept.codes, kept.exponents[:, :0])), lambda: K.dequantize_8bit((kept.codes.view(torch.uint8), kept.exponents)),
                 lambda: K.weight_grad_8bit(g, K.Quantized8(kept.codes[:, :30], kept.exponents))):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: K.quantize_8bit(x.double()), lambda: K.dequantize_8bit(kept, torch.float64), lambda: K.weight_grad_8bit(g, kept, dtype=torch.float64),
                 lambda: K.weight_grad_8bit(g.double(), kept)):
        with pytest.raises(TypeError):
            call()
    for call in (lambda: K.quantize_8bit(x.cpu()), lambda: K.weight_grad_8bit(g.cpu(), kept), lambda: K.dequantize_8bit(K.Quantized8(kept.codes.cpu(), kept.exponents.cpu()))):
        with pytest.raises(RuntimeError, match='ROCm device'):
            call()


# ------------------------------------------------------------------------------------------------ together
def program(K, seed, rows=300, classes=1500, width=96, dtype=BF16):
    """A step's calls around a block: lookup, activation, weight gradient, loss and all gradients, the table's added to the head's."""
    inputs = dict(tokens=ints(classes, rows, seed=seed), targets=ints(classes, rows, seed=seed + 1), table=rand(classes, width, seed=seed + 2, dtype=dtype),
                  weight=rand(width, width, seed=seed + 3, dtype=dtype, scale=0.1))

    def run():
        x = K.embedding(inputs['tokens'], inputs['table'], 2.0)
        kept = K.quantize_8bit(x)
        y, inner = K.gelu_8bit(x)
        loss, lse = K.linear_cross_entropy(y, inputs['table'], inputs['targets'])
        dy, dtable, _ = K.linear_cross_entropy_backward(torch.ones_like(loss), y, inputs['table'], inputs['targets'], lse)
        dx = K.gelu_8bit_backward(dy, inner)
        dw, db = K.weight_grad_8bit(dx, kept)
        K.embedding_backward(dx, inputs['tokens'], classes, 2.0, out=dtable, beta=1.0)
        return [x, y, loss, lse, dy, dx, dw, db, dtable]
    return inputs, run


def test_decoder_ends_run_on_the_current_stream(K):
    inputs, run = program(K, 1)
    want = run()
    torch.cuda.synchronize()
    table = inputs['table'].clone()
    inputs['table'].zero_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = torch.zeros(4096, 4096, device='cuda')
        for _ in range(20):
            a = a @ a
        inputs['table'].copy_(table + a[0, 0].to(BF16))
        got = run()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize('dtype', [BF16, F32])
def test_decoder_ends_in_two_captured_graphs(K, dtype):
    made = []
    for seed in (1, 20):
        inputs, run = program(K, seed, dtype=dtype)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = run()
        made.append((inputs, run, graph, outs, side))
    for turn in range(4):
        for inputs, _, _, outs, _ in made:
            inputs['table'].mul_(0.9)
            inputs['tokens'].copy_(inputs['tokens'].roll(1) // 2)
            inputs['targets'].copy_(inputs['targets'].roll(2))
            for o in outs:
                o.zero_()
        torch.cuda.synchronize()
        for _, _, graph, _, side in made:
            with torch.cuda.stream(side):
                graph.replay()
        torch.cuda.synchronize()
        for _, run, _, outs, _ in made:
            got = [o.clone() for o in outs]
            assert all(torch.equal(a, b) for a, b in zip(got, run())), turn


def test_decoder_ends_from_two_threads(K):
    import threading
    made = [program(K, seed) for seed in (1, 50)]
    want = [run() for _, run in made]
    torch.cuda.synchronize()
    wrong, errors = [], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for turn in range(40):
                    got = made[i][1]()
                    torch.cuda.current_stream().synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                        wrong.append((i, turn))
        except Exception as e:
            errors.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors and not wrong
