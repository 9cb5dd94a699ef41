"""Layer norm (with its gradients and Fisher blocks), filtered draws and the norm of all gradients against their definitions in 64 bits.

Tolerances.  u = 2^-24 is half a step of float32.
Layer norm: the mean of n terms is off by at most (n/64 + 8) u mean|x| (64 lanes add n / 64 terms each, then 6 + 4 levels), which enters h
through r; the mean square likewise, halved by the root.  With data whose mean is not much larger than its deviation all of it stays below
40 u for n <= 8192 in the root mean square, whose random roundings grow like sqrt(n / 64); 64 u is allowed in the 2-norm, then half a step
of the type that is stored.  Sums over rows: fp32 chains of at most 256 terms, joined by at most 32: random roundings of sqrt(288) u, 64 u
again of the sum of magnitudes, i.e. relative to sqrt(sum of squares) of the terms.
The norm of gradients: sums are double, the result is rounded to float32 once, and the factor and the product once each: 4 u.
Draws are whole numbers and equal."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = 2.0 ** -24
NORM_TOL = 64 * U


@pytest.fixture(scope='module')
def K():
    from asdl_amd import kernels
    return kernels


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def off(got, want, magnitude=None):
    """The 2-norm of the difference relative to that of ``magnitude`` (the terms behind a sum; the result itself otherwise)."""
    want = want.double()
    scale = (want if magnitude is None else magnitude.double()).norm()
    return float((got.detach().double() - want).norm() / scale.clamp_min(1e-300))


def rand(*shape, seed, dtype=F32, scale=1.0, shift=0.0):
    gen = torch.Generator('cuda').manual_seed(seed)
    return (torch.randn(shape, device='cuda', generator=gen) * scale + shift).to(dtype)


# ------------------------------------------------------------------------------------------------ layer norm
def norm64(x, w, b, eps):
    x = x.double()
    m = x.mean(-1, keepdim=True)
    v = (x - m).square().mean(-1, keepdim=True)
    r = (v + eps).rsqrt()
    h = (x - m) * r
    y = h if w is None else h * w.double()
    return (y if b is None else y + b.double()), m.squeeze(-1), r.squeeze(-1), h


def norm64_backward(g, w, r, h):
    g = g.double()
    gw = g if w is None else g * w.double()
    dx = r.unsqueeze(-1) * (gw - gw.mean(-1, keepdim=True) - h * (gw * h).mean(-1, keepdim=True))
    g, h = g.reshape(-1, g.shape[-1]), h.reshape(-1, h.shape[-1])
    gh = g * h
    blocks = torch.stack([(gh * gh).sum(0), (gh * g).sum(0), (gh * g).sum(0), (g * g).sum(0)], -1).view(-1, 2, 2)
    # for the sums over rows: the root of the sum of squares of the terms
    return dx, gh.sum(0), g.sum(0), blocks, gh.square().sum(0).sqrt(), g.square().sum(0).sqrt()


def check_norm(K, x, w, b, g, eps, out_dtype=None, with_blocks=True, strict_dx=True):
    y, mean, rstd = K.layer_norm(x, w, b, eps, out_dtype=out_dtype)
    ry, rm, rr, rh = norm64(x, w, b, eps)
    assert y.dtype == (out_dtype or x.dtype) and y.shape == x.shape and mean.shape == x.shape[:-1]
    assert off(y, ry) < NORM_TOL + half_step(y.dtype)
    assert off(mean, rm, x.double().abs().mean(-1)) < NORM_TOL and off(rstd, rr) < NORM_TOL
    F = x.shape[-1]
    blocks = rand(F, 2, 2, seed=5) if with_blocks else None
    before = blocks.clone() if with_blocks else None
    dx, dw, db = K.layer_norm_backward(g, x, mean, rstd, w, blocks=blocks, alpha=0.25, beta=0.5)
    rdx, rdw, rdb, rblocks, mw, mb = norm64_backward(g, w, rr, rh)
    wt = w.dtype if w is not None else F32
    assert dx.dtype == x.dtype and dx.shape == x.shape and dw.dtype == db.dtype == wt
    gw = (g.double() if w is None else g.double() * w.double()) * rr.unsqueeze(-1)
    assert off(dx, rdx, None if strict_dx else gw) < NORM_TOL + half_step(x.dtype)
    assert off(dw, rdw, mw + rdw.abs()) < NORM_TOL + half_step(wt) and off(db, rdb, mb + rdb.abs()) < NORM_TOL + half_step(wt)
    if with_blocks:
        want = 0.5 * before.double() + 0.25 * rblocks
        assert off(blocks, want, 0.5 * before.double().abs() + 0.25 * rblocks.abs()) < NORM_TOL
        assert torch.equal(blocks[:, 0, 1], blocks[:, 1, 0]) or bool((before[:, 0, 1] != before[:, 1, 0]).any())
    return y, mean, rstd, dx, dw, db


SIZES = [(1, 16), (3, 17), (1, 768), (70, 64), (257, 100), (33, 511), (5, 1021), (300, 768), (65, 1536), (19, 2050), (9, 4096), (6, 8191), (3, 16400)]


@pytest.mark.parametrize('rows,F', SIZES)
@pytest.mark.parametrize('xt,yt,wt', [(F32, F32, F32), (BF16, BF16, BF16), (BF16, F32, F32), (F16, F16, F32), (F16, F32, F16), (BF16, BF16, F32)])
def test_layer_norm_matches_its_definition(K, rows, F, xt, yt, wt):
    print(f'layer_norm {rows}x{F} {xt} {yt} {wt}', flush=True)
    x = rand(rows, F, seed=rows + F, dtype=xt, scale=2.0, shift=0.5)
    w, b = rand(F, seed=1, dtype=wt, scale=0.2, shift=1.0), rand(F, seed=2, dtype=wt)
    g = rand(rows, F, seed=3, dtype=yt)
    check_norm(K, x, w, b, g, 1e-5, out_dtype=yt)


@pytest.mark.parametrize('weight,bias', [(False, False), (True, False), (False, True)])
def test_layer_norm_without_weight_or_bias(K, weight, bias):
    x, g = rand(40, 300, seed=1), rand(40, 300, seed=2)
    check_norm(K, x, rand(300, seed=3) if weight else None, rand(300, seed=4) if bias else None, g, 1e-6)


def test_layer_norm_many_rows(K):
    x, g = rand(20011, 96, seed=1, dtype=BF16), rand(20011, 96, seed=2, dtype=BF16)
    check_norm(K, x, rand(96, seed=3), rand(96, seed=4), g, 1e-5)


@pytest.mark.parametrize('F', [1, 2, 3, 5, 8, 15])
def test_layer_norm_of_few_features(K, F):
    """h of one feature is 0 and of two +-1 up to eps: dx is a difference that nearly vanishes, so its error counts against what it is
    the difference of."""
    x, g = rand(200, F, seed=F, scale=3.0), rand(200, F, seed=9)
    check_norm(K, x, rand(F, seed=3), rand(F, seed=4), g, 1e-3, strict_dx=False)


def test_layer_norm_of_equal_and_of_large_values(K):
    x = torch.full((4, 300), 7.25, device='cuda')
    x[1] = 0
    x[2] = 1e18
    y, mean, rstd = K.layer_norm(x, None, rand(300, seed=1), 1e-5)
    assert torch.equal(y, rand(300, seed=1).expand(4, 300)) and torch.equal(mean, x[:, 0])
    assert off(rstd, torch.full((4,), 1e-5, device='cuda', dtype=torch.float64).rsqrt()) < 4 * U
    # a deviation far below the mean: 2^-12 of it, so the mean's rounding (64 u of it) is 2^12 * 64 u of the deviation
    z = 4096 + rand(50, 768, seed=2)
    assert off(K.layer_norm(z)[0], norm64(z, None, None, 1e-5)[0]) < 4096 * NORM_TOL
    # large and small scales keep their digits (eps = 0)
    for scale in (1e-15, 1e15):
        z = rand(50, 768, seed=3) * scale
        assert off(K.layer_norm(z, eps=0.0)[0], norm64(z, None, None, 0.0)[0]) < NORM_TOL


def test_layer_norm_passes_nan_and_infinity_on_in_their_row_alone(K):
    x = rand(9, 200, seed=1)
    x[3, 5], x[6, 199] = float('nan'), float('inf')
    y, mean, rstd = K.layer_norm(x)
    bad = torch.isnan(y).all(1)
    assert bad.tolist() == [i in (3, 6) for i in range(9)]
    assert bool(torch.isfinite(y[~bad]).all())
    g = rand(9, 200, seed=2)
    dx = K.layer_norm_backward(g, x, mean, rstd, need_weight=False, need_bias=False)[0]
    assert torch.isnan(dx).all(1).tolist() == bad.tolist() and bool(torch.isfinite(dx[~bad]).all())


def test_layer_norm_reads_strided_rows_and_any_alignment(K):
    wide = rand(3, 50, 1100, seed=1)
    for x in (wide[:, ::2, 3:1024], wide[..., 1:770], wide[1:2, :, 5:6], wide.transpose(0, 1)[..., :768], wide[0, :1].expand(50, 1100)):
        g = rand(3, 50, 1101, seed=2)[..., 1:][:x.shape[0], :, :x.shape[-1]] if x.ndim == 3 else rand(50, 1100, seed=2)
        g = g[:, :x.shape[1]] if x.ndim == 3 else g
        g = g.expand(x.shape) if g.shape != x.shape and g.shape[0] == 1 else g
        if g.shape != x.shape:
            g = rand(*x.shape, seed=4)
        F = x.shape[-1]
        check_norm(K, x, rand(F, seed=3), rand(F, seed=4), g, 1e-3, strict_dx=False)
    # a gradient that is one number for all (a mean's): stride 0 everywhere
    x = rand(30, 70, seed=5)
    _, mean, rstd = K.layer_norm(x)
    got = K.layer_norm_backward(torch.ones((), device='cuda').expand(30, 70), x, mean, rstd)
    want = K.layer_norm_backward(torch.ones(30, 70, device='cuda'), x, mean, rstd)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_layer_norm_of_no_rows(K):
    x = torch.empty(0, 64, device='cuda')
    y, mean, rstd = K.layer_norm(x, torch.ones(64, device='cuda'))
    blocks = torch.ones(64, 2, 2, device='cuda')
    dx, dw, db = K.layer_norm_backward(x, x, mean, rstd, blocks=blocks, alpha=1.0, beta=0.5)
    assert y.shape == dx.shape == (0, 64) and mean.shape == (0,)
    assert not dw.any() and not db.any() and bool((blocks == 0.5).all())
    K.layer_norm_backward(x, x, mean, rstd, blocks=blocks, beta=0.0)
    assert not blocks.any()


def test_layer_norm_gives_what_is_asked_for(K):
    x, g = rand(100, 768, seed=1), rand(100, 768, seed=2)
    w = rand(768, seed=3)
    _, mean, rstd = K.layer_norm(x, w)
    full = K.layer_norm_backward(g, x, mean, rstd, w)
    for mask in range(8):
        need = [bool(mask & 1), bool(mask & 2), bool(mask & 4)]
        got = K.layer_norm_backward(g, x, mean, rstd, w, need_x=need[0], need_weight=need[1], need_bias=need[2])
        for a, b, n in zip(got, full, need):
            assert (a is None) == (not n) and (a is None or torch.equal(a, b))
    # beta = 0 does not read the blocks; the same call twice has the same bits
    blocks = torch.full((768, 2, 2), float('nan'), device='cuda')
    K.layer_norm_backward(g, x, mean, rstd, w, blocks=blocks, need_x=False, need_weight=False, need_bias=False)
    again = torch.zeros(768, 2, 2, device='cuda')
    K.layer_norm_backward(g, x, mean, rstd, w, blocks=again)
    assert torch.equal(blocks, again) and bool(torch.isfinite(again).all())


def test_layer_norm_blocks_are_unit_wise_stats(K):
    x, g = rand(333, 768, seed=1), rand(333, 768, seed=2)
    w, b = rand(768, seed=3, scale=0.2, shift=1.0), rand(768, seed=4)
    y, mean, rstd = K.layer_norm(x, w, b)
    blocks = torch.zeros(768, 2, 2, device='cuda')
    K.layer_norm_backward(g, x, mean, rstd, w, blocks=blocks, alpha=1 / 333)
    # (y - b) / w loses digits where b is large against h w: up to |y| / |h w| more than h itself
    assert off(blocks, K.unit_wise_stats(y, g, w, b, alpha=1 / 333)) < 4 * NORM_TOL


def test_layer_norm_refuses(K):
    x, w = rand(4, 64, seed=1), rand(64, seed=2)
    _, mean, rstd = K.layer_norm(x)
    for call, kind in [(lambda: K.layer_norm(x.double()), TypeError), (lambda: K.layer_norm(x, w[:63]), ValueError),
                       (lambda: K.layer_norm(x, w, w.bfloat16()), TypeError), (lambda: K.layer_norm(x, w.bfloat16()), TypeError), (lambda: K.layer_norm(x, eps=-1e-5), ValueError),
                       (lambda: K.layer_norm(x, eps=float('nan')), ValueError), (lambda: K.layer_norm(x, out_dtype=F16), TypeError),
                       (lambda: K.layer_norm(x.bfloat16(), out_dtype=F16), TypeError), (lambda: K.layer_norm(x[:, :0]), ValueError),
                       (lambda: K.layer_norm(x[0, 0]), ValueError), (lambda: K.layer_norm(x, w.cpu()), RuntimeError),
                       (lambda: K.layer_norm_backward(x[:3], x, mean, rstd), ValueError),
                       (lambda: K.layer_norm_backward(x.bfloat16(), x, mean, rstd), TypeError),
                       (lambda: K.layer_norm_backward(x, x, mean[:3], rstd), ValueError),
                       (lambda: K.layer_norm_backward(x, x, mean.double(), rstd), ValueError),
                       (lambda: K.layer_norm_backward(x, x, mean, rstd, blocks=torch.zeros(64, 4, device='cuda')), ValueError),
                       (lambda: K.layer_norm_backward(x, x, mean, rstd, weight_dtype=torch.int32), TypeError)]:
        with pytest.raises(kind):
            call()


# ------------------------------------------------------------------------------------------------ filtered draws
def draw64(logits, u, temperature=1.0, top_k=None, top_p=None, min_p=None):
    """The definition, row by row, in extended precision on the host.  Also says how near the nearest border was (relative to the sums
    that meet there): a draw is pinned where that is far from 2^-40."""
    rows, n = logits.shape
    x = logits.double().cpu().numpy().astype(np.longdouble)
    u = u.double().cpu().numpy()

    def each(v, default):
        return v.double().cpu().numpy() if torch.is_tensor(v) else np.full(rows, default if v is None else v, dtype=np.float64)
    ts, ks, ps, ms = each(temperature, 1), each(top_k, 0), each(top_p, 1), each(min_p, 0)
    out = []
    for r in range(rows):
        if np.isnan(x[r]).any() or (x[r] == np.inf).any() or (x[r] == -np.inf).all():
            out.append(-1)
            continue
        order = np.lexsort((np.arange(n), -x[r]))
        if ts[r] == 0:
            out.append(int(order[0]))
            continue
        if ks[r] > 0:
            order = order[:int(ks[r])]
        w = np.exp((x[r][order] - x[r][order[0]]) / ts[r])
        keep = np.ones(len(order), bool)
        if ps[r] < 1:
            before = np.concatenate([[0], np.cumsum(w)[:-1]])
            keep = before < ps[r] * w.sum()
        keep &= w >= min(ms[r], 1)
        keep[0] = True
        at = order[keep]
        by_index = np.argsort(at)
        upto = np.cumsum(w[keep][by_index])
        i = min(int(np.searchsorted(upto, u[r] * upto[-1], side='right')), len(at) - 1)
        out.append(int(at[by_index][i]))
    return torch.tensor(out)


FILTERS = [dict(), dict(temperature=0.7), dict(top_k=5), dict(top_p=0.6), dict(min_p=0.1), dict(temperature=1.3, top_k=40, top_p=0.9, min_p=0.01),
           dict(temperature=0.0), dict(top_k=1), dict(top_p=0.0), dict(top_p=1.0, min_p=1.0), dict(temperature=0.05, top_p=0.95),
           dict(top_k=10 ** 9, top_p=0.999)]


@pytest.mark.parametrize('dtype', [F32, BF16, F16])
@pytest.mark.parametrize('rows,n', [(1, 1), (5, 2), (64, 10), (7, 257), (40, 1000), (9, 2047), (9, 2049), (6, 5003), (3, 50257), (2, 131072)])
def test_filtered_draws_match_their_definition(K, dtype, rows, n):
    print(f'sample_filtered {rows}x{n} {dtype}', flush=True)
    logits = rand(rows, n, seed=rows + n, dtype=dtype, scale=2.5)
    for i, filters in enumerate(FILTERS):
        u = torch.rand(rows, device='cuda', dtype=torch.float64, generator=torch.Generator('cuda').manual_seed(i))
        assert torch.equal(K.sample_filtered(logits, u, **filters).cpu(), draw64(logits, u, **filters)), filters


@pytest.mark.parametrize('n', [100, 3000, 20000])
def test_filtered_draws_with_parameters_for_every_row(K, n):
    rows = 61
    gen = torch.Generator('cuda').manual_seed(n)

    def pick(values, dtype=F32):
        return torch.tensor(values, device='cuda', dtype=dtype)[torch.randint(0, len(values), (rows,), device='cuda', generator=gen)]
    logits = rand(rows, n, seed=1, dtype=BF16, scale=3.0)
    u = torch.rand(rows, device='cuda', generator=gen)
    filters = dict(temperature=pick([0.0, 0.3, 1.0, 2.0]), top_k=pick([-1, 0, 1, 2, 50, 10 ** 6], torch.int64), top_p=pick([0.0, 0.1, 0.5, 0.9, 1.0, 2.0]),
                   min_p=pick([-1.0, 0.0, 0.05, 0.5, 1.0, 3.0]))
    assert torch.equal(K.sample_filtered(logits, u, **filters).cpu(), draw64(logits, u, **filters))


@pytest.mark.parametrize('n', [64, 1024, 4096, 50000])
def test_filtered_draws_take_the_lowest_of_equal_classes(K, n):
    """Equal logits: every sum is a whole number of equal weights, so the borders are met exactly."""
    logits = torch.zeros(1, n, device='cuda')
    logits[0, ::2] = -0.0
    u0, u1 = torch.zeros(1, device='cuda', dtype=torch.float64), torch.full((1,), 1 - 2.0 ** -53, device='cuda', dtype=torch.float64)
    for k in (1, 2, n // 2, n - 1, n):
        assert int(K.sample_filtered(logits, u0, top_k=k)) == 0 and int(K.sample_filtered(logits, u1, top_k=k)) == k - 1
    for p in (0.25, 0.5):
        assert int(K.sample_filtered(logits, u1, top_p=p)) == int(p * n) - 1
        assert int(K.sample_filtered(logits, u1, top_p=p, top_k=n // 2)) == int(p * (n // 2)) - 1
    assert int(K.sample_filtered(logits, u1)) == n - 1 and int(K.sample_filtered(logits, u1, temperature=0.0)) == 0
    half = torch.full((1,), 0.5, device='cuda')
    assert int(K.sample_filtered(logits, half)) == n // 2
    # two levels: n/4 - 1 classes of 0 (all below n/4 but class 3), and of the classes of -1, which are 3, n/4, n/4 + 1, ..., three or one
    logits[0, n // 4:] = -1.0
    logits[0, 3] = -1.0
    assert int(K.sample_filtered(logits, u1, top_k=n // 4 + 2)) == n // 4 + 1
    assert int(K.sample_filtered(logits, u1, top_k=n // 4)) == n // 4 - 1
    assert int(K.sample_filtered(logits, u1, min_p=0.5)) == n // 4 - 1


def test_filtered_draws_leave_masked_classes_out(K):
    n = 6001
    logits = rand(64, n, seed=1)
    mask = torch.rand(64, n, device='cuda', generator=torch.Generator('cuda').manual_seed(2)) < 0.9
    logits[mask] = -float('inf')
    logits[5] = -float('inf')
    logits[5, 77] = -3.0                       # one class is left
    logits[6] = torch.finfo(F32).min           # masks of the type's lowest value are numbers
    u = torch.rand(64, device='cuda')
    for filters in (dict(), dict(top_k=3), dict(top_k=4000), dict(top_p=0.5), dict(top_p=0.9999), dict(min_p=1e-6), dict(temperature=50.0)):
        got = K.sample_filtered(logits, u, **filters)
        assert torch.equal(got.cpu(), draw64(logits, u, **filters)), filters
        assert int(got[5]) == 77
    wide = torch.tensor([[3e38, -3e38, 0.0, 2.9e38]], device='cuda')       # differences beyond float32
    assert int(K.sample_filtered(wide, torch.full((1,), 0.999, device='cuda'))) == 0


@pytest.mark.parametrize('n', [10, 5000])
def test_filtered_draws_mark_rows_without_a_distribution(K, n):
    logits = rand(8, n, seed=1)
    logits[1, 3], logits[2, n - 1], logits[3] = float('nan'), float('inf'), -float('inf')
    u = torch.full((8,), 0.5, device='cuda')
    want = draw64(logits, u)
    assert want[1:4].tolist() == [-1] * 3
    assert torch.equal(K.sample_filtered(logits, u, check=False).cpu(), want)
    with pytest.raises(RuntimeError, match='probability tensor'):
        K.sample_filtered(logits, u)
    targets, drawn = K.sample_filtered(logits, u, late=True)
    with pytest.raises(RuntimeError, match='probability tensor'):
        drawn.check()
    assert torch.equal(targets.cpu(), want)
    clean = rand(8, n, seed=1)
    nan = torch.tensor([1.0, float('nan')] * 4, device='cuda')
    for filters in (dict(temperature=nan), dict(top_p=nan), dict(min_p=nan), dict(temperature=-nan)):
        got = K.sample_filtered(clean, u, check=False, **filters)
        assert bool((got[1::2] == -1).all())
        assert bool((got[0::2] >= 0).all()) or 'temperature' in filters
    assert K.sample_filtered(clean, nan, check=False).tolist()[1::2] == [-1] * 4
    assert K.sample_filtered(clean, torch.full((8,), 5.0, device='cuda')).tolist() == [n - 1] * 8       # numbers outside [0, 1): the ends
    assert K.sample_filtered(clean, torch.full((8,), -5.0, device='cuda')).tolist() == [0] * 8
    K.sample_filtered(clean, u)                # the word is clear again


def test_filtered_draws_of_strided_logits(K):
    wide = rand(4, 9, 5003, seed=1, dtype=BF16)
    u = torch.rand(4, 9, device='cuda', dtype=torch.float64)
    for cut in (slice(0, 5000), slice(1, 5000), slice(3, 1026)):
        logits = wide[:, :, cut]
        got = K.sample_filtered(logits, u, top_p=0.8)
        assert got.shape == (4, 9) and torch.equal(got.cpu().flatten(), draw64(logits.flatten(0, 1), u.flatten(), top_p=0.8))
    last = wide[:, -1]
    assert torch.equal(K.sample_filtered(last, u[:, 0], top_k=50).cpu(), draw64(last, u[:, 0], top_k=50))
    one = wide[0, 0]
    assert K.sample_filtered(one, u[0, 0], top_k=7).shape == () and int(K.sample_filtered(one, u[0, 0], top_k=7)) == int(draw64(one[None], u[0, :1], top_k=7))
    assert K.sample_filtered(wide[:0, 0], u[:0, 0]).shape == (0,)
    turned = rand(300, 40, seed=2).t()
    assert torch.equal(K.sample_filtered(turned, u.flatten()[:1].expand(40)).cpu(), draw64(turned, u.flatten()[:1].expand(40)))


def test_filtered_draws_follow_the_distribution(K):
    """Without numbers of its own the call draws them: frequencies over 2^18 draws of 8 classes, 6 standard deviations."""
    logits = torch.tensor([1.0, 0.0, 2.0, -1.0, 0.5, -9.0, 1.5, 0.0], device='cuda')
    p = torch.softmax(logits.double(), 0)
    p[[0, 1, 3, 4, 5, 7]] = 0
    n = 1 << 18
    torch.manual_seed(1)
    got = torch.bincount(K.sample_filtered(logits.expand(n, 8).contiguous(), top_k=2), minlength=8).double() / n
    p /= p.sum()
    assert bool(((got - p).abs() <= 6 * (p * (1 - p) / n).sqrt()).all())


def test_filtered_draws_refuse(K):
    logits, u = rand(4, 50, seed=1), torch.rand(4, device='cuda')
    for call, kind in [(lambda: K.sample_filtered(logits.double(), u), TypeError), (lambda: K.sample_filtered(logits, u[:3]), ValueError),
                       (lambda: K.sample_filtered(logits, u.half()), ValueError), (lambda: K.sample_filtered(logits, u, temperature=-1.0), ValueError),
                       (lambda: K.sample_filtered(logits, u, temperature=float('nan')), ValueError),
                       (lambda: K.sample_filtered(logits, u, top_p=float('nan')), ValueError),
                       (lambda: K.sample_filtered(logits, u, top_p=u[:2]), ValueError), (lambda: K.sample_filtered(logits, u, top_k=u), ValueError),
                       (lambda: K.sample_filtered(logits, u, temperature=u.double()), ValueError),
                       (lambda: K.sample_filtered(logits, u, top_p=u.cpu()), RuntimeError), (lambda: K.sample_filtered(logits[:, :0], u), ValueError),
                       (lambda: K.sample_filtered(logits, u.cpu()), RuntimeError)]:
        with pytest.raises(kind):
            call()


# ------------------------------------------------------------------------------------------------ norm of all gradients
def norm_of(grads, kind):
    parts = [g.detach().double().flatten() for g in grads if g.numel()]
    if not parts:
        return 0.0
    if kind == 2:
        return math.sqrt(math.fsum(float(p @ p) for p in parts))
    return math.fsum(float(p.abs().sum()) for p in parts) if kind == 1 else max(float(p.abs().max()) for p in parts)


def gradients(shapes, seed, dtypes=(F32,)):
    return [rand(*s, seed=seed + i, dtype=dtypes[i % len(dtypes)], scale=10.0 ** (i % 4 - 2)) for i, s in enumerate(shapes)]


LISTS = [[(1,)], [(512, 784), (512,), (10, 512), (10,)], [(3, 5, 7), (0, 4), (), (16384,), (16385,), (16383,), (33, 1021)], [(7,)] * 400,
         [(64, 3, 7, 7), (1 << 22,), (1,), (1000003,)]]


@pytest.mark.parametrize('kind', [2, 1, float('inf')])
@pytest.mark.parametrize('dtypes', [(F32,), (BF16,), (F16, F32), (F32, BF16, F16)])
@pytest.mark.parametrize('which', range(len(LISTS)))
def test_norms_and_clipped_gradients(K, which, dtypes, kind):
    grads = gradients(LISTS[which], seed=which, dtypes=dtypes)
    print(f'grad_norm list {which} {dtypes} {kind}', flush=True)
    want = norm_of(grads, kind)
    assert abs(float(K.grad_norm(grads, kind)) - want) <= 2 * U * want
    for most in (want / 3, want * 3):
        factor = min(1.0, most / (want + 1e-6))
        outs = [torch.full_like(g, float('nan')) for g in grads]
        norm = K.clip_grad_norm(grads, most, kind, outs=outs)
        assert norm.shape == () and norm.dtype == F32 and abs(float(norm) - want) <= 2 * U * want
        inplace = [g.clone() for g in grads]
        assert torch.equal(K.clip_grad_norm(inplace, most, kind), norm)
        for g, o, i in zip(grads, outs, inplace):
            assert torch.equal(o, i)
            if most > want:
                assert torch.equal(o, g)
            elif g.numel():
                assert off(o, g.double() * factor) < 4 * U + (half_step(g.dtype) if g.dtype != F32 else 0) + (2.0 ** -25 * g.numel() ** 0.5 / float(
                    (g.double() * factor).norm()) if g.dtype == F16 else 0)      # (fp16 below 2^-14 has steps of 2^-24)


def test_gradients_of_any_layout_are_clipped(K):
    base = rand(40, 30, seed=1)
    conv = rand(16, 8, 3, 3, seed=2).contiguous(memory_format=torch.channels_last)
    sliced = rand(64, 65, seed=3)[:, 1:50]
    part = rand(1001, seed=4)[1:]
    grads = [base.t(), conv, sliced, part, rand(6, 4, seed=5)[::2], rand(5, 1, 7, seed=6).transpose(0, 2)]
    want = norm_of(grads, 2)
    factor = (1.0 / (want + 1e-6))
    expect = [g.double() * factor for g in grads]
    around = sliced.clone()
    for layout in (lambda g: torch.empty_like(g), lambda g: torch.empty(g.shape, device='cuda'), lambda g: torch.empty(*g.shape, 2, device='cuda')[..., 0]):
        outs = [layout(g) for g in grads]
        assert abs(float(K.clip_grad_norm(grads, 1.0, outs=outs)) - want) <= 2 * U * want
        assert all(off(o, e) < 4 * U for o, e in zip(outs, expect))
    assert torch.equal(sliced, around)
    whole = sliced._base.clone()
    K.clip_grad_norm(grads, 1.0)
    assert all(off(g, e) < 4 * U for g, e in zip(grads, expect))
    assert torch.equal(sliced._base[:, 50:], whole[:, 50:]) and torch.equal(sliced._base[:, :1], whole[:, :1])
    assert abs(float(K.grad_norm([torch.ones(3, 1, device='cuda').expand(3, 5)])) - math.sqrt(15)) < 1e-6


def test_results_may_be_float32(K):
    grads = [rand(300, 7, seed=1, dtype=BF16), rand(55, seed=2, dtype=F16), rand(9, seed=3)]
    outs = [torch.empty(g.shape, device='cuda') for g in grads]
    want = norm_of(grads, 2)
    K.clip_grad_norm(grads, want / 2, outs=outs)
    assert all(off(o, g.double() * (want / 2 / (want + 1e-6))) < 4 * U for o, g in zip(outs, grads))


def test_a_gradient_listed_twice_counts_once(K):
    g, h = rand(100, seed=1), rand(50, seed=2)
    want = norm_of([g, h], 2)
    assert abs(float(K.grad_norm([g, h, g.view(10, 10)])) - want) <= 2 * U * want
    expect = [t.double() * (0.5 / (want + 1e-6)) for t in (g, h)]
    outs = [torch.empty(100, device='cuda'), torch.empty(50, device='cuda'), torch.empty(10, 10, device='cuda')]
    assert abs(float(K.clip_grad_norm([g, h, g.view(10, 10)], 0.5, outs=outs)) - want) <= 2 * U * want
    assert torch.equal(outs[0], outs[2].flatten()) and off(outs[0], expect[0]) < 4 * U
    K.clip_grad_norm([g, h, g], 0.5)
    assert off(g, expect[0]) < 4 * U and off(h, expect[1]) < 4 * U


def test_norms_beyond_the_range_of_squares(K):
    big, small = torch.full((1000,), 1e30, device='cuda'), torch.full((1000,), 1e-30, device='cuda')
    assert abs(float(K.grad_norm([big])) / (1e30 * math.sqrt(1000)) - 1) < 1e-6
    assert abs(float(K.grad_norm([small])) / (1e-30 * math.sqrt(1000)) - 1) < 1e-6
    K.clip_grad_norm([big], 2.0)
    assert off(big, torch.full((1000,), 2 / math.sqrt(1000), device='cuda')) < 4 * U
    top = torch.full((1000,), 3e38, device='cuda')                  # the norm itself has no float32: infinite, the factor is not
    assert float(K.clip_grad_norm([top], 1.0)) == float('inf')
    assert off(top, torch.full((1000,), 1 / math.sqrt(1000), device='cuda')) < 1e-5     # (a factor below 2^-126 has few digits)


@pytest.mark.parametrize('kind', [2, 1, float('inf')])
@pytest.mark.parametrize('bad', [float('nan'), float('inf'), -float('inf')])
def test_norms_of_gradients_that_are_not_finite(K, kind, bad):
    for at in (0, 70000):
        grads = [rand(9, seed=1), rand(100000, seed=2), rand(9, seed=3)]
        grads[1][at] = bad
        want = [g.clone() for g in grads]
        got = K.clip_grad_norm(grads, 1.0, kind)
        assert math.isnan(float(got)) if math.isnan(bad) else float(got) == float('inf')
        factor = float('nan') if math.isnan(bad) else 0.0
        for g, w in zip(grads, want):
            assert torch.equal(torch.isnan(g), torch.isnan(w * factor)) and torch.equal(torch.nan_to_num(g), torch.nan_to_num(w * factor))


def test_clipping_to_nothing_and_of_nothing(K):
    g = rand(100, seed=1)
    K.clip_grad_norm([g], 0.0)
    assert not g.any()
    assert float(K.clip_grad_norm([g], 1.0)) == 0 and not g.any()
    assert float(K.grad_norm([torch.empty(0, device='cuda')])) == 0
    assert float(K.clip_grad_norm([torch.empty(0, 3, device='cuda')], 1.0)) == 0


def test_norms_refuse(K):
    g = rand(8, seed=1)
    for call, kind in [(lambda: K.grad_norm([]), ValueError), (lambda: K.grad_norm([g], 3), ValueError), (lambda: K.grad_norm([g.double()]), TypeError),
                       (lambda: K.grad_norm([g, g.cpu()]), RuntimeError), (lambda: K.clip_grad_norm([g], -1.0), ValueError),
                       (lambda: K.clip_grad_norm([g], float('nan')), ValueError), (lambda: K.clip_grad_norm([g], 1.0, outs=[]), ValueError),
                       (lambda: K.clip_grad_norm([g], 1.0, outs=[g[:4]]), ValueError), (lambda: K.clip_grad_norm([g], 1.0, outs=[g.bfloat16()]), ValueError),
                       (lambda: K.clip_grad_norm([g[:1].expand(8)], 1.0), ValueError)]:
        with pytest.raises(kind):
            call()


# ------------------------------------------------------------------------------------------------ streams and graphs
def test_operators_run_on_the_current_stream(K):
    """On a side stream, behind work of that stream that is still running."""
    side = torch.cuda.Stream()
    x, logits = rand(2000, 768, seed=1), rand(64, 5000, seed=2)
    u = torch.rand(64, device='cuda')
    with torch.cuda.stream(side):
        a = torch.zeros(4096, 4096, device='cuda')
        for _ in range(20):
            a = a @ a
        z = x + a[0, 0]
        y, mean, rstd = K.layer_norm(z)
        grads = K.layer_norm_backward(y, z, mean, rstd)
        drawn = K.sample_filtered(logits + a[0, 0], u, top_p=0.9, check=False)
        clipped = [z.clone()]
        norm = K.clip_grad_norm(clipped, 1.0)
    torch.cuda.synchronize()
    y2, mean2, rstd2 = K.layer_norm(x)
    assert torch.equal(y, y2) and all(torch.equal(p, q) for p, q in zip(grads, K.layer_norm_backward(y2, x, mean2, rstd2)))
    assert torch.equal(drawn, K.sample_filtered(logits, u, top_p=0.9)) and torch.equal(norm, K.grad_norm([x]))
    K.clip_grad_norm([x], 1.0)
    assert torch.equal(clipped[0], x)


def test_two_captured_graphs_replayed_side_by_side(K):
    """Each graph has scratch memory of its own: replays on two streams at once, several times, against the eager results."""
    def program(seed):
        x, logits = rand(3000, 768, seed=seed), rand(300, 9000, seed=seed + 1)
        g, u = rand(3000, 768, seed=seed + 2), torch.rand(300, device='cuda', generator=torch.Generator('cuda').manual_seed(seed))
        grads = gradients([(700, 300), (5000,), (64, 3, 7, 7)], seed + 3)
        blocks = torch.zeros(768, 2, 2, device='cuda')

        def run():
            y, mean, rstd = K.layer_norm(x)
            back = K.layer_norm_backward(g, x, mean, rstd, blocks=blocks)
            outs = [torch.empty_like(t) for t in grads]
            return [y, *back, blocks, K.sample_filtered(logits, u, top_k=300, top_p=0.9, check=False), K.clip_grad_norm(grads, 0.5, outs=outs), *outs]
        return (x, logits, g, grads), run
    made = []
    for seed in (1, 20):
        inputs, run = program(seed)
        graph = torch.cuda.CUDAGraph()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            outs = run()
        made.append((inputs, run, graph, outs, side))
    for turn in range(4):
        for (x, logits, g, grads), _, _, outs, _ in made:
            x.mul_(1.25)
            g.add_(0.125)
            logits.mul_(0.9)
            grads[0].mul_(1.5)
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


@pytest.mark.parametrize('dtype', [F32, BF16, F16])
@pytest.mark.parametrize('rows,n', [(300, 2500), (257, 9001)])
def test_filtered_draws_of_many_rows(K, dtype, rows, n):
    print(f'sample_filtered {rows}x{n} {dtype}', flush=True)
    logits = rand(rows, n, seed=n, dtype=dtype, scale=2.5)
    for i, filters in enumerate(FILTERS):
        u = torch.rand(rows, device='cuda', dtype=torch.float64, generator=torch.Generator('cuda').manual_seed(i))
        assert torch.equal(K.sample_filtered(logits, u, **filters).cpu(), draw64(logits, u, **filters)), filters


@pytest.mark.parametrize('dtype,rows,n', [(F32, 2, 600001), (BF16, 1, 1100003), (F16, 2, 300007), (F32, 261, 140002)])
def test_filtered_draws_of_long_rows(K, dtype, rows, n):
    print(f'sample_filtered {rows}x{n} {dtype}', flush=True)
    logits = rand(rows, n, seed=n, dtype=dtype, scale=2.5)
    looked_at = slice(None, None, 52)
    for i, filters in enumerate([dict(), dict(top_k=40), dict(top_k=30000, top_p=0.9), dict(top_p=0.7), dict(top_p=0.9999), dict(min_p=0.01), dict(temperature=0.0)]):
        u = torch.rand(rows, device='cuda', dtype=torch.float64, generator=torch.Generator('cuda').manual_seed(i))
        assert torch.equal(K.sample_filtered(logits, u, **filters)[looked_at].cpu(), draw64(logits[looked_at], u[looked_at], **filters)), filters


@pytest.mark.parametrize('n', [5000, 60000])
def test_filtered_draws_of_few_levels_and_of_clusters(K, n):
    """Borders among thousands of equal classes, and among thousands whose logits differ in their last bits only."""
    gen = torch.Generator('cuda').manual_seed(n)
    rows = 6
    levels = torch.randint(0, 4, (rows, n), device='cuda', generator=gen).float() * -0.75
    levels[:, 17] = 0.5
    cluster = -20 + torch.randn(rows, n, device='cuda', generator=gen) * 1e-4
    cluster[:, n // 2] = 0
    narrow = -20 + torch.randn(rows, n, device='cuda', generator=gen) * 1e-5
    narrow[:, ::1000] -= 0.005
    narrow[:, 3] = 0
    u = torch.rand(rows, device='cuda', dtype=torch.float64, generator=gen)
    for name, logits, t in (('levels', levels, 1.0), ('levels', levels.to(BF16), 0.9), ('cluster', cluster, 5.0), ('narrow', narrow, 4.0)):
        for filters in (dict(top_p=0.3), dict(top_p=0.9), dict(top_p=0.9999), dict(top_k=2100), dict(top_k=n - 1), dict(top_k=3000, top_p=0.5),
                        dict(top_k=n - n // 3, top_p=0.95), dict(top_p=0.8, min_p=0.2), dict(top_k=4000, top_p=0.97, min_p=0.01)):
            got = K.sample_filtered(logits, u, temperature=t, **filters)
            assert torch.equal(got.cpu(), draw64(logits, u, temperature=t, **filters)), (name, logits.dtype, filters)


@pytest.mark.parametrize('dtype', [F32, BF16, F16])
@pytest.mark.parametrize('masked', ['infinite', 'lowest', 'large'])
def test_filtered_draws_of_masked_rows(K, dtype, masked):
    """Most classes masked, by -inf, the type's lowest value or -1e4: fewer classes than top_k are left in some rows."""
    rows, n = 8, 20011
    gen = torch.Generator('cuda').manual_seed(3)
    logits = rand(rows, n, seed=1, dtype=dtype, scale=2.0)
    left = torch.tensor([0.5, 0.1, 0.01, 0.001, 0.0005, 0.9, 0.0, 0.05], device='cuda').unsqueeze(1)
    mask = torch.rand(rows, n, device='cuda', generator=gen) >= left
    mask[:, 777] = False
    logits[mask] = dict(infinite=-float('inf'), lowest=torch.finfo(dtype).min, large=-1e4)[masked]
    u = torch.rand(rows, device='cuda', dtype=torch.float64, generator=gen)
    for filters in (dict(top_k=4), dict(top_k=40), dict(top_k=1500), dict(top_k=5000), dict(top_k=40, top_p=0.9), dict(top_k=9000, top_p=0.99),
                    dict(top_p=0.9), dict(top_k=30, min_p=0.1), dict(top_k=60, temperature=3.0), dict(top_k=60, temperature=1e-3)):
        got = K.sample_filtered(logits, u, **filters)
        assert torch.equal(got.cpu(), draw64(logits, u, **filters)), filters
        assert int(got[6]) == 777


def test_filtered_draws_of_infinite_temperature(K):
    """All classes that are not masked are equally likely."""
    logits, inf = rand(5, 4001, seed=1), float('inf')
    logits[:, ::2] = -inf
    u = torch.tensor([0.0, 0.25, 0.5, 0.75, 0.9999], device='cuda', dtype=torch.float64)
    want = [1, 1001, 2001, 3001, 3999]
    assert K.sample_filtered(logits, u, temperature=inf).tolist() == want
    assert K.sample_filtered(logits, u, temperature=inf, top_k=3999).tolist() == want
    got = K.sample_filtered(logits, u, temperature=inf, top_k=4)
    by_index = logits.topk(4).indices.sort(-1).values
    assert got.tolist() == [int(by_index[i, min(3, int(4 * float(u[i])))]) for i in range(5)]


def test_more_rows_than_a_launch_takes(K):
    rows = (1 << 22) + 77
    logits, u = rand(rows, 3, seed=1), torch.rand(rows, device='cuda', dtype=torch.float64, generator=torch.Generator('cuda').manual_seed(1))
    w = (logits.double() - logits.double().amax(-1, keepdim=True)).exp()
    want = (w.cumsum(-1)[:, :2] <= (u * w.sum(-1)).unsqueeze(-1)).sum(-1)
    assert torch.equal(K.sample_filtered(logits, u), want)


def test_draws_beyond_32_bits(K):
    base = rand(8, 50257, seed=1, dtype=BF16, scale=2.0)
    logits = base.repeat(5400, 1)
    assert logits.numel() > 1 << 31
    u = torch.rand(logits.shape[0], device='cuda', dtype=torch.float64, generator=torch.Generator('cuda').manual_seed(2))
    for filters in (dict(), dict(top_k=50, top_p=0.9)):
        got = K.sample_filtered(logits, u, **filters)
        assert torch.equal(got[-24:].cpu(), draw64(logits[-24:], u[-24:], **filters))
        assert torch.equal(got[-2400:], K.sample_filtered(base.repeat(300, 1), u[-2400:], **filters))
    rows = torch.zeros(0, device='cuda', dtype=F16).new_empty((1 << 31) + 5000).as_strided((3, 5000), (1 << 30, 1))
    rows.copy_(rand(3, 5000, seed=3, dtype=F16))
    assert torch.equal(K.sample_filtered(rows, u[:3], top_p=0.7).cpu(), draw64(rows, u[:3], top_p=0.7))


def test_layer_norm_beyond_32_bits(K):
    """One block of rows again and again: each row's result is the block's, and sums over rows are its sums times the repetitions, up to
    chains of at most rows / 512 + 512 additions, each off by u of the magnitudes' sum at most."""
    F, block, times = 768, 4000, 700
    x0, g0, w = rand(block, F, seed=1, dtype=BF16), rand(block, F, seed=2, dtype=BF16), rand(F, seed=3)
    x, g = x0.repeat(times, 1), g0.repeat(times, 1)
    assert x.numel() > 1 << 31
    y, mean, rstd = K.layer_norm(x, w, None, 1e-5)
    y0, mean0, rstd0 = K.layer_norm(x0, w, None, 1e-5)
    assert torch.equal(y[-block:], y0) and torch.equal(y[:block], y0) and torch.equal(mean[-block:], mean0) and torch.equal(rstd[-block:], rstd0)
    dx, dw, db = K.layer_norm_backward(g, x, mean, rstd, w)
    dx0 = K.layer_norm_backward(g0, x0, mean0, rstd0, w)[0]
    assert torch.equal(dx[-block:], dx0) and torch.equal(dx[block:2 * block], dx0)
    h = (x0.double() - mean0.double().unsqueeze(-1)) * rstd0.double().unsqueeze(-1)
    bound = (block * times / 512 + 512 + 64) * U
    for got, terms in ((dw, g0.double() * h), (db, g0.double())):
        assert bool(((got.double() - times * terms.sum(0)).abs() <= bound * times * terms.abs().sum(0)).all())


def test_norms_beyond_32_bits(K):
    n = (1 << 31) + 4099
    big = torch.full((n,), 0.5, device='cuda', dtype=BF16)
    small = torch.full((n % 1000, 3), 0.5, device='cuda')
    total = 0.5 * math.sqrt(n + small.numel())
    norm = K.clip_grad_norm([small, big], total / 4)
    assert abs(float(norm) - total) <= 4 * U * total
    want = 0.5 * (total / 4) / (float(norm) + 1e-6)
    assert bool((big[-5000:] == torch.tensor(want, device='cuda').to(BF16)).all()) and bool((big[:5000] == big[-1]).all())
    assert bool(((small.double() - want).abs() <= 4 * U * want).all())


def test_two_threads_at_once(K):
    """Two threads with a stream each call the operators at the same time: every call's result is that of the call alone."""
    import threading

    def inputs(seed):
        return (rand(200, 768, seed=seed), rand(768, seed=seed + 1), rand(64, 5000, seed=seed + 2),
                torch.rand(64, device='cuda', generator=torch.Generator('cuda').manual_seed(seed)), gradients([(300, 70), (4099,)] * 8, seed))

    def run(x, w, logits, u, grads):
        y, mean, rstd = K.layer_norm(x, w)
        outs = [torch.empty_like(t) for t in grads]
        return [y, *K.layer_norm_backward(y, x, mean, rstd, w), K.sample_filtered(logits, u, top_k=50), K.sample_filtered(logits, u, top_p=0.9, check=False),
                K.clip_grad_norm(grads, 0.1, outs=outs), *outs]
    made = [inputs(seed) for seed in (1, 50)]
    want = [run(*m) for m in made]
    torch.cuda.synchronize()
    wrong, errors = [], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for turn in range(100):
                    got = run(*made[i])
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


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('n', [900, 30011])
def test_filtered_draws_where_min_p_and_top_p_are_close(K, dtype, n):
    """min-p from far below top-p's border to far above it, the share of its classes on both sides of top_p."""
    rows = 12
    logits = rand(rows, n, seed=n, dtype=dtype, scale=2.0)
    u = torch.rand(rows, device='cuda', dtype=torch.float64, generator=torch.Generator('cuda').manual_seed(7))
    w = torch.softmax(logits.double(), -1)
    for min_p in (0.002, 0.05, 0.3, 1.0):
        share = float((w * (w >= min_p * w.amax(-1, keepdim=True))).sum(-1).mean())
        for top_p in (share - 0.05, share - 1e-3, share, share + 5e-4, share + 2e-3, share + 0.05):
            filters = dict(top_p=min(max(top_p, 1e-3), 0.9999), min_p=min_p)
            for t in (1.0, 0.3):
                assert torch.equal(K.sample_filtered(logits, u, temperature=t, **filters).cpu(), draw64(logits, u, temperature=t, **filters)), (filters, t)


def levels(rows_of, u):
    """Logits of rows given as [(value, how often), ...], each row in an order of its own, and one number per row."""
    n = sum(count for _, count in rows_of[0])
    gen = torch.Generator().manual_seed(n)
    rows = [torch.cat([torch.full((count,), value, dtype=torch.float64) for value, count in row])[torch.randperm(n, generator=gen)] for row in rows_of]
    return torch.stack(rows).float().cuda(), torch.tensor(u, device='cuda', dtype=torch.float64).expand(len(rows)).contiguous()


@pytest.mark.parametrize('row,t,p,m', [
    ([(100000.0, 1), (99999.9921875, 145), (99999.9765625, 254)], 0.01, 0.7244, 0.277),
    ([(1e6, 1), (999994.75, 3666), (999993.9375, 363)], 1.0, 0.95941, 0.0035),
    ([(300.0, 1), (299.99475, 3666), (299.99395, 363)], 0.001, 0.9594, 0.0035),
    ([(2000.0, 1), (1999.947, 3666), (1999.939, 363)], 0.01, 0.9594, 0.0035)])
def test_filtered_draws_of_few_levels_far_from_zero(K, row, t, p, m):
    """min-p keeps a little more than top-p would: top-p has to cut.  float32 has some steps only between these logits."""
    for u in (0.0, 0.5, 0.99, 0.999, 0.9999, 0.99999, 1 - 2.0 ** -53):
        logits, numbers = levels([row] * 8, u)
        for top_p in (p, p - 1e-4, p + 1e-4, p + 2e-3):
            filters = dict(temperature=t, top_p=top_p, min_p=m)
            assert torch.equal(K.sample_filtered(logits, numbers, **filters).cpu(), draw64(logits, numbers, **filters)), (u, top_p)
            each = dict(temperature=torch.full((8,), t, device='cuda'), top_p=torch.full((8,), top_p, device='cuda'), min_p=torch.full((8,), m, device='cuda'))
            assert torch.equal(K.sample_filtered(logits, numbers, **each).cpu(), draw64(logits, numbers, **each)), (u, top_p)


@pytest.mark.parametrize('n', [400, 3000, 30000])
@pytest.mark.parametrize('offset', [-1e4, 1e4, 1e5, 1e6])
def test_filtered_draws_with_an_offset_large_against_the_temperature(K, offset, n):
    """Two levels below the largest logit, min-p between them, top_p on both sides of what min-p keeps; and spread logits."""
    gen = torch.Generator().manual_seed(n)
    rows = 8
    for t in (0.01, 0.1, 1.0):
        for _ in range(6):
            r = torch.rand(3, generator=gen, dtype=torch.float64).tolist()
            first = 1 + int((n - 2) * (0.1 + 0.8 * r[0]))
            high = torch.tensor(offset, dtype=torch.float64)
            step = float(torch.finfo(F32).eps) * abs(offset)           # one to two steps of float32
            a, b = (float((high - max(t * d, least * step)).float()) for d, least in ((0.5 + 4 * r[1], 1), (5.0 + 3 * r[2], 3)))
            wa, wb = (math.exp((x - offset) / t) for x in (a, b))
            if wb < 1e-30 or wa / wb < 1.01:
                continue
            kept = 1 + first * wa
            share, m = kept / (kept + (n - 1 - first) * wb), math.sqrt(wa * wb)
            logits, u = levels([[(offset, 1), (a, first), (b, n - 1 - first)]] * rows, 0.0)
            u = torch.linspace(0, 1, rows, device='cuda', dtype=torch.float64) * (1 - 1e-9)
            for d in (-0.02, -2e-3, -1.1e-3, -5e-4, 5e-4, 1.1e-3, 2e-3):
                if 0 < share + d < 1:
                    filters = dict(temperature=t, top_p=share + d, min_p=m)
                    assert torch.equal(K.sample_filtered(logits, u, **filters).cpu(), draw64(logits, u, **filters)), (t, first, a, b, d)
        logits = rand(rows, n, seed=n, scale=2 * t, shift=offset)
        for filters in (dict(top_p=0.6, min_p=0.05), dict(top_p=0.9, min_p=0.2), dict(top_k=n // 3, top_p=0.8, min_p=0.01), dict(top_p=0.3)):
            got = K.sample_filtered(logits, u, temperature=t, **filters)
            assert torch.equal(got.cpu(), draw64(logits, u, temperature=t, **filters)), (t, filters)


@pytest.mark.parametrize('results', ['in place', 'copies'])
@pytest.mark.parametrize('usual', [True, False])
def test_clipped_tensors_are_marked_as_changed(K, usual, results):
    """As every operation in place does, for autograd to notice; the norm alone changes nothing.  ``usual``: the call in one step."""
    grads = gradients([(30, 40), (7,), (64, 3, 5, 5)], 1)
    if not usual:
        grads.append(rand(20, 30, seed=2)[:, ::2])
    outs = None if results == 'in place' else [torch.empty_like(g) for g in grads]
    changed = grads if outs is None else outs
    before = [t._version for t in changed]
    K.grad_norm(grads)
    assert [t._version for t in changed] == before
    K.clip_grad_norm(grads, 0.5, outs=outs)
    assert all(t._version > v for t, v in zip(changed, before))
    if outs is not None:
        assert all(g._version == 0 for g in grads)
    # a graph that keeps one of them
    x = torch.ones_like(changed[0]).requires_grad_()
    loss = (x * changed[0]).sum()
    K.clip_grad_norm(grads, 0.25, outs=outs)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        loss.backward()
    with torch.inference_mode():
        made = gradients([(30, 40), (7,), (64, 3, 5, 5)], 3)
        want = K.clip_grad_norm(made, 0.5)
    assert abs(norm_of(made, 2) - 0.5) < 1e-5 and float(want) > 0.5
    K.clip_grad_norm(made, 0.25)                   # (such tensors keep no count)
    assert abs(norm_of(made, 2) - 0.25) < 1e-5


@pytest.mark.parametrize('rows,F', [(1, 16), (257, 100), (300, 768), (19, 2050), (6, 8191), (3, 16400)])
@pytest.mark.parametrize('xt', [F32, BF16, F16])
def test_symmetric_fisher_blocks_stay_symmetric(K, rows, F, xt):
    """To the bit: both cross terms are one sum.  Block by block against the definition: each term is an fp32 sum in chains of at most 256
    products, joined by at most 64 more, each addition off by u of the sum of magnitudes; h is off by 64 u of what it is a difference of
    (twice in its square) and the products' own roundings stay below another 64 u."""
    x, g, w = rand(rows, F, seed=1, dtype=xt, scale=2.0, shift=0.5), rand(rows, F, seed=2, dtype=xt), rand(F, seed=3)
    _, mean, rstd = K.layer_norm(x, w)
    h = norm64(x, w, None, 1e-5)[3]
    g64 = g.double()
    size = h.abs() + 1 + x.double().abs() * rstd.double().unsqueeze(-1)
    terms = torch.stack([(g64 * h).square().sum(0), (g64 * g64 * h).sum(0), (g64 * g64).sum(0)], -1)
    sizes = torch.stack([(g64 * size).square().sum(0), (g64 * g64 * size).sum(0), (g64 * g64).sum(0)], -1)
    blocks = rand(F, 2, 2, seed=5)
    blocks[:, 1, 0] = blocks[:, 0, 1]
    first = blocks.clone()
    for beta in (0.5, 0.0):
        before = first.double() if beta else torch.zeros_like(first, dtype=torch.float64)
        blocks.copy_(first)
        K.layer_norm_backward(g, x, mean, rstd, w, blocks=blocks, alpha=0.25, beta=beta)
        assert torch.equal(blocks[:, 0, 1], blocks[:, 1, 0])
        for at, q in (((0, 0), 0), ((0, 1), 1), ((1, 1), 2)):
            old = before[:, at[0], at[1]]
            want, most = beta * old + 0.25 * terms[:, q], beta * old.abs() + 0.25 * sizes[:, q]
            assert bool(((blocks[:, at[0], at[1]].double() - want).abs() <= (min(rows, 256) + 3 * 64 + 64) * U * most).all()), (beta, at)
