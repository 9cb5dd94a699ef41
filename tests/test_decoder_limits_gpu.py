"""The cross entropy of a linear layer, embeddings and activations in 8 bits at the ends of what they take, against their definitions in
64 bits.  The tolerances are those of test_decoder_step_gpu; what a test adds to them it derives."""
import math

import pytest
import torch

from tests.test_decoder_step_gpu import BF16, F16, F32, INF, K, U, check_loss, gelu64, gradient_of, half_step, ints, loss64, rand, within     # noqa: F401

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ cross entropy of a linear layer
@pytest.mark.parametrize('dtype', [F32, BF16, F16])
@pytest.mark.parametrize('rows', [8, 100, 700])
@pytest.mark.parametrize('mask', [-INF, torch.finfo(F32).min, -1e30, -1e10, -3e6, -1e5])
def test_linear_cross_entropy_of_neighbouring_masked_classes(K, mask, rows, dtype):     # noqa: F811
    """The classes of whole tiles taken out, as those behind a vocabulary that is padded: loss and gradients are those of the others.  (A
    share of the masked classes is 0 in 64 bits, too.)"""
    classes, width = 2000, 64
    h, w = rand(rows, width, seed=1, dtype=dtype), rand(classes, width, seed=2, dtype=dtype, scale=0.2)
    b = rand(classes, seed=3)
    b[:300], b[1100:] = mask, mask
    t = 300 + ints(800, rows, seed=4)
    check_loss(K, h, w, t, b, g=gradient_of('mean', t, 5))
    loss, lse = K.linear_cross_entropy(h, w, t, b, reduction='none')
    _, dw, db = K.linear_cross_entropy_backward(torch.ones_like(loss), h, w, t, lse, b, reduction='none')
    for d in (dw, db):
        assert bool((d[:300] == 0).all()) and bool((d[1100:] == 0).all()) and bool((d[300:1100] != 0).any())


@pytest.mark.parametrize('dtype', [F32, BF16, F16])
@pytest.mark.parametrize('rows', [8, 100, 700])
def test_linear_cross_entropy_of_a_row_of_the_lowest_values(K, rows, dtype):     # noqa: F811
    """All scores are the lowest float32 number (scores of less than half a step of it, 2^103, are lost in the sum): the loss is the log of
    the number of classes, as torch's."""
    h, w = rand(rows, 64, seed=1, dtype=dtype), rand(2000, 64, seed=2, dtype=dtype)
    loss, _ = K.linear_cross_entropy(h, w, ints(2000, rows, seed=3), torch.full((2000,), torch.finfo(F32).min, device='cuda'), reduction='none')
    within(loss, torch.full_like(loss, math.log(2000), dtype=torch.float64), torch.full_like(loss, 2.0 ** -20 * 9, dtype=torch.float64), 'loss')


@pytest.mark.parametrize('dtype', [F32, BF16, F16])
def test_linear_cross_entropy_beside_rows_of_large_scores(K, dtype):     # noqa: F811
    """A row of scores beyond 2^20 leaves the bits of its neighbours as they are."""
    h, w, t = rand(300, 64, seed=1, dtype=dtype), rand(900, 64, seed=2, dtype=dtype, scale=0.5), ints(900, 300, seed=3)
    loss, lse = K.linear_cross_entropy(h, w, t, reduction='none')
    g = gradient_of('none', t, 4)
    dh = K.linear_cross_entropy_backward(g, h, w, t, lse, reduction='none')[0]
    large = h.clone()
    large[[5, 177]] = 6e4 * w[t[[5, 177]]].float().sign().to(dtype)          # (some 6e4 * 64 * 0.4 = 1.5e6)
    other, lse = K.linear_cross_entropy(large, w, t, reduction='none')
    rest = torch.ones(300, dtype=torch.bool, device='cuda')
    rest[[5, 177]] = False
    assert torch.equal(other[rest], loss[rest])
    assert torch.equal(K.linear_cross_entropy_backward(g, large, w, t, lse, reduction='none')[0][rest], dh[rest])


@pytest.mark.parametrize('dtype', [F32, BF16, F16])
@pytest.mark.parametrize('rows', [3, 70])
def test_linear_cross_entropy_of_the_last_token_of_long_sequences(K, rows, dtype):     # noqa: F811
    """Rows further apart than the entry point takes them: 4096 * 768 elements."""
    hidden = rand(rows, 4096, 768, seed=1, dtype=dtype)
    w, t = rand(500, 768, seed=2, dtype=dtype, scale=0.07), ints(500, rows, seed=3)
    check_loss(K, hidden[:, -1], w, t, g=gradient_of('mean', t, 4))
    assert all(torch.equal(a, b) for a, b in zip(K.linear_cross_entropy(hidden[:, -1], w, t), K.linear_cross_entropy(hidden[:, -1].contiguous(), w, t)))


def test_linear_cross_entropy_of_weights_far_apart(K):     # noqa: F811
    w = rand(40, (1 << 21) + 8, seed=1, dtype=BF16)[:, 3:75]
    h, t = rand(90, 72, seed=2, dtype=BF16), ints(40, 90, seed=3)
    check_loss(K, h, w, t, g=gradient_of('mean', t, 4))


def test_weight_gradients_of_rows_far_apart(K):     # noqa: F811
    g = rand(40, (1 << 24) + 8, seed=1, dtype=BF16)[:, 5:29]
    kept = K.quantize_8bit(rand(40, 72, seed=2, dtype=BF16))
    assert all(torch.equal(a, b) for a, b in zip(K.weight_grad_8bit(g, kept), K.weight_grad_8bit(g.contiguous(), kept)))


def test_memory_of_a_decoders_loss(K):     # noqa: F811
    """8192 x 768 x 50257: no copies of the operands (90 MB), and nothing for a gradient that is not asked for."""
    h, w, t = rand(8192, 768, seed=1, dtype=BF16), rand(50257, 768, seed=2, dtype=BF16, scale=0.03), ints(50257, 8192, seed=3)

    def peak(call):
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        out = call()
        return out, torch.cuda.max_memory_allocated() - before
    (loss, lse), used = peak(lambda: K.linear_cross_entropy(h, w, t))
    assert used < 20e6                            # (8 bytes for a row and 256 classes: 13 MB)
    piece, results, sums = 8192 * 25344 * 2, (8192 + 50257) * 768 * 2, 8192 * 768 * 4
    g = torch.ones_like(loss)
    for at in (h, torch.cat([h, h[:, :8]], 1)[:, :768]):          # (in one step, and by Python's way)
        _, used = peak(lambda: K.linear_cross_entropy_backward(g, at, w, t, lse))
        # (the sum over a piece's 25344 classes is in six parts: the query says 566.3 MB with dh, 415.3 MB without, which is 6 * 25.2 MB)
        assert used < piece + results + 6 * sums + 3e6
        _, used = peak(lambda: K.linear_cross_entropy_backward(g, at, w, t, lse, need_h=False))
        assert used < piece + 50257 * 768 * 2 + 3e6
    g = rand(8192, 2304, seed=4, dtype=BF16)
    kept = K.quantize_8bit(h)
    for at in (g, torch.cat([g, g[:, :8]], 1)[:, :2304]):
        _, used = peak(lambda: K.weight_grad_8bit(at, kept))
        assert used < 8192 * 768 * 2 + 4 * 2304 * 768 * 4 + 2304 * 768 * 2 + 2e6          # (the input, four parts of the sum, the result)
        _, used = peak(lambda: K.weight_grad_8bit(at, kept, need_weight=False))
        assert used < 2e6


# ------------------------------------------------------------------------------------------------ launches of 2^32 threads and more
def test_linear_cross_entropy_of_more_tiles_than_a_launch_takes(K):     # noqa: F811
    """2^23 tiles of 512 threads and more: rows at both ends, and the sum of all."""
    rows, classes, width = (1 << 22) + 1000, (1 << 17) + 300, 8
    print(f'linear_cross_entropy {rows}x{classes}x{width}', flush=True)
    h, w = rand(rows, width, seed=1, dtype=BF16), rand(classes, width, seed=2, dtype=BF16, scale=0.3)
    t, at = ints(classes, rows, seed=3), torch.cat([torch.arange(300, device='cuda'), rows - 300 + torch.arange(300, device='cuda')])
    loss, lse = K.linear_cross_entropy(h, w, t, reduction='none')
    want = loss64(h[at], w, t[at], reduction='none')
    within(lse[at], *want['lse'], 'lse')
    within(loss[at], *want['loss'], 'loss')
    total = loss.double().sum()
    within(K.linear_cross_entropy(h, w, t, reduction='sum')[0], total, 2 * U * total, 'sum')


def test_activations_of_more_blocks_than_a_launch_takes(K):     # noqa: F811
    """Rows of one feature, 16 threads each."""
    rows = (1 << 28) + 1000
    print(f'quantize_8bit {rows}x1', flush=True)
    at = torch.cat([torch.arange(700, device='cuda'), (1 << 27) - 300 + torch.arange(700, device='cuda'), rows - 700 + torch.arange(700, device='cuda')])
    x = torch.zeros(rows, 1, device='cuda', dtype=BF16)
    x[at] = rand(len(at), 1, seed=1, dtype=BF16)
    kept, few = K.quantize_8bit(x), K.quantize_8bit(x[at])
    rest = torch.ones(rows, dtype=torch.bool, device='cuda')
    rest[at] = False
    assert torch.equal(kept.codes.view(torch.uint8)[at], few.codes.view(torch.uint8)) and torch.equal(kept.exponents[at], few.exponents)
    assert bool((kept.codes.view(torch.uint8)[rest] == 0).all()) and bool((kept.exponents[rest] == -127).all())
    values = K.dequantize_8bit(kept, BF16)
    assert torch.equal(values[at], K.dequantize_8bit(few, BF16)) and bool((values[rest] == 0).all())
    y, also = K.gelu_8bit(x)
    assert torch.equal(y[at], K.gelu_8bit(x[at])[0]) and bool((y[rest] == 0).all()) and torch.equal(also.exponents, kept.exponents)
    back = K.gelu_8bit_backward(y, kept)
    assert torch.equal(back[at], K.gelu_8bit_backward(y[at], few)) and bool((back[rest] == 0).all())
    del y, also, back, values
    g = torch.zeros(rows, 3, device='cuda', dtype=BF16)
    g[at] = rand(len(at), 3, seed=2, dtype=BF16)
    dw, db = K.weight_grad_8bit(g, kept, dtype=F32)
    values, gd = K.dequantize_8bit(few).double(), g[at].double()
    # (the other rows add zeros)
    within(dw, gd.t() @ values, 2 * (len(at) + 8) * U * (gd.abs().t() @ values.abs()), 'dw')
    within(db, gd.sum(0), (len(at) + 8) * U * gd.abs().sum(0), 'db')


def test_embedding_of_more_tokens_than_a_launch_takes(K):     # noqa: F811
    """Rows of one feature, eight threads each."""
    tokens = (1 << 29) + 1000
    print(f'embedding of {tokens} tokens', flush=True)
    table = rand(7, 1, seed=1, dtype=BF16)
    t = torch.arange(tokens, device='cuda', dtype=torch.int32).remainder_(7)
    y = K.embedding(t, table)
    for i in range(7):
        assert bool((y[i::7] == table[i]).all())


# ------------------------------------------------------------------------------------------------ what is written in place
def test_an_embeddings_gradient_that_is_added_to_counts_as_changed(K):     # noqa: F811
    """A graph that has saved the tensor does not go on with other values in it."""
    out, tokens, g = rand(10, 8, seed=1), ints(10, 30, seed=2), rand(30, 8, seed=3)
    x = torch.ones(10, 8, device='cuda', requires_grad=True)
    y = (x * out).sum()
    version = out._version
    K.embedding_backward(g, tokens, 10, out=out, beta=1.0)
    assert out._version > version
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.backward()
    with torch.inference_mode():
        K.embedding_backward(g, tokens, 10, out=rand(10, 8, seed=1), beta=1.0)


# ------------------------------------------------------------------------------------------------ the largest float32 numbers
def test_numbers_that_bfloat16_rounds_to_infinity(K):     # noqa: F811
    """From 2^128 - 2^119 on, in the operands that go through the matrix cores in pieces."""
    most = torch.finfo(F32).max
    large = torch.tensor([most, 2.0 ** 128 - 2.0 ** 119, 2.0 ** 128 - 2.0 ** 119 - 2.0 ** 104, 2.0 ** 127], device='cuda', dtype=torch.float64).to(F32)
    g = torch.zeros(20, 5, device='cuda')
    g[3:7, 2], g[9, 1] = large, -most
    x = torch.zeros(20, 9, device='cuda')
    x[3:7, :4], x[9, 8] = torch.eye(4, device='cuda') / 4, 0.5
    dw, db = K.weight_grad_8bit(g, K.quantize_8bit(x), need_bias=False)
    within(dw, g.double().t() @ x.double(), torch.zeros(5, 9, device='cuda', dtype=torch.float64), 'dw')         # (one product each: exact)
    for rows in (8, 100):
        h, w, t = rand(rows, 24, seed=1), rand(300, 24, seed=2), ints(300, rows, seed=3)
        h[:, 5], w[:, 5] = 0, 0
        h[::2, 5], w[7, 5], w[9, 5] = 2.0 ** -126, most, -large[1]
        check_loss(K, h, w, t, reduction='none', g=gradient_of('none', t, 4))
        check_loss(K, w[:rows].contiguous(), h, ints(rows, rows, seed=5), reduction='none')


# ------------------------------------------------------------------------------------------------ tiles of 256
@pytest.mark.parametrize('dtype', [F32, BF16, F16])
@pytest.mark.parametrize('rows,classes,width', [(1030, 5003, 1000), (2050, 5003, 1000), (300, 9001, 2050), (4100, 4100, 1030), (4200, 70001, 520)])
def test_linear_cross_entropy_of_the_widest_tiles(K, rows, classes, width, dtype):     # noqa: F811
    """Gradients whose products go by tiles of 256: with the sum over the rows in one part and (fp32) several, in several pieces of the classes, of operands
    that are copied (1030 and 2050 features) and that are not."""
    print(f'linear_cross_entropy {rows}x{classes}x{width} {dtype}', flush=True)
    h, w = rand(rows, width, seed=1, dtype=dtype), rand(classes, width, seed=2, dtype=dtype, scale=2 / math.sqrt(width))
    t = ints(classes, rows, seed=3)
    t[::7] = -100
    check_loss(K, h, w, t, rand(classes, seed=4, dtype=dtype), g=torch.tensor(1.5 if dtype != F16 else 300.0, device='cuda'))


@pytest.mark.parametrize('dtype', [F32, BF16, F16])
@pytest.mark.parametrize('rows,width,out', [(300, 2900, 3000), (1030, 4100, 2304), (70, 130, 70001)])
def test_weight_gradients_of_the_widest_tiles(K, rows, width, out, dtype):     # noqa: F811
    """More than 512 tiles of 128."""
    print(f'weight_grad_8bit {rows}x{width}->{out} {dtype}', flush=True)
    x, g = rand(rows, width, seed=rows, dtype=dtype), rand(rows, out, seed=out, dtype=dtype)
    kept = K.quantize_8bit(x)
    values, gd = K.dequantize_8bit(kept).double(), g.double()
    want, size = gd.t() @ values, gd.abs().t() @ values.abs()
    for made in (dtype, F32):
        dw, db = K.weight_grad_8bit(g, kept, dtype=made)
        tiny = 2.0 ** -25 if made == F16 else 0
        within(dw, want, half_step(made) * want.abs() + 2 * (rows + 8) * U * size + tiny, 'dw')
        within(db, gd.sum(0), half_step(made) * gd.sum(0).abs() + (rows + 8) * U * gd.abs().sum(0) + tiny, 'db')
        assert torch.equal(dw, K.weight_grad_8bit(g, kept, dtype=made)[0])


# ------------------------------------------------------------------------------------------------ the tail of GELU
def test_gelu_of_negative_numbers(K):     # noqa: F811
    """Relative to the result, which falls to 1e-32: the argument of exp(-x^2 / 2) is rounded twice and has a rounded factor, 3 u of x^2 / 2; the rest (the
    reciprocal, a polynomial of eight terms, four products, the power of two) is at most 16 u."""
    x = torch.cat([torch.linspace(-12, -1, 4001, device='cuda'), -torch.rand(4000, device='cuda', generator=torch.Generator('cuda').manual_seed(1)) * 11 - 1])
    x = x.to(F32).view(-1, 1)                     # (a block each: the kept values are x to 2^-4, all of them)
    y, kept = K.gelu_8bit(x)
    at = x.double()
    want = gelu64(x, 'none')[0]
    within(y, want, (1.5 * at * at + 16) * U * want.abs(), 'gelu')
    at = K.dequantize_8bit(kept).double()
    below = 0.5 * torch.special.erfc(-at / math.sqrt(2))
    slope = at * torch.exp(-at * at / 2) / math.sqrt(2 * math.pi)
    within(K.gelu_8bit_backward(torch.ones_like(x), kept), below + slope, (1.5 * at * at + 16) * U * (below + slope.abs()), 'its gradient')


def test_linear_cross_entropy_refuses_an_ignored_target_that_is_no_int64(K):     # noqa: F811
    """2^64 is not class 0."""
    h, w, t = rand(6, 8, seed=1), rand(10, 8, seed=2), torch.zeros(6, dtype=torch.int64, device='cuda')
    loss, lse = K.linear_cross_entropy(h, w, t)
    for ignore in (1 << 64, 1 << 63, -(1 << 63) - 1):
        with pytest.raises(ValueError, match='int64'):
            K.linear_cross_entropy(h, w, t, ignore_index=ignore)
        with pytest.raises(ValueError, match='int64'):
            K.linear_cross_entropy_backward(loss, h, w, t, lse, ignore_index=ignore)
