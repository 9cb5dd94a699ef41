"""The cross entropy of a linear layer, embeddings and activations in 8 bits without a GPU: what a pass that goes back twice, or not at all,
asks of the kernels, which are replaced by their definitions."""
import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.utils.checkpoint import checkpoint

import asdl_amd
from tests.test_decoder_step_cpu import coarse, stand     # noqa: F401


# ------------------------------------------------------------------------------------------------ second derivatives
def gelu_of(x, w):
    return asdl_amd.gelu_8bit(x * w)


def linear_of(x, w):
    return asdl_amd.linear_8bit(x, w)


@pytest.mark.parametrize('checkpointed', [False, True])
@pytest.mark.parametrize('f', [gelu_of, linear_of])
def test_a_penalty_on_a_gradient_raises(stand, f, checkpointed):     # noqa: F811
    """Also where the first derivative's own gradient needs none (a sum), and where the penalty comes with a loss that leads to the same
    leaves; whichever of them it is taken of."""
    for first in (0, 1):
        for second in ([0], [1], [0, 1]):
            leaves = [coarse(6, 6, seed=1).requires_grad_(), coarse(6, 6, seed=2).requires_grad_()]
            y = checkpoint(f, *leaves, use_reentrant=False) if checkpointed else f(*leaves)
            d, = torch.autograd.grad(y.sum(), leaves[first], create_graph=True)
            if f is linear_of and first == 0 and second == [0]:
                # (the gradient of x does not depend on x: the loss's is left)
                got, = torch.autograd.grad(y.sum() + d.square().sum(), leaves[first])
                assert torch.equal(got, d)
                continue
            assert d.requires_grad
            with pytest.raises(RuntimeError, match='differentiable once'):
                torch.autograd.grad(y.sum() + d.square().sum(), [leaves[i] for i in second])
    leaves = [coarse(6, 6, seed=1).requires_grad_(), coarse(6, 6, seed=2).requires_grad_()]
    y = f(*leaves)
    d, = torch.autograd.grad(y.sum(), leaves[0], create_graph=True)
    with pytest.raises(RuntimeError, match='differentiable once'):
        (y.sum() + d.square().sum()).backward()


def test_gradients_with_a_graph_are_the_same(stand):     # noqa: F811
    x, w = coarse(6, 6, seed=1).requires_grad_(), coarse(6, 6, seed=2).requires_grad_()
    for f in (gelu_of, linear_of):
        want = torch.autograd.grad(f(x, w).sum(), (x, w))
        assert all(torch.equal(a, b) for a, b in zip(want, torch.autograd.grad(f(x, w).sum(), (x, w), create_graph=True)))
    for frozen in ((x.detach(), w), (x, w.detach())):
        d, = torch.autograd.grad(linear_of(*frozen).sum(), [t for t in frozen if t.requires_grad], create_graph=True)
        torch.testing.assert_close(d, torch.autograd.grad(F.linear(*frozen).sum(), [t for t in frozen if t.requires_grad])[0])


def test_nothing_of_the_input_is_held(stand):     # noqa: F811
    """The results lead to the input, but do not keep its values."""
    from torch.multiprocessing.reductions import StorageWeakRef
    for f in (asdl_amd.gelu_8bit, lambda x: asdl_amd.linear_8bit(x, nn.Parameter(torch.ones(3, 4)))):
        x = coarse(5, 4, seed=1).requires_grad_() * 1
        values = StorageWeakRef(x.untyped_storage())
        y = f(x)
        assert not values.expired()
        del x
        assert values.expired() and y.requires_grad


# ------------------------------------------------------------------------------------------------ passes without a way back
def test_nothing_is_kept_where_nothing_goes_back(stand):     # noqa: F811
    """Evaluation, and the first pass of a reentrant checkpoint: parameters need gradients there, too."""
    model = nn.Sequential(nn.Linear(4, 6), nn.GELU(), nn.Linear(6, 3))
    want = model(coarse(5, 4, seed=1)).detach()
    asdl_amd.keep_activations_8bit(model)

    def kept():
        count, stand.calls[:] = len([c for c in stand.calls if c[0] == 'keep']), []
        return count
    for mode in (torch.no_grad, torch.inference_mode):
        with mode():
            assert torch.equal(model(coarse(5, 4, seed=1)), want)
        assert kept() == 0
    x = coarse(5, 4, seed=1).requires_grad_()
    y = checkpoint(model, x, use_reentrant=True)
    assert kept() == 0 and torch.equal(y, want)
    y.sum().backward()
    assert kept() == 3 and all(p.grad is not None for p in model.parameters())
    model(x.detach())
    assert kept() == 3
    model.requires_grad_(False)
    model(x.detach())
    assert kept() == 0


# ------------------------------------------------------------------------------------------------ workspaces
def test_workspaces_hold_what_a_call_makes():
    """No copies of operands that are read where they lie, no sums of gradients that are not asked for; never more than the query for any operands."""
    from asdl_amd import _lib
    lib = _lib.load()
    F32, BF16, F16 = 0, 1, 4
    even, odd = 4096, 4098                       # stand for addresses

    def loss(dtype, rows, classes, width, gradients, h=even, w=even, pitch=None, bias=-1):
        return lib.ak_linear_cross_entropy_ws_bytes_of(h, dtype, pitch or width, w, pitch or width, bias, rows, classes, width, gradients)
    for dtype in (F32, BF16, F16):
        for rows in (1, 8, 9, 16, 17, 64, 65, 500, 8192):
            for classes in (1, 300, 50257, 1 << 25):
                for width in (1, 8, 151, 768):
                    if rows * classes > 1 << 32:
                        continue
                    for kw in (dict(), dict(h=odd), dict(w=odd), dict(pitch=width + 1), dict(bias=dtype)):
                        assert 0 < loss(dtype, rows, classes, width, 0, **kw) <= lib.ak_linear_cross_entropy_ws_bytes(dtype, rows, classes, width, 0)
                        whole = loss(dtype, rows, classes, width, 7, **kw)
                        assert whole <= lib.ak_linear_cross_entropy_ws_bytes(dtype, rows, classes, width, 1)
                        assert all(0 < loss(dtype, rows, classes, width, bits, **kw) <= whole for bits in range(1, 7))
    # the operands of 4096 x 128000 x 2048: 541 MB
    copies = (4096 + 128000) * 2048 * 2
    assert loss(F16, 4096, 128000, 2048, 0) < 40e6 and loss(F16, 4096, 128000, 2048, 0, h=odd, w=odd) - loss(F16, 4096, 128000, 2048, 0) == copies
    assert loss(F16, 4096, 128000, 2048, 7, h=odd, w=odd) - loss(F16, 4096, 128000, 2048, 7) == copies
    assert loss(F16, 4096, 128000, 2048, 7) - loss(F16, 4096, 128000, 2048, 6) >= 4096 * 2048 * 4
    assert loss(F32, 4096, 128000, 2048, 7) > 3 * copies and loss(9, 8, 8, 8, 0) == loss(BF16, 0, 8, 8, 0) == loss(BF16, 8, 8, 1 << 21, 0) == 0

    def weight(dtype, rows, width, out, gradients=3, g=even, pitch=None):
        return lib.ak_weight_grad_8bit_ws_bytes_of(g, dtype, pitch or out, rows, width, out, gradients)
    for dtype in (F32, BF16, F16):
        for rows, width, out in ((1, 1, 1), (40, 33, 70), (8192, 768, 2304), (16384, 4096, 4096)):
            for kw in (dict(), dict(g=odd), dict(pitch=out + 3), dict(gradients=1), dict(gradients=2)):
                assert 0 < weight(dtype, rows, width, out, **kw) <= lib.ak_weight_grad_8bit_ws_bytes(dtype, rows, width, out)
    assert weight(BF16, 16384, 4096, 4096, g=odd) - weight(BF16, 16384, 4096, 4096) == 16384 * 4096 * 2
    assert weight(BF16, 16384, 4096, 4096) < 16384 * 4096 * 2 + 3e6 and weight(BF16, 16384, 4096, 4096, 2) < 3e6 and weight(9, 4, 4, 4) == weight(BF16, 0, 4, 4) == 0

    # the entry points ask for no more and no less (the call itself is not made: a byte is missing)
    a = even
    need = loss(BF16, 8192, 50257, 768, 0)
    assert lib.ak_linear_cross_entropy(a, BF16, 768, a, 768, None, -1, a, 8192, 50257, 768, -100, 2, a, a, a, need - 1, None) == -2
    for bits in (1, 2, 3, 7):
        need = loss(BF16, 8192, 50257, 768, bits, bias=BF16)
        out = [a if bits & b else None for b in (1, 2, 4)]
        assert lib.ak_linear_cross_entropy_backward(a, a, BF16, 768, a, 768, a, BF16, a, a, 8192, 50257, 768, -100, 2, *out, a, need - 1, None) == -2
    assert lib.ak_weight_grad_8bit(a, BF16, 4096, a, a, 16384, 4096, 4096, a, a, BF16, a, weight(BF16, 16384, 4096, 4096) - 1, None) == -2
