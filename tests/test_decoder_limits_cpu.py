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
