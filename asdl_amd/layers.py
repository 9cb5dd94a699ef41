"""Layer norm on the kernels of csrc/layer_norm.hip as a function and as a module that stands in for torch.nn.LayerNorm.

Under the hooks of a gradient maker such a module has its unit-wise Fisher blocks computed by its own backward pass, from the values
that pass reads anyway, where torch.nn.LayerNorm has its output and output gradient read once more
(asdl/operations/layernorm.py:69-78)."""
import torch
import torch.nn as nn

from . import kernels

__all__ = ['layer_norm', 'FusedLayerNorm', 'fuse_layer_norms']


class BlocksRequest:
    """Fisher blocks that a hook wants of a backward pass that is about to run: blocks <- beta*blocks + alpha * sums for the output
    gradient ``g``.  Served once, by the backward pass or, where that does not run or sees another gradient, by settle().

    The saved tensors are unpacked by whoever serves, not for the request: torch.utils.checkpoint, which runs the forward pass again for
    them, lets a pass unpack them once.  ``keep``: other hooks follow, which may write to the gradient; the request has a copy then."""

    def __init__(self, node, g, blocks, alpha, beta, keep=False):
        self.node, self.g, self.version = node, g, g._version
        self.kept = g.clone() if keep else None
        self.blocks, self.alpha, self.beta = blocks, alpha, beta
        self.open = True
        node.blocks_requests.append(self)

    def fits(self, g):
        return g.data_ptr() == self.g.data_ptr() and g.numel() == self.g.numel() and g.is_contiguous() and self.g.is_contiguous() and \
            self.g._version == self.version

    def close(self):
        """Holds nothing from here on."""
        self.open = False
        if self.node is not None:
            self.node.blocks_requests.remove(self)
        self.node = self.g = self.kept = self.blocks = None

    def settle(self, saved=None):
        """``saved``: the node's saved tensors, where the caller has them."""
        if self.open:
            g = self.g if self.kept is None else self.kept
            if self.kept is None and g._version != self.version:
                self.close()
                raise RuntimeError('The gradient of a layer norm\'s result was changed in place, behind the hooks on this result, before its Fisher '
                                   'blocks were computed. Return a new gradient instead.')
            x, _, mean, rstd = self.node.saved_tensors if saved is None else saved
            kernels.layer_norm_backward(g.reshape(x.shape), x, mean, rstd, blocks=self.blocks, alpha=self.alpha, beta=self.beta,
                                        need_x=False, need_weight=False, need_bias=False)
            self.close()


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, out_dtype):
        y, mean, rstd = kernels.layer_norm(x, weight, bias, eps, out_dtype)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.has_bias = bias is not None
        ctx.weight_dtype = weight.dtype if weight is not None else bias.dtype if bias is not None else None
        ctx.blocks_requests = []
        return y

    @staticmethod
    def backward(ctx, g):
        if torch.is_grad_enabled():
            x, weight, _, _ = saved = ctx.saved_tensors
            return _Once.apply(ctx, saved, g, x, weight) + (None, None)
        return _LayerNorm.gradients(ctx, ctx.saved_tensors, g) + (None, None)

    @staticmethod
    def gradients(ctx, saved, g):
        x, weight, mean, rstd = saved
        blocks, alpha, beta = None, 1.0, 0.0
        for request in list(ctx.blocks_requests):         # (one for each set of hooks on the module)
            if blocks is None and request.fits(g):
                blocks, alpha, beta = request.blocks, request.alpha, request.beta
                request.close()
            else:
                request.settle(saved)
        need_x, need_weight, need_bias = ctx.needs_input_grad[:3]
        return kernels.layer_norm_backward(g, x, mean, rstd, weight, blocks, alpha, beta, need_x, need_weight, need_bias,
                                           weight_dtype=ctx.weight_dtype)


class _Once(torch.autograd.Function):
    """The gradients of _LayerNorm in a graph of their own, which has no way back.  (torch's once_differentiable() ends the graph at the
    gradients: a second derivative with respect to x is None or 0 then, where the pass does not come across the end.)"""

    @staticmethod
    def forward(ctx, node, saved, g, x, weight):
        return _LayerNorm.gradients(node, saved, g)

    @staticmethod
    def backward(ctx, *gradients):
        raise RuntimeError('layer_norm() is differentiable once (once_differentiable): it has no second derivative.')


def layer_norm(x, normalized_shape, weight=None, bias=None, eps=1e-5):
    """torch.nn.functional.layer_norm for tensors on a ROCm device (float32, bfloat16 or float16; weight and bias of the type of x or
    float32), differentiable once: a second derivative raises.  Under autocast the result is float32, as there, and x is read as it is.
    Not taken, where torch's takes them: tensors on the CPU, float64, forward mode, and torch.func (grad, vmap and their kin); each raises."""
    shape = (normalized_shape,) if isinstance(normalized_shape, int) else tuple(normalized_shape)
    if not shape or tuple(x.shape[-len(shape):]) != shape:
        raise ValueError(f'x has to end in the dimensions {shape}. Got the shape {tuple(x.shape)}.')
    for name, v in (('weight', weight), ('bias', bias)):
        if v is not None and tuple(v.shape) != shape:
            raise ValueError(f'{name} has to have the shape {shape}. Got {tuple(v.shape)}.')
    autocast = torch.is_autocast_enabled()
    out_dtype = torch.float32 if autocast else x.dtype
    if autocast:
        weight = weight.float() if weight is not None and weight.dtype != x.dtype else weight
        bias = bias.float() if bias is not None and (bias.dtype != x.dtype or (weight is not None and weight.dtype != x.dtype)) else bias
        weight = weight.float() if weight is not None and bias is not None and weight.dtype != bias.dtype else weight
    if len(shape) == 1:
        return _LayerNorm.apply(x, weight, bias, eps, out_dtype)
    flat = x.flatten(-len(shape))
    return _LayerNorm.apply(flat, None if weight is None else weight.flatten(), None if bias is None else bias.flatten(), eps, out_dtype).view(x.shape)


class FusedLayerNorm(nn.LayerNorm):
    """torch.nn.LayerNorm (the same arguments, parameters and state dict) on layer_norm() above, which says what it does not take."""

    def forward(self, input):
        return layer_norm(input, self.normalized_shape, self.weight, self.bias, self.eps)


def fuse_layer_norms(model: nn.Module) -> int:
    """Makes every torch.nn.LayerNorm of ``model`` (not subclasses of it) a FusedLayerNorm, in place: parameters, hooks and names stay.
    Returns how many there were.  The model then runs on a ROCm device only, in float32, bfloat16 or float16 (see layer_norm())."""
    found = [m for m in model.modules() if type(m) is nn.LayerNorm]
    for m in found:
        m.__class__ = FusedLayerNorm
    return len(found)
