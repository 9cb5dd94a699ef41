"""Layers on the framework's own kernels, as functions and as modules that stand in for torch's: layer norm (csrc/layer_norm.hip),
embeddings (csrc/embedding.hip), the cross entropy of a model's last linear layer (csrc/linear_cross_entropy.hip), and linear layers and
GELU that keep their inputs in 8 bits for the backward pass (csrc/keep_8bit.hip).

Under the hooks of a gradient maker a FusedLayerNorm has its unit-wise Fisher blocks computed by its own backward pass, from the values
that pass reads anyway, where torch.nn.LayerNorm has its output and output gradient read once more
(asdl/operations/layernorm.py:69-78)."""
import torch
import torch.nn as nn
import torch.nn.functional as F

from . import kernels

__all__ = ['layer_norm', 'FusedLayerNorm', 'fuse_layer_norms', 'linear_cross_entropy', 'embedding', 'FusedEmbedding', 'fuse_embeddings', 'gelu_8bit',
           'linear_8bit', 'GELU8bit', 'Linear8bit', 'keep_activations_8bit']


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


class _Last(torch.autograd.Function):
    """Gradients in a graph of their own, which has no way back (see _Once).  gradients(g) is called once; ``tensors``: what it reads."""

    @staticmethod
    def forward(ctx, gradients, name, g, *tensors):
        ctx.name = name
        return gradients(g)

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError(f'{ctx.name}() is differentiable once (once_differentiable): it has no second derivative.')


def _last(gradients, name, g, *tensors):
    """gradients(g), or the same in a graph where one is asked for (create_graph)."""
    return _Last.apply(gradients, name, g, *tensors) if torch.is_grad_enabled() else gradients(g)


def _through(t):
    """A leaf behind a node of its own, which _wanted() can ask about (the engine does not say it of leaves themselves)."""
    return t.view_as(t) if t is not None and t.requires_grad and t.grad_fn is None and torch.is_grad_enabled() else t


def _wanted(ctx, index):
    """Whether the running backward pass takes the gradient of an input: one that is restricted to other leaves or edges, as the passes
    of a sampled Fisher matrix are, does not."""
    node = ctx.next_functions[index][0] if ctx.needs_input_grad[index] else None
    return node is not None and torch._C._will_engine_execute_node(node)


def _autocast(*tensors):
    """Floating-point tensors in the type that a linear layer computes in, autocast's where it is on; leaves behind nodes of their own."""
    if torch.is_autocast_enabled('cuda'):
        dtype = torch.get_autocast_dtype('cuda')
        tensors = (t if t is None else t.to(dtype) for t in tensors)
    return tuple(_through(t) for t in tensors)


# ------------------------------------------------------------------------------ the loss at the vocabulary's end
class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, h, weight, target, bias, ignore_index, reduction):
        loss, lse = kernels.linear_cross_entropy(h, weight, target, bias, ignore_index, reduction)
        ctx.save_for_backward(h, weight, target, bias, lse)
        ctx.options = ignore_index, reduction
        return loss

    @staticmethod
    def backward(ctx, g):
        h, weight, target, bias, lse = ctx.saved_tensors
        need = [_wanted(ctx, i) for i in (0, 1, 3)]
        dh, dw, db = _last(lambda g: kernels.linear_cross_entropy_backward(g, h, weight, target, lse, bias, *ctx.options, *need), 'linear_cross_entropy', g,
                           h, weight, bias)
        return dh, dw, None, db, None, None


def linear_cross_entropy(input, weight, target, bias=None, ignore_index=-100, reduction='mean'):
    """torch.nn.functional.cross_entropy(torch.nn.functional.linear(input, weight, bias), target) without the logits: they are formed in pieces of
    the classes, forward and once more on the way back, and never kept.  input [..., features] and weight [classes, features] (a model's head)
    of one type, float32, bfloat16 or float16; under autocast both are cast to its type, as a linear layer does.  target [...] int64;
    the loss is float32.  Differentiable once.  A gradient maker takes it as its loss call: the model call then returns the input of the head,
    e.g. ``maker.setup_loss_call(linear_cross_entropy, maker.setup_model_call(features, x), head.weight, target)`` (not with a sampled or
    exact Fisher matrix, which need the logits)."""
    input, weight, bias = _autocast(input, weight, bias)
    return _LinearCrossEntropy.apply(input, weight, target, bias, ignore_index, reduction)


# ------------------------------------------------------------------------------ embeddings
class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, weight, padding_idx, scale):
        ctx.save_for_backward(tokens)
        ctx.options = weight.shape[0], scale, padding_idx
        ctx.weight_dtype = weight.dtype
        return kernels.embedding(tokens, weight, scale)

    @staticmethod
    def backward(ctx, g):
        tokens, = ctx.saved_tensors
        rows, scale, padding_idx = ctx.options
        # (linear in g: a second derivative with respect to it would be another lookup, which nobody asks for)
        return None, _last(lambda g: kernels.embedding_backward(g, tokens, rows, scale, padding_idx, dtype=ctx.weight_dtype), 'embedding', g), None, None


def embedding(input, weight, padding_idx=None, scale=1.0):
    """scale * torch.nn.functional.embedding(input, weight, padding_idx): rows of ``weight`` for int32 or int64 ``input``, differentiable once.  The
    gradient is summed by tokens in sorted order, in fp32: the same bits every time, where torch's adds rows in the order in which
    they come.  A token that names no row gives NaN and takes no gradient."""
    if padding_idx is not None and not -weight.shape[0] <= padding_idx < weight.shape[0]:
        raise ValueError(f'padding_idx has to be within {weight.shape[0]} rows. Got {padding_idx}.')
    return _Embedding.apply(input, weight, padding_idx, float(scale))


class FusedEmbedding(nn.Embedding):
    """torch.nn.Embedding (the same arguments, parameters and state dict) on embedding() above; ``scale``: a factor of the rows that are looked
    up.  max_norm, scale_grad_by_freq and sparse are not taken."""
    scale = 1.0

    def __init__(self, *args, scale=1.0, **kwargs):
        super().__init__(*args, **kwargs)
        self.scale = scale
        _plain_embedding(self)

    def forward(self, input):
        return embedding(input, self.weight, self.padding_idx, self.scale)


def _plain_embedding(module, refuse=True):
    plain = module.max_norm is None and not module.scale_grad_by_freq and not module.sparse
    if refuse and not plain:
        raise ValueError('max_norm, scale_grad_by_freq and sparse are not taken by a FusedEmbedding.')
    return plain


def _stand_in(model, kinds):
    """Modules of exactly these classes become their stand-ins in place: parameters, hooks and names stay.  Returns how many there were."""
    found = [m for m in model.modules() if type(m) in kinds and (type(m) is not nn.Embedding or _plain_embedding(m, refuse=False))]
    for m in found:
        m.__class__ = kinds[type(m)]
    return len(found)


def fuse_embeddings(model: nn.Module) -> int:
    """Makes every torch.nn.Embedding of ``model`` (not subclasses of it, nor those with max_norm, scale_grad_by_freq or sparse) a
    FusedEmbedding, in place.  Returns how many there were.  The model then runs on a ROCm device only."""
    return _stand_in(model, {nn.Embedding: FusedEmbedding})


# ------------------------------------------------------------------------------ activations in 8 bits
# The gradients below depend on an input of which only codes are kept.  For a second derivative to come across their end, whatever it is
# taken of, _last() needs a tensor whose graph leads to that input: a result without elements does, and holds nothing of it.
class _GELU8bit(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, approximate):
        y, kept = kernels.gelu_8bit(x, approximate)
        link = x.new_empty(0)
        ctx.save_for_backward(*kept, link)
        ctx.set_materialize_grads(False)
        ctx.approximate = approximate
        return y, link

    @staticmethod
    def backward(ctx, g, _):
        if g is None:
            return None, None
        codes, exponents, link = ctx.saved_tensors
        kept = kernels.Quantized8(codes, exponents)
        return _last(lambda g: kernels.gelu_8bit_backward(g, kept, ctx.approximate), 'gelu_8bit', g, link), None


def gelu_8bit(input, approximate='none'):
    """torch.nn.functional.gelu whose backward pass reads the input from 8 bits (kernels.quantize_8bit): the result is that of the input
    itself, its gradient that of the kept values.  Differentiable once."""
    if not (input.requires_grad and torch.is_grad_enabled()):
        return F.gelu(input, approximate=approximate)
    return _GELU8bit.apply(input, approximate)[0]


class _Linear8bit(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias):
        kept = kernels.quantize_8bit(x) if ctx.needs_input_grad[1] else (None, None)
        link = x.new_empty(0) if ctx.needs_input_grad[0] and ctx.needs_input_grad[1] else None
        ctx.save_for_backward(weight, *kept, link)
        ctx.set_materialize_grads(False)
        return F.linear(x, weight, bias), link

    @staticmethod
    def backward(ctx, g, _):
        if g is None:
            return None, None, None
        weight, codes, exponents, link = ctx.saved_tensors
        need_x, need_weight, need_bias = (_wanted(ctx, i) for i in range(3))
        dx = _last(lambda g: torch.matmul(g, weight), 'linear_8bit', g, weight) if need_x else None
        if not (need_weight or need_bias):
            return dx, None, None
        kept = kernels.Quantized8(codes, exponents) if need_weight else None
        return dx, *_last(lambda g: kernels.weight_grad_8bit(g, kept, need_weight, need_bias, weight.dtype), 'linear_8bit', g, link if need_weight else None)


def linear_8bit(input, weight, bias=None):
    """torch.nn.functional.linear whose backward pass reads the input from 8 bits (kernels.quantize_8bit): the result and the gradient of the
    input are those of torch's, the gradient of the weight is that of the kept values.  float32, bfloat16 or float16, autocast as there.
    Differentiable once."""
    if not torch.is_grad_enabled():          # (needs_input_grad says true of a parameter there, too)
        return F.linear(input, weight, bias)
    input, weight, bias = _autocast(input, weight, bias)
    return _Linear8bit.apply(input, weight, bias)[0]


class GELU8bit(nn.GELU):
    """torch.nn.GELU on gelu_8bit() above."""

    def forward(self, input):
        return gelu_8bit(input, self.approximate)


class Linear8bit(nn.Linear):
    """torch.nn.Linear (the same arguments, parameters and state dict) on linear_8bit() above.  The Kronecker factors that a gradient maker takes of
    it are those of the input itself."""

    def forward(self, input):
        return linear_8bit(input, self.weight, self.bias)


def keep_activations_8bit(model: nn.Module) -> int:
    """Makes every torch.nn.Linear and torch.nn.GELU of ``model`` (not subclasses of them) a Linear8bit and a GELU8bit, in place: they keep their
    inputs for the backward pass in a byte a value, and one for 128 of them.  Returns how many there were.  The model then runs on a ROCm
    device only, in float32, bfloat16 or float16."""
    return _stand_in(model, {nn.Linear: Linear8bit, nn.GELU: GELU8bit})
