"""The norm of all gradients of a model, and clipping to a largest one (kernels.grad_norm, kernels.clip_grad_norm)."""
import math

import torch

from . import kernels

__all__ = ['clip_grad_norm_']


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False):
    """torch.nn.utils.clip_grad_norm_ for parameters on one ROCm device: scales their gradients in place by
    min(1, max_norm / (norm + 1e-6)) and returns the norm before, a 0-d float32 tensor.  ``norm_type``: 2, 1 or inf.  Gradients may be
    float32, bfloat16 or float16, also mixed; one that two parameters share counts once.  ``max_norm`` may be inf: the norm alone.
    ``error_if_nonfinite`` reads the norm on the host (which waits for it) and raises RuntimeError, with the gradients as they were."""
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    grads = [p.grad for p in parameters if p.grad is not None]
    if not grads:
        return torch.tensor(0.)
    if not max_norm >= 0:
        raise ValueError(f'max_norm has to be at least 0. Got {max_norm}.')
    if not error_if_nonfinite and max_norm != math.inf:
        return kernels.clip_grad_norm(grads, max_norm, norm_type)
    norm = kernels.grad_norm(grads, norm_type)
    if error_if_nonfinite and not math.isfinite(float(norm)):
        raise RuntimeError(f'The total norm of order {norm_type} for gradients is non-finite, so it cannot be clipped.')
    return norm if max_norm == math.inf else kernels.clip_grad_norm(grads, max_norm, norm_type)
