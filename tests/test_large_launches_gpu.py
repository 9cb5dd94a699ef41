"""Calls whose threads, at one launch, would be 2^32 and more: the runtime counts them in 32 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('rows,classes', [((1 << 26) + 1000, 3), ((1 << 24) + 1000, 1025)])
def test_draws_of_more_rows_than_a_launch_takes(rows, classes):
    """Rows that have one class each: the draw is that one."""
    from asdl_amd import kernels
    print(f'sample_categorical {rows}x{classes}', flush=True)
    logits = torch.full((rows, classes), -float('inf'), device='cuda')
    only = torch.arange(rows, device='cuda').remainder_(classes)
    logits.scatter_(1, only[:, None], 0.0)
    assert torch.equal(kernels.sample_categorical(logits), only)
