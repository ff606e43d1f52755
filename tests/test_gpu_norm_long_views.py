"""Group norm of one very long view: the join of its chunks adds no more rounding than a short one's.

The view is a channel slice with an odd stride, which is read by single elements, so that 24 rows to
a thread make 250000 chunks of 1.5 GB. With u = 2^-24 a sum of equal terms is off by at most half a
unit for each addition in a row (the partial sums grow evenly): 12 u in a thread, 5 u over a warp,
4 u over a block's 8 lines, then whatever the chunks add, and 2 u and 5 u over the lanes of a join,
and 1 u for each of the final products and roundings: 32 u, if the chunks add nothing."""

import pytest
import torch

import diffrast_b200 as dr
from feature_reference import U

pytestmark = pytest.mark.gpu
CUDA = "cuda"


@pytest.mark.parametrize("value", [0.1, 1.7, 3.3])
def test_sums_over_a_long_view(value):
    pixels, channels = 24_000_000, 32
    x = torch.zeros(1, pixels, channels + 1, dtype=torch.float16, device=CUDA)
    x[:, ::2] = 1
    x = x[..., 1:].requires_grad_(True)
    grad = torch.full((1, pixels, channels), value, dtype=torch.float16, device=CUDA)
    bias = torch.zeros(channels, device=CUDA, requires_grad=True)
    y = dr.group_norm(x, channels, None, bias, eps=0.0)
    got, = torch.autograd.grad(y, bias, grad)
    want = pixels * float(grad[0, 0, 0])
    off = (got.double() / want - 1).abs().max().item() / U
    assert off <= 32, f"{off:.1f} u"
    # The mean is 1/2 and the deviation 1/2 exactly, so y is 1 or -1: off by what the deviation is
    # (half of the same 32 u twice, for sums of squares and of values) in float16.
    assert bool((y[:, ::2] == 1).all()) and bool((y[:, 1::2] == -1).all())
    del x, y, grad
    torch.cuda.empty_cache()
