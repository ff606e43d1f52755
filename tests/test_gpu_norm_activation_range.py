"""SiLU and its slope in ``dr.group_norm`` over the whole range of float32, against 64 bits.

With weights of zero, z is the channel's bias exactly, so that the activation's own error is all
there is. With u = 2^-24, t = z / ln 2 rounded and its power of two are off by 1.23 |z| u + 4 u
relative (a product, its constant, 2^-22 for the power), which counts as an error of z of that size.
The sum, the reciprocal (within 2 u) and the products add at most 5 u to s and 6 u to 1 - s. So

- y = z s is off by (10 + 1.25 |z|) u |y| below zero, 8 u |y| + 2 u above it (|z s (1 - s)| < 0.23
  and z^2 s (1 - s) < 0.45 multiply the error of z);
- the slope s (1 + z (1 - s)) is off by 12 u (|slope'| <= 0.5 and |z slope'| <= 0.6 multiply the
  error of z, 1.1 the error of s, 0.23 that of 1 - s), whatever z;
- powers of two below 2^-126 are zero, so results below 128 * 2^-126 may be.
"""

import pytest
import torch

import diffrast_b200 as dr
from feature_reference import U

pytestmark = pytest.mark.gpu
CUDA = "cuda"
FLUSH = 2.0**-119

# Clusters, whole vectors in passes, folded pixels that start anywhere (with elements left over),
# and single elements (a slice with an odd stride) in clusters and in passes.
LAYOUTS = {"clusters": (2, 5, 5, 64, 0), "passes": (1, 70, 71, 64, 0), "turned": (2, 101, 103, 63, 0),
           "slice": (2, 5, 5, 64, 1), "slice in passes": (1, 70, 71, 64, 1)}


def silu_and_slope(z):
    z = z.double()
    s, rest = torch.sigmoid(z), torch.sigmoid(-z)
    return z * s, s * (1 + z * rest)


def run(layout, bias, dtype=torch.float32):
    """y and the gradient of bias, which gets one pixel of each channel with an upstream 1, so that
    it is the slope at bias: the first pixel, the last, and others."""
    batch, height, width, channels, extra = LAYOUTS[layout]
    gen = torch.Generator().manual_seed(3)
    x = torch.randn(batch, height, width, channels + extra, generator=gen).to(dtype).to(CUDA)[..., extra:]
    x.requires_grad_(True)
    pixel = torch.randint(0, height * width, (channels,), generator=gen)
    pixel[0::5], pixel[1::5] = 0, height * width - 1
    grad = torch.zeros(batch, height * width, channels)
    grad[batch - 1, pixel, torch.arange(channels)] = 1
    grad = grad.view(batch, height, width, channels).to(dtype).to(CUDA)
    bias = bias[:channels].to(CUDA).requires_grad_(True)
    weight = torch.zeros(channels, device=CUDA, requires_grad=True)
    y = dr.group_norm(x, channels, weight, bias, activation="silu")
    grad_x, slope = torch.autograd.grad(y, (x, bias), grad)
    assert bool((grad_x == 0).all())
    return y.detach().double().cpu().view(-1, channels), slope.double().cpu()


def within(got, want, bound):
    """Compared out of the test, so that a failure does not print the tensors."""
    ratio = ((got - want).abs() / bound).nan_to_num(nan=float("inf"))
    worst = int(ratio.view(-1, ratio.shape[-1]).amax(0).argmax())
    assert float(ratio.max()) <= 1, f"{float(ratio.max()):.3g} of the bound where {float(want[worst]):.5g} is wanted"


def values(magnitudes, seed):
    """64 float32 of both signs in an order that brings unlike ones together."""
    z = torch.cat([magnitudes, -magnitudes]).float()
    assert z.numel() == 64
    return z[torch.randperm(64, generator=torch.Generator().manual_seed(seed))]


MODERATE = torch.logspace(-2, 1.6, 32, dtype=torch.float64)          # 0.01 .. 39.8
LARGE = torch.logspace(1.2, 4.5, 32, dtype=torch.float64)             # 16 .. 31623


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("seed", range(3))
def test_slope_is_exact_to_rounding_at_any_size(layout, seed):
    for magnitudes in (MODERATE, LARGE):
        z = values(magnitudes, seed)
        y, slope = run(layout, z)
        want, want_slope = silu_and_slope(z[:slope.numel()])
        within(y[:, want > 0], want[want > 0], 8 * U * want[want > 0] + 2 * U)
        within(slope, want_slope, 12 * U)


FAR = torch.logspace(19, 38, 32, dtype=torch.float64)


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("seed", range(3))
def test_large_values_beside_very_negative_ones(layout, seed):
    """No value passes float32's range, or changes, because of what its neighbour is."""
    z = torch.cat([FAR, -torch.logspace(1.5, 2, 32, dtype=torch.float64)]).float()
    z = z[torch.randperm(64, generator=torch.Generator().manual_seed(seed))]
    y, slope = run(layout, z)
    want, want_slope = silu_and_slope(z[:slope.numel()])
    within(y[:, want > 0], want[want > 0], 8 * U * want[want > 0])
    within(slope, want_slope, 12 * U)


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("seed", range(3))
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_very_negative_values_go_to_zero(layout, seed, dtype):
    """SiLU and its slope below zero to the digits of their own size, down to the smallest float32,
    whatever the neighbours; the slope's factor 1 + z (1 - s) adds 7 u there."""
    below = [torch.linspace(20, 90, 32, dtype=torch.float64), torch.logspace(1.9, 38.5, 32, dtype=torch.float64)]
    for magnitudes in below:
        z = torch.cat([-magnitudes, MODERATE if seed == 0 else -below[0] if seed == 1 else FAR]).float()
        z = z[torch.randperm(64, generator=torch.Generator().manual_seed(seed))]
        y, slope = run(layout, z, dtype)
        z = z[:slope.numel()].double()
        want, want_slope = silu_and_slope(z)
        near = z.abs().clamp(max=128)
        rounded = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0
        within(y[:, z < 0], want[z < 0], ((10 + 1.25 * near) * U * want.abs() + rounded * want.abs() + FLUSH)[z < 0])
        within(slope[z < -20], want_slope[z < -20], ((20 + 1.25 * near) * U * want_slope.abs() + FLUSH)[z < -20])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("layout", LAYOUTS)
def test_groups_whose_squares_pass_the_range_are_normalised_to_zero(layout, dtype):
    batch, height, width, channels, extra = LAYOUTS[layout]
    gen = torch.Generator(device=CUDA).manual_seed(4)
    x = 1e20 * torch.randn(batch, height, width, channels + extra, generator=gen, device=CUDA)
    x = x.to(dtype)[..., extra:].requires_grad_(True)
    bias = torch.linspace(-3, 3, channels, device=CUDA, requires_grad=True)
    y = dr.group_norm(x, 1, None, bias)
    assert torch.equal(y.float(), bias.to(dtype).float().expand_as(y))
    grad_x, grad_bias = torch.autograd.grad(y, (x, bias), torch.ones_like(y))
    assert bool((grad_x == 0).all()) and bool((grad_bias == batch * height * width).all())
